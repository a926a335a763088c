// How the attention over a paged cache is cut into work, shared by its kernels.
//
// A tile is the query rows of up to tile_tokens new tokens of a sequence that
// read one cache head: token i's query head g of the group is row i * group + g
// (of the half that the token lies in, where the kernel has two of 128 rows).
// Its keys are cut into units of KEYS positions.  All units of all
// tiles, in the order (sequence, cache head, tile, unit), are one line, and CTA
// c of W takes the c-th equal stretch of it: sequences of any mix of lengths
// keep every SM busy to the end, and one long context is spread over all of
// them.  A stretch that covers a whole tile writes its rows out; a cut tile
// leaves (unnormalised sums, maximum, sum of weights) of each part in the
// workspace, and k_paged_merge adds the parts up in their order, so results do
// not depend on timing.  A tile counts `extra` units more than it has, for what
// it costs to begin and end (a CTA of the first, short tiles of a causal prompt
// would else be the last to finish, by a third).  Tiles of at most `snap` units
// are never cut, nor is one within its first `extra`: the cut moves to its start.
// Everything is derived on the device from the batch's arrays (each CTA finds
// its stretch with one scan), so a captured graph replays with new lengths.
#pragma once
#include "cn_heads.cuh"

namespace cn {

struct PagedArgs {
  BatchArgs b;
  const void* q;
  void* out;
  long long q_token, q_head, o_token, o_head;
  const void *k, *v;
  const uint8_t *k_exp, *v_exp;
  int heads, group;     // cache heads, query heads of each
  uint32_t group_mul;   // divides rows by group: see div_by
  int tile_tokens, half_tokens;
  int q_map;            // tcgen05 kernel: Q comes by TMA
  float scale;          // the caller's scale * log2(e)
  int causal, window;
  int rows_min, rows_max;  // this launch takes the sequences with rows in [rows_min, rows_max]
  int ctas, min_units, snap, extra;
  struct PagedCut* cuts;   // [ctas + 1]
  // A row's values in groups of four, rows beside each other: whole lines for a warp of rows.
  float* part_o;           // [2 * ctas][DIM / 4][ROWS][4]
  float* part_ml;          // [2 * ctas][ROWS][2]
  float* part_x;           // tcgen05 kernel: [ctas][2][2][DIM / 8][128][4], between the halves of a dual part
};

// Where CTA c's stretch begins: unit `start` of the line, inside tile (seq,
// head, tile), which covers [first, first + units), its `extra` ahead of the others.
struct PagedCut {
  long long start, first, total;
  int seq, head, tile, units;
};

struct PagedSeq {
  int tok0, n, len, past, tiles;
};

// n / d for mul = min(2^32 / d, 2^32 - 1): the product is the quotient or one less.
__device__ __forceinline__ int div_by(int n, int d, uint32_t mul) {
  const int q = (int)__umulhi((uint32_t)n, mul);
  return n - q * d >= d ? q + 1 : q;
}

__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int s) {
  PagedSeq q;
  const long long t0 = min((long long)max(a.b.cu[s], 0), a.b.tokens);
  const long long t1 = min((long long)max(a.b.cu[s + 1], 0), a.b.tokens);
  q.tok0 = (int)t0;
  q.n = (int)max(t1 - t0, 0ll);
  const int len = max(a.b.lengths[s], 0);
  q.past = len - q.n;
  q.len = min(len, a.b.table_width << a.b.page_shift);
  if (q.len < len && q.n > 0) set_dev_error(kErrPage);
  const int rows = q.n * a.group;
  q.tiles = rows < a.rows_min || rows > a.rows_max ? 0 : (q.n + a.tile_tokens - 1) / a.tile_tokens;
  return q;
}

// Tokens of tile b.
__host__ __device__ __forceinline__ int paged_tokens(const PagedArgs& a, const PagedSeq& q, int b) {
  return min(q.n - b * a.tile_tokens, a.tile_tokens);
}

// Keys [lo, hi) that tokens [t0, t0 + n) see, lo rounded down to a unit.
template <int KEYS>
__host__ __device__ __forceinline__ void paged_range(const PagedArgs& a, const PagedSeq& q, int t0, int n, int* lo, int* hi) {
  const int first = q.past + t0, last = first + n - 1;  // positions
  *hi = last < 0 ? 0 : a.causal ? min(q.len, last + 1) : q.len;
  *lo = a.window > 0 ? max(first - a.window + 1, 0) / KEYS * KEYS : 0;
}

// Blocks of keys of tile b: at least one, so that rows without keys are written too.
template <int KEYS>
__host__ __device__ __forceinline__ int paged_blocks(const PagedArgs& a, const PagedSeq& q, int b) {
  int lo, hi;
  paged_range<KEYS>(a, q, b * a.tile_tokens, paged_tokens(a, q, b), &lo, &hi);
  return max((hi - lo + KEYS - 1) / KEYS, 1);
}
// Units that it counts.
template <int KEYS>
__host__ __device__ __forceinline__ int paged_units(const PagedArgs& a, const PagedSeq& q, int b) {
  return paged_blocks<KEYS>(a, q, b) + a.extra;
}
// Units of every 32nd tile of one head, from tile `lane` on.  A tile's fit 32 bits (2^30 keys); those of
// a head grow with the square of a prompt: 10^6 tokens in tiles of two are 2^32.
template <int KEYS>
__host__ __device__ __forceinline__ long long paged_lane_units(const PagedArgs& a, const PagedSeq& q, int lane) {
  long long w = 0;
  for (int b = lane; b < q.tiles; b += 32) w += paged_units<KEYS>(a, q, b);
  return w;
}
// Block at which unit `at` of the line begins, in a tile from `first` on with n blocks.
__device__ __forceinline__ int paged_block_at(const PagedArgs& a, long long at, long long first, int n) {
  return (int)min(max(at - first - a.extra, 0ll), (long long)n);
}

// Exclusive scan over the block and its total; `scratch` has a long long for each warp.
template <int THREADS>
__device__ __forceinline__ long long block_scan(long long v, long long* scratch, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  // each warp adds up the warps' sums with its lanes
  long long y = lane < THREADS / 32 ? scratch[lane] : 0;
#pragma unroll
  for (int o = 1; o < THREADS / 32; o <<= 1) {
    const long long z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  *total = __shfl_sync(0xffffffffu, y, THREADS / 32 - 1);
  const long long before = __shfl_sync(0xffffffffu, y, max(warp - 1, 0));
  __syncthreads();
  return (warp ? before : 0) + x - v;  // exclusive
}

// What a block needs to find its stretch (shared memory).
template <int THREADS>
struct PagedScratch {
  long long warp_sum[THREADS / 32];
  long long seq_units[THREADS];  // units of one head of a sequence
  long long seq_at[2], seq_each[2];
  PagedCut cut[2];
};

// Units of one head of sequence s0 + (this thread), 0 behind the last.  A thread
// takes a sequence of one tile at most, a warp one of several, its lanes the
// tiles.  (A warp for every sequence is a chain of loads for each that a warp has:
// 512 sequences of one token took the four warps 100 us.)
template <int KEYS, int THREADS>
__device__ __forceinline__ long long paged_count(const PagedArgs& a, int s0, PagedScratch<THREADS>* sc) {
  constexpr int WARPS = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31;
  const int n = min(a.b.n_seqs - s0, THREADS);
  const bool by_thread = n > WARPS;
  if (by_thread) {
    long long w = 0;
    if (tid < n) {
      const PagedSeq q = paged_seq(a, s0 + tid);
      w = q.tiles > 1 ? -1 : q.tiles ? paged_units<KEYS>(a, q, 0) : 0;
      sc->seq_units[tid] = w;
    }
    if (!__syncthreads_or(w < 0)) return w;
  }
  for (int i = tid >> 5; i < n; i += WARPS) {
    if (by_thread && sc->seq_units[i] >= 0) continue;
    const PagedSeq q = paged_seq(a, s0 + i);
    long long w = paged_lane_units<KEYS>(a, q, lane);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (lane == 0) sc->seq_units[i] = w;
  }
  __syncthreads();
  return tid < n ? sc->seq_units[tid] : 0;
}

// total * c / n (64-bit divisions take about as long as all the rest here).
__device__ __forceinline__ long long paged_share(long long total, int c, int n) {
  if (total < (1ll << 22)) return (uint32_t)total * (uint32_t)c / (uint32_t)n;
  return total * c / n;
}

// The stretch of CTA `c`: sc->cut[0] where it begins, sc->cut[1] where it ends,
// valid for all threads on return.  Called by the whole block.
template <int KEYS, int THREADS>
__device__ __forceinline__ void paged_find(const PagedArgs& a, int c, PagedScratch<THREADS>* sc) {
  const int tid = threadIdx.x, lane = tid & 31;
  long long total = 0, before = 0, at = 0, each = 0;
  for (int s0 = 0; s0 < a.b.n_seqs; s0 += THREADS) {
    long long all;
    each = paged_count<KEYS, THREADS>(a, s0, sc);
    at = block_scan<THREADS>(a.heads * each, sc->warp_sum, &all);
    total += all;
  }
  // CTAs that take part: each has min_units units or more
  int ctas = a.ctas;
  if (total < (long long)a.ctas * a.min_units) ctas = max(((int)total + a.min_units - 1) / a.min_units, 1);
  const long long u[2] = {c < ctas ? paged_share(total, c, ctas) : total,
                          c + 1 < ctas ? paged_share(total, c + 1, ctas) : total};
  if (tid < 2) {
    PagedCut& k = sc->cut[tid];
    k.start = k.first = k.total = total;
    k.seq = -1;
    k.head = k.tile = k.units = 0;
  }
  __syncthreads();
  for (int s0 = 0; s0 < a.b.n_seqs; s0 += THREADS) {
    if (a.b.n_seqs > THREADS) {  // else the only pass's results are still at hand
      long long all;
      each = paged_count<KEYS, THREADS>(a, s0, sc);
      at = before + block_scan<THREADS>(a.heads * each, sc->warp_sum, &all);
      before += all;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (u[i] >= at && u[i] < at + a.heads * each) {  // the sequence's thread
        sc->cut[i].seq = s0 + tid;
        sc->seq_at[i] = at;
        sc->seq_each[i] = each;
      }
  }
  __syncthreads();
  if (tid < 64) {  // a warp for each end: the tile of its sequence
    PagedCut& k = sc->cut[tid >> 5];
    if (k.seq >= 0) {
      const PagedSeq q = paged_seq(a, k.seq);
      const long long rel = u[tid >> 5] - sc->seq_at[tid >> 5];
      const long long each1 = sc->seq_each[tid >> 5];
      const int head = (rel | each1) >> 32 ? (int)(rel / each1) : (int)((uint32_t)rel / (uint32_t)each1);
      const long long in_head = rel - head * each1;
      long long begin = 0;  // units of the head before tile b0
      for (int b0 = 0; b0 < q.tiles; b0 += 32) {
        const int n = b0 + lane < q.tiles ? paged_units<KEYS>(a, q, b0 + lane) : 0;
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        const bool here = in_head >= begin + x - n && in_head < begin + x;
        if (here) {
          k.head = head;
          k.tile = b0 + lane;
          k.first = sc->seq_at[tid >> 5] + head * each1 + begin + x - n;
          k.units = n;
          k.start = n - a.extra <= a.snap || u[tid >> 5] - k.first <= a.extra ? k.first : u[tid >> 5];
        }
        if (__any_sync(0xffffffffu, here)) break;
        begin += __shfl_sync(0xffffffffu, x, 31);
      }
    }
  }
  __syncthreads();
}

// The tile behind (s, head, b); false at the end of the line.
__device__ __forceinline__ bool paged_next(const PagedArgs& a, PagedSeq* q, int* s, int* head, int* b) {
  if (++*b < q->tiles) return true;
  *b = 0;
  if (++*head < a.heads) return true;
  *head = 0;
  while (++*s < a.b.n_seqs) {
    *q = paged_seq(a, *s);
    if (q->tiles) return true;
  }
  return false;
}

}  // namespace cn
