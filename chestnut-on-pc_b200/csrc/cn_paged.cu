// Attention of new tokens over the paged cache: the kernel for sequences of few
// query rows, and the merge of cut tiles.
//
// k_paged_few.  One token (or a few) of a sequence against its whole context
// reads K and V once and computes little with them: it is bound by HBM.  What
// counts is that enough bytes are in flight on every SM (6.5 TB/s at ~1 us of
// latency is ~45 KB an SM) and that nothing stalls the stream.  So each of the 4
// warps of a CTA works alone: it takes every fourth slice of 16 keys, keeps a
// ring of slices (K and V, cp.async, swizzled against bank conflicts) in shared
// memory, and has its own running maximum, sum and 16 x DIM accumulator; there
// is no barrier in the loop.  64 clips of 50 to 8190 tokens, 8 cache heads x 128
// bf16: 188 us, 5.7 TB/s, 88% of the copy rate.  The 16 query rows of a tile are the M of
// mma.sync m16n8k16; the tensor work is far below its rate, the unused rows of a
// single token cost nothing that is short.  The warps' results are joined once a
// tile part, through shared memory.
//
// An 8-bit cache halves the bytes (48 clips of 1200 to 4800 tokens, 16 heads x 128:
// 156 us, 3.8 TB/s; issue slots are half used and DRAM too: what is left is each
// warp's chain of expansion, products and exponentials) and is expanded on the way to the registers:
// e4m3 codes are f16 values exactly, so the products run in f16, with
// S = (q . codes_k) * 2^ek and the weights of the codes of V
// 2^(s + ev - m), m the running maximum of s + ev (in powers of two), which puts
// a row's power of two into the exponent; the sum of the weights themselves is
// that of 2^(s + ev - m) * 2^-ev in f32.  |ev| <= 48, so it loses nothing above
// 2^-78 of the largest weight.  A V row far smaller than the largest so far has
// weights below f16's normal numbers for its power of two alone; what their
// rounding takes is added in f32 (see kFewLoss).  K's and V's fragments are read as 16-byte pieces
// of a row, with the order of the head's values permuted alike in q (K) or in
// the output (V), which the sums do not see.
// Weights are rounded to 16 bits for the product with V: off by 2^-11 of themselves at
// most in f16, 2^-8 in bf16 (the outputs' own rounding), f16 ones below 2^-29 of the
// largest by 2^-40 of it.  The sum of weights is that of the unrounded ones.
#include "cn_paged.cuh"

namespace cn {

namespace {

constexpr int kFewRows = 16;
constexpr int kFewKeys = 64;   // keys of a unit: a slice of 16 for each warp
constexpr int kFewWarps = 4;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kSlice = 16;
// f16 weights are 2^15 at most, so they are normal numbers down to 2^-29 of the largest and numbers
// down to 2^-39; of bf16 ones, whose exponents are f32's, the largest is 1.
template <typename M>
struct FewTop {
  static constexpr float value = std::is_same_v<M, __half> ? 15.f : 0.f;
};
// Over an 8-bit cache a weight holds its V row's power of two.  One that is no normal number is off by
// up to 2^-25 in f16, which stands for 2^-25 / 2^ev of a weight; where that is more than kFewLoss of the
// row's sum of weights, what the rounding took is added in f32.
constexpr float kFewLow = 0x1p-14f, kFewLoss = 0x1p-33f;

template <int DIM, bool CODED>
struct Few {
  static constexpr int RB = DIM * (CODED ? 1 : 2);                    // bytes of a row
  static constexpr int Stage = 2 * kSlice * RB + (CODED ? 32 : 0);    // K, V and their 16 + 16 exponents
  static constexpr int Stages = (CODED ? 16384 : 24576) / (2 * kSlice * RB);  // a warp's ring: 3, 4, 6 or 8 slices
  static constexpr int Warp = Stage * Stages;
  static constexpr int Join = kFewWarps * kFewRows * (DIM + 4) * 4 + kFewWarps * kFewRows * 2 * 4;
  static constexpr size_t Smem = kFewWarps * Warp > Join ? kFewWarps * Warp : Join;
};

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma16816(c, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16-byte piece `ch` of row `row` of a slice: where it lies.
template <int RB, bool CODED>
__device__ __forceinline__ int few_swizzle_k(int row, int ch) {
  if constexpr (!CODED) return ch ^ (row & 7);         // ldmatrix: 8 rows, one piece each
  else if constexpr (RB == 128) return ch ^ ((row & 1) << 2);  // 4 neighbouring pieces of 2 neighbouring rows
  else return ch;                                      // 64-byte rows: two of them are one line
}
template <int RB, bool CODED>
__device__ __forceinline__ int few_swizzle_v(int row, int ch) {
  if constexpr (!CODED) return ch ^ (row & 7);
  else if constexpr (RB == 128) return ch ^ (row & 6);  // neighbouring pieces of rows 0, 2, 4, 6 (or 1, 3, 5, 7)
  else return ch ^ ((row >> 1) & 3);
}

// T: type of q, out (and of the cache unless CODED); M: of the products.
template <typename T, int DIM, bool CODED>
__global__ void __launch_bounds__(kFewThreads, CODED ? 3 : 2) k_paged_few(const PagedArgs a) {
  using F = Few<DIM, CODED>;
  using M = std::conditional_t<CODED, __half, T>;
  constexpr int RB = F::RB, ST = F::Stages;
  constexpr int KS = DIM / 16;  // k steps of q . k
  constexpr int NB = DIM / 8;   // n tiles of the output
  extern __shared__ __align__(128) uint8_t few_smem[];
  __shared__ PagedScratch<kFewThreads> sc;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  pdl_trigger();
  pdl_wait();
  paged_find<kFewKeys, kFewThreads>(a, blockIdx.x, &sc);
  long long at = sc.cut[0].start;
  const long long end = sc.cut[1].start;
  if (tid == 0) a.cuts[blockIdx.x] = sc.cut[0];
  if (at >= end) return;
  int s = sc.cut[0].seq, head = sc.cut[0].head, b = sc.cut[0].tile;
  long long first = sc.cut[0].first;
  PagedSeq sq = paged_seq(a, s);
  uint8_t* ring = few_smem + warp * F::Warp;
  const uint32_t ring_u = smem_u32(ring);
  const int page_rows = 1 << a.b.page_shift;

  while (true) {
    const int units = paged_blocks<kFewKeys>(a, sq, b);
    int lo, hi;
    const int tok0 = b * a.tile_tokens, toks = paged_tokens(a, sq, b);
    paged_range<kFewKeys>(a, sq, tok0, toks, &lo, &hi);
    const int u0 = paged_block_at(a, at, first, units), u1 = paged_block_at(a, end, first, units);
    const int rows = toks * a.group;
    auto token_of = [&](int r) { return div_by(r, a.group, a.group_mul); };
    // positions of this thread's rows g and g + 8; none: -1 sees nothing
    const int pos_a = g < rows ? sq.past + tok0 + token_of(g) : -1;
    const int pos_b = g + 8 < rows ? sq.past + tok0 + token_of(g + 8) : -1;
    // every row of the tile sees the keys [all_lo, all_hi)
    const int first_pos = sq.past + tok0, last_pos = first_pos + toks - 1;
    const int all_hi = first_pos < 0 ? 0 : a.causal ? min(sq.len, first_pos + 1) : sq.len;
    const int all_lo = a.window > 0 ? last_pos - a.window + 1 : 0;

    // ---- queries to A fragments
    uint32_t qf[KS][4];
    float rs_a = a.scale, rs_b = a.scale;  // powers of two (of log2 e / scale) that a product stands for
    {
      const int ra = min(g, rows - 1), rb = min(g + 8, rows - 1);
      const int ta = token_of(ra), tb = token_of(rb);
      const T* qa = static_cast<const T*>(a.q) + (long long)(sq.tok0 + tok0 + ta) * a.q_token +
                    (long long)(head * a.group + ra - ta * a.group) * a.q_head;
      const T* qb = static_cast<const T*>(a.q) + (long long)(sq.tok0 + tok0 + tb) * a.q_token +
                    (long long)(head * a.group + rb - tb * a.group) * a.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        // value index of the k pair (lo: 2 t4, hi: 2 t4 + 8); coded: the order of the codes' pieces
        const int d0 = CODED ? (ks >> 2) * 64 + 16 * t4 + 4 * (ks & 3) : ks * 16 + 2 * t4;
        const int d1 = CODED ? d0 + 2 : d0 + 8;
        qf[ks][0] = *reinterpret_cast<const uint32_t*>(qa + d0);
        qf[ks][1] = *reinterpret_cast<const uint32_t*>(qb + d0);
        qf[ks][2] = *reinterpret_cast<const uint32_t*>(qa + d1);
        qf[ks][3] = *reinterpret_cast<const uint32_t*>(qb + d1);
      }
      if constexpr (CODED && std::is_same_v<T, __nv_bfloat16>) {
        // bf16 rows to f16 by a power of two that brings the largest value to 2^13: exact down to
        // 2^-27 of it, below that off by 2^-38 of it at most
        float ma = 0.f, mb = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = Num<T>::unpack(qf[ks][i]);
            float& m = i & 1 ? mb : ma;
            m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
          ma = fmaxf(ma, __shfl_xor_sync(0xffffffffu, ma, o));
          mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, o));
        }
        // exponent bytes within 16 .. 238: the scale and its inverse are normal numbers
        const uint32_t ea = min(max(__float_as_uint(ma) >> 23, 16u), 238u), eb = min(max(__float_as_uint(mb) >> 23, 16u), 238u);
        const float fa = __uint_as_float((254u + 13u - ea) << 23), fb = __uint_as_float((254u + 13u - eb) << 23);
        rs_a *= __uint_as_float((ea - 13u) << 23);
        rs_b *= __uint_as_float((eb - 13u) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = Num<T>::unpack(qf[ks][i]);
            const float m = i & 1 ? fb : fa;
            qf[ks][i] = Num<__half>::pack(f.x * m, f.y * m);
          }
      }
    }

    // ---- this warp's slices: i = 0, 1, ... at position lo + (u0 * 4 + warp + 4 i) * 16
    const int p0 = lo + u0 * kFewKeys + warp * kSlice;
    const int p_end = min(lo + u1 * kFewKeys, hi);  // keys behind it are another part's, or nobody's
    const int n = p_end > p0 ? (p_end - p0 + kFewKeys - 1) / kFewKeys : 0;
    // (what lies in front of every row's window is not looked up: its page may be given up already)
    const int from = a.window > 0 ? first_pos - a.window + 1 : 0;
    auto page_at = [&](int pos) { return pos + kSlice > from ? page_of(a.b, s, pos) : -1; };
    int next_page = n > 0 ? page_at(p0) : -1;
    auto load = [&](int i) {
      if (i < n) {
        const int pos = p0 + i * kFewKeys;
        const int page = next_page;
        if (i + 1 < n) next_page = page_at(pos + kFewKeys);
        const long long row = page < 0 ? 0 : (((long long)page * a.heads + head) << a.b.page_shift) + (pos & (page_rows - 1));
        const int there = page < 0 ? 0 : sq.len - pos;  // rows of the slice that exist
        const uint32_t st = ring_u + (i % ST) * F::Stage;
        const uint8_t* k = static_cast<const uint8_t*>(a.k) + row * RB;
        const uint8_t* v = static_cast<const uint8_t*>(a.v) + row * RB;
#pragma unroll
        for (int c = 0; c < kSlice * RB / 16; c += 32) {
          const int r = (c + lane) / (RB / 16), ch = (c + lane) % (RB / 16);
          cp_async16_or_zero(st + r * RB + few_swizzle_k<RB, CODED>(r, ch) * 16, k + (c + lane) * 16, r < there);
          cp_async16_or_zero(st + kSlice * RB + r * RB + few_swizzle_v<RB, CODED>(r, ch) * 16, v + (c + lane) * 16,
                             r < there);
        }
        if constexpr (CODED)
          if (lane < 2) {
            if (page >= 0) cp_async16(ring + (i % ST) * F::Stage + 2 * kSlice * RB + lane * 16, (lane ? a.v_exp : a.k_exp) + row);
            else  // no page: zeros, times 2^0
              *reinterpret_cast<uint4*>(ring + (i % ST) * F::Stage + 2 * kSlice * RB + lane * 16) =
                  make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
          }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float o[NB][4];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
    for (int i = 0; i < ST - 1; ++i) load(i);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
      __syncwarp();  // slice i is there for all lanes; all of them are done with slice i - 1
      load(i + ST - 1);
      uint8_t* st = ring + (i % ST) * F::Stage;
      const uint32_t st_u = ring_u + (i % ST) * F::Stage;
      const int pos = p0 + i * kFewKeys;

      // ---- S = q . k: rows g, g + 8; keys 8 j + 2 t4 + {0, 1}
      float sv[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      if constexpr (!CODED) {
        const int mi = lane >> 3, r = (lane & 7) + (mi >> 1) * 8;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t kb[4];
          ldsm_x4(kb, st + r * RB + few_swizzle_k<RB, CODED>(r, 2 * ks + (mi & 1)) * 16);
          mma_16816<M>(sv[0], qf[ks], kb[0], kb[1]);
          mma_16816<M>(sv[1], qf[ks], kb[2], kb[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < DIM / 64; ++h) {
            const int r = 8 * j + g;
            const uint4 w = *reinterpret_cast<const uint4*>(st + r * RB + few_swizzle_k<RB, CODED>(r, 4 * h + t4) * 16);
            const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int x = 0; x < 4; ++x)
              mma_16816<M>(sv[j], qf[4 * h + x], codes_to_h2(c[x] & 0xffffu), codes_to_h2(c[x] >> 16));
          }
      }

      // ---- scores in powers of two; the weights' maximum
      float ev[2][2], back[2][2];  // coded: V's exponents of this thread's keys, 2^-ev
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float fa = rs_a, fb = rs_b;
          ev[j][e] = 0.f;
          back[j][e] = 1.f;
          if constexpr (CODED) {
            const uint8_t* x = st + 2 * kSlice * RB + 8 * j + 2 * t4 + e;
            const float ek = exp_byte(x[0]);
            fa *= ek;
            fb *= ek;
            ev[j][e] = (float)((int)x[16] - 127);
            back[j][e] = inverse_exp_byte(x[16]);
          }
          sv[j][e] = fmaf(sv[j][e], fa, ev[j][e]);
          sv[j][2 + e] = fmaf(sv[j][2 + e], fb, ev[j][e]);
        }
      const bool whole = pos >= all_lo && pos + kSlice <= all_hi;
      uint32_t bad = 0;  // keys whose V is not finite, in a slice that some row does not see whole
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = pos + 8 * j + 2 * t4 + e;
            const bool in = key < p_end;
            if (!in || pos_a < 0 || (a.causal && key > pos_a) || (a.window > 0 && key <= pos_a - a.window)) sv[j][e] = -INFINITY;
            if (!in || pos_b < 0 || (a.causal && key > pos_b) || (a.window > 0 && key <= pos_b - a.window))
              sv[j][2 + e] = -INFINITY;
          }
        // 0 * inf would carry what a row does not see into it: such rows of V leave the product
        bool odd = false;
        uint8_t* vr = st + kSlice * RB + (lane >> 1) * RB + (lane & 1) * (RB / 2);
#pragma unroll 1
        for (int c = 0; c < RB / 2; c += 4) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(vr + c);
          if constexpr (CODED) {
#pragma unroll
            for (int x = 0; x < 4; ++x) odd |= ((w >> (8 * x)) & 0x7fu) == 0x7fu;
          } else {
            const float2 f = Num<M>::unpack(w);
            odd |= !isfinite(f.x) || !isfinite(f.y);
          }
        }
        bad = __ballot_sync(0xffffffffu, odd);
        if (bad) {
          if ((bad >> (lane & ~1)) & 3u)
            for (int c = 0; c < RB / 2; c += 4) *reinterpret_cast<uint32_t*>(vr + c) = 0u;
          __syncwarp();
        }
      }
      float mx_a = fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[1][0], sv[1][1]));
      float mx_b = fmaxf(fmaxf(sv[0][2], sv[0][3]), fmaxf(sv[1][2], sv[1][3]));
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1) {
        mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, x));
        mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, x));
      }
      if (__any_sync(0xffffffffu, mx_a > m_a || mx_b > m_b)) {
        const float na = fmaxf(m_a, mx_a), nb = fmaxf(m_b, mx_b);
        // a row that has seen nothing: its sums are zero, whatever they are multiplied by
        const float ca = m_a == -INFINITY ? 0.f : exp2_approx(m_a - na), cb = m_b == -INFINITY ? 0.f : exp2_approx(m_b - nb);
        m_a = na;
        m_b = nb;
        l_a *= ca;
        l_b *= cb;
#pragma unroll
        for (int x = 0; x < NB; ++x) {
          o[x][0] *= ca;
          o[x][1] *= ca;
          o[x][2] *= cb;
          o[x][3] *= cb;
        }
      }
      const float sub_a = m_a == -INFINITY ? 0.f : m_a - FewTop<M>::value, sub_b = m_b == -INFINITY ? 0.f : m_b - FewTop<M>::value;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sv[j][e] = exp2_approx(sv[j][e] - sub_a);
          sv[j][2 + e] = exp2_approx(sv[j][2 + e] - sub_b);
          l_a = fmaf(sv[j][e], back[j][e], l_a);
          l_b = fmaf(sv[j][2 + e], back[j][e], l_b);
        }
      uint32_t low_keys = 0;  // see kFewLoss
      const uint32_t pf[4] = {Num<M>::pack(sv[0][0], sv[0][1]), Num<M>::pack(sv[0][2], sv[0][3]),
                              Num<M>::pack(sv[1][0], sv[1][1]), Num<M>::pack(sv[1][2], sv[1][3])};
      if constexpr (CODED) {
        if (__any_sync(0xffffffffu, fminf(fminf(fminf(sv[0][0], sv[0][1]), fminf(sv[1][0], sv[1][1])),
                                          fminf(fminf(sv[0][2], sv[0][3]), fminf(sv[1][2], sv[1][3]))) <= kFewLow)) {
          float sum_a = l_a, sum_b = l_b;
#pragma unroll
          for (int x = 1; x <= 2; x <<= 1) {
            sum_a += __shfl_xor_sync(0xffffffffu, sum_a, x);
            sum_b += __shfl_xor_sync(0xffffffffu, sum_b, x);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = 8 * j + 2 * t4 + (e & 1);
              const float off = 0x1p-25f * inverse_exp_byte(st[2 * kSlice * RB + 16 + key]);
              if (sv[j][e] > 0.f && sv[j][e] <= kFewLow && off > kFewLoss * (e < 2 ? sum_a : sum_b)) low_keys |= 1u << key;
            }
          low_keys = __reduce_or_sync(0xffffffffu, low_keys);
        }
      }

      // ---- O += P V
      if constexpr (!CODED) {
        const int mi = lane >> 3, r = (mi & 1) * 8 + (lane & 7);
#pragma unroll
        for (int x = 0; x < NB; x += 2) {
          uint32_t vb[4];
          ldsm_x4_t(vb, st + kSlice * RB + r * RB + few_swizzle_v<RB, CODED>(r, x + (mi >> 1)) * 16);
          mma_16816<M>(o[x], pf, vb[0], vb[1]);
          mma_16816<M>(o[x + 1], pf, vb[2], vb[3]);
        }
      } else {
        // this thread's column g of n tile x is value g * NB + x: NB codes of 4 rows in one piece each
        constexpr int W = NB / 4;  // words of a piece
        uint32_t c[4][W];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 2 * t4 + (j & 1) + (j >> 1) * 8;
          const uint8_t* vr = st + kSlice * RB + r * RB;
          if constexpr (W == 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(vr + few_swizzle_v<RB, CODED>(r, g) * 16);
            c[j][0] = w.x, c[j][1] = w.y, c[j][2] = w.z, c[j][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(vr + few_swizzle_v<RB, CODED>(r, g >> 1) * 16 + (g & 1) * 8);
            c[j][0] = w.x, c[j][1] = w.y;
          }
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint32_t lo01 = __byte_perm(c[0][w], c[1][w], 0x5140), lo23 = __byte_perm(c[0][w], c[1][w], 0x7362);
          const uint32_t hi01 = __byte_perm(c[2][w], c[3][w], 0x5140), hi23 = __byte_perm(c[2][w], c[3][w], 0x7362);
          mma_16816<M>(o[4 * w + 0], pf, codes_to_h2(lo01 & 0xffffu), codes_to_h2(hi01 & 0xffffu));
          mma_16816<M>(o[4 * w + 1], pf, codes_to_h2(lo01 >> 16), codes_to_h2(hi01 >> 16));
          mma_16816<M>(o[4 * w + 2], pf, codes_to_h2(lo23 & 0xffffu), codes_to_h2(hi23 & 0xffffu));
          mma_16816<M>(o[4 * w + 3], pf, codes_to_h2(lo23 >> 16), codes_to_h2(hi23 >> 16));
        }
      }
      // rows of V that are not finite, for the rows that see them, and what the rounding of weights left out: from the
      // cache itself
      if (bad | low_keys) {
#pragma unroll 1
        for (int x = 0; x < kSlice; ++x) {
          const bool is_bad = (bad >> (2 * x)) & 3u;
          if (!is_bad && !((low_keys >> x) & 1u)) continue;
          const int key = pos + x;
          const float w00 = x & 1 ? sv[0][1] : sv[0][0], w01 = x & 1 ? sv[0][3] : sv[0][2];
          const float w10 = x & 1 ? sv[1][1] : sv[1][0], w11 = x & 1 ? sv[1][3] : sv[1][2];
          const int from = (lane & ~3) | ((x & 7) >> 1);
          float wa = __shfl_sync(0xffffffffu, x < 8 ? w00 : w10, from);
          float wb = __shfl_sync(0xffffffffu, x < 8 ? w01 : w11, from);
          const bool in = key < p_end;
          const bool see_a = in && pos_a >= 0 && !(a.causal && key > pos_a) && !(a.window > 0 && key <= pos_a - a.window);
          const bool see_b = in && pos_b >= 0 && !(a.causal && key > pos_b) && !(a.window > 0 && key <= pos_b - a.window);
          if (!is_bad) {
            wa -= __half2float(__float2half_rn(wa));
            wb -= __half2float(__float2half_rn(wb));
          }
          const int page = page_of(a.b, s, key);
          if (page < 0) continue;  // its V is zeros
          const long long row = (((long long)page * a.heads + head) << a.b.page_shift) + (key & (page_rows - 1));
#pragma unroll
          for (int y = 0; y < NB; ++y)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float v;
              if constexpr (CODED) {
                const uint32_t code = static_cast<const uint8_t*>(a.v)[row * DIM + (2 * t4 + e) * NB + y];
                v = Num<__half>::unpack(codes_to_h2(code)).x;
              } else {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.v) + row * DIM + 8 * y + 2 * t4);
                const float2 f = Num<T>::unpack(w);
                v = e ? f.y : f.x;
              }
              if (see_a) o[y][e] = fmaf(wa, v, o[y][e]);
              if (see_b) o[y][2 + e] = fmaf(wb, v, o[y][2 + e]);
            }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      l_a += __shfl_xor_sync(0xffffffffu, l_a, x);
      l_b += __shfl_xor_sync(0xffffffffu, l_b, x);
    }

    // ---- join the warps: [warp][row][DIM + 4] sums, then (m, l)
    __syncthreads();  // every warp is done with its ring
    constexpr int LD = DIM + 4;
    float* jo = reinterpret_cast<float*>(few_smem);
    float* jm = jo + kFewWarps * kFewRows * LD;
    {
      float* oa = jo + (warp * kFewRows + g) * LD;
      float* ob = oa + 8 * LD;
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = CODED ? (2 * t4 + e) * NB + x : 8 * x + 2 * t4 + e;
          oa[d] = o[x][e];
          ob[d] = o[x][2 + e];
        }
      if (t4 == 0) {
        jm[(warp * kFewRows + g) * 2] = m_a;
        jm[(warp * kFewRows + g) * 2 + 1] = l_a;
        jm[(warp * kFewRows + g + 8) * 2] = m_b;
        jm[(warp * kFewRows + g + 8) * 2 + 1] = l_b;
      }
    }
    __syncthreads();
    const bool complete = u0 == 0 && u1 == units;
    const long long slot = 2ll * blockIdx.x + (u0 == 0 ? 1 : 0);
    // complete rows go out row by row, parts in the workspace's layout
    for (int x = tid; x < kFewRows * (DIM / 4); x += kFewThreads) {
      const int r = complete ? x / (DIM / 4) : x % kFewRows, d = (complete ? x % (DIM / 4) : x / kFewRows) * 4;
      if (r >= rows) continue;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) m = fmaxf(m, jm[(w * kFewRows + r) * 2]);
      float l = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float mw = jm[(w * kFewRows + r) * 2];
        const float c = mw == -INFINITY ? 0.f : exp2_approx(mw - m);
        l = fmaf(c, jm[(w * kFewRows + r) * 2 + 1], l);
        const float4 f = *reinterpret_cast<const float4*>(jo + (w * kFewRows + r) * LD + d);
        sum.x = fmaf(c, f.x, sum.x);
        sum.y = fmaf(c, f.y, sum.y);
        sum.z = fmaf(c, f.z, sum.z);
        sum.w = fmaf(c, f.w, sum.w);
      }
      if (complete) {
        const float inv = m == -INFINITY ? 0.f : 1.f / l;
        const int i = token_of(r);
        T* out = static_cast<T*>(a.out) + (long long)(sq.tok0 + tok0 + i) * a.o_token +
                 (long long)(head * a.group + r - i * a.group) * a.o_head + d;
        *reinterpret_cast<uint2*>(out) = make_uint2(Num<T>::pack(sum.x * inv, sum.y * inv), Num<T>::pack(sum.z * inv, sum.w * inv));
      } else {
        *reinterpret_cast<float4*>(a.part_o + ((slot * (DIM / 4) + d / 4) * kFewRows + r) * 4) = sum;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * kFewRows + r) * 2) = make_float2(m, l);
      }
    }
    first += units + a.extra;
    at = first;
    if (at >= end) break;
    if (!paged_next(a, &sq, &s, &head, &b)) break;
    __syncthreads();  // the join's memory becomes rings again
  }
}

// Adds up the parts of a cut tile in their order; one launch for both kernels.  A
// block looks at the boundary between CTAs c - 1 and c of the launch before.  If
// it is the first one inside a tile, the tile's parts are the last one of CTA
// c - 1 and the first ones of CTA c and of all behind it that begin inside.
// A block takes ROWS rows of it (all 16 of the few, 32 of the many), a thread 4 x
// `Q` columns of a row, four parts at a time.  One context that is cut into
// hundreds of parts is what takes long here: the few's parts are shared out
// between four groups of threads, whose sums are joined in their order.
template <typename T, int DIM, int TILE_ROWS, int ROWS, int GROUPS>
__device__ __forceinline__ void paged_merge(const PagedArgs& a, int c, int row_group, float* smem) {
  constexpr int COLS = 256 / ROWS / GROUPS;  // threads of a row (in a group)
  constexpr int Q = DIM / 4 / COLS;          // float4s of a thread
  constexpr int HALF = TILE_ROWS == 256 ? 128 : TILE_ROWS;
  const PagedCut cut = a.cuts[c];
  if (cut.start >= cut.total || cut.start <= cut.first || a.cuts[c - 1].start > cut.first) return;
  const PagedSeq sq = paged_seq(a, cut.seq);
  const int r = row_group * ROWS + threadIdx.x % ROWS, col = threadIdx.x / ROWS % COLS, grp = threadIdx.x / ROWS / COLS;
  // row r: of half r / HALF, there token i0, query head h of the group
  const int in_half = r % HALF, i0 = div_by(in_half, a.group, a.group_mul);
  const int i = r / HALF * a.half_tokens + i0, h = in_half - i0 * a.group;
  const bool live = i0 < a.half_tokens && i < paged_tokens(a, sq, cut.tile);
  int last = c;  // the last CTA with a part
  while (last + 1 < a.ctas && a.cuts[last + 1].start < cut.first + cut.units) ++last;
  const int n = last - c + 2;
  const int p0 = n * grp / GROUPS, p1 = n * (grp + 1) / GROUPS;
  float m = -INFINITY, l = 0.f;
  float4 o[Q];
#pragma unroll
  for (int x = 0; x < Q; ++x) o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    constexpr int U = 4;
    for (int p = p0; p < p1; p += U) {
      float2 ml[U];
      float4 f[U][Q];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ml[u] = make_float2(-INFINITY, 0.f);
        if (p + u < p1) {
          const long long slot = 2ll * (c - 1 + p + u) + (p + u == 0 ? 1 : 0);
          ml[u] = *reinterpret_cast<const float2*>(a.part_ml + (slot * TILE_ROWS + r) * 2);
#pragma unroll
          for (int x = 0; x < Q; ++x)
            f[u][x] = *reinterpret_cast<const float4*>(a.part_o + ((slot * (DIM / 4) + col * Q + x) * TILE_ROWS + r) * 4);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p + u >= p1) continue;
        const float top = fmaxf(m, ml[u].x);
        const float co = m == -INFINITY ? 0.f : exp2_approx(m - top), cp = ml[u].x == -INFINITY ? 0.f : exp2_approx(ml[u].x - top);
        m = top;
        l = l * co + ml[u].y * cp;
#pragma unroll
        for (int x = 0; x < Q; ++x) {
          o[x].x = o[x].x * co + f[u][x].x * cp;
          o[x].y = o[x].y * co + f[u][x].y * cp;
          o[x].z = o[x].z * co + f[u][x].z * cp;
          o[x].w = o[x].w * co + f[u][x].w * cp;
        }
      }
    }
  }
  if constexpr (GROUPS > 1) {
    constexpr int PER = 256 / GROUPS;
    float* mine = smem + threadIdx.x % PER;
    float* ml = smem + (GROUPS - 1) * Q * 4 * PER + threadIdx.x % PER;
    if (grp > 0) {
#pragma unroll
      for (int x = 0; x < Q; ++x) {
        float* at = mine + (grp - 1) * Q * 4 * PER + x * 4 * PER;
        at[0] = o[x].x, at[PER] = o[x].y, at[2 * PER] = o[x].z, at[3 * PER] = o[x].w;
      }
      ml[(grp - 1) * 2 * PER] = m;
      ml[(grp - 1) * 2 * PER + PER] = l;
    }
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) {
      const float mg = ml[(g - 1) * 2 * PER], lg = ml[(g - 1) * 2 * PER + PER];
      const float top = fmaxf(m, mg);
      const float co = m == -INFINITY ? 0.f : exp2_approx(m - top), cp = mg == -INFINITY ? 0.f : exp2_approx(mg - top);
      m = top;
      l = l * co + lg * cp;
#pragma unroll
      for (int x = 0; x < Q; ++x) {
        const float* at = mine + (g - 1) * Q * 4 * PER + x * 4 * PER;
        o[x].x = o[x].x * co + at[0] * cp;
        o[x].y = o[x].y * co + at[PER] * cp;
        o[x].z = o[x].z * co + at[2 * PER] * cp;
        o[x].w = o[x].w * co + at[3 * PER] * cp;
      }
    }
  }
  if (!live) return;
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  T* out = static_cast<T*>(a.out) + (long long)(sq.tok0 + cut.tile * a.tile_tokens + i) * a.o_token +
           (long long)(cut.head * a.group + h) * a.o_head + col * Q * 4;
#pragma unroll
  for (int x = 0; x < Q; ++x)
    *reinterpret_cast<uint2*>(out + x * 4) = make_uint2(Num<T>::pack(o[x].x * inv, o[x].y * inv), Num<T>::pack(o[x].z * inv, o[x].w * inv));
}

constexpr int kManyMergeRows = 32;

// grid: few_ctas - 1 blocks (none: 0), then 8 for each of many_ctas - 1 boundaries.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) k_paged_merge(const PagedArgs few, const PagedArgs many, int few_blocks) {
  __shared__ float smem[3 * 64 * (DIM / 4 / 4 * 4 + 2)];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x;
  if (b < few_blocks)
    paged_merge<T, DIM, kFewRows, kFewRows, 4>(few, b + 1, 0, smem);
  else
    paged_merge<T, DIM, 256, kManyMergeRows, 1>(many, (b - few_blocks) / 8 + 1, (b - few_blocks) % 8, smem);
}

}  // namespace
}  // namespace cn
