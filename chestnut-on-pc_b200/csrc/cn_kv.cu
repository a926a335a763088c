// The paged K/V cache: rows written (8 bits: quantised on the way) and read back.
//
// A row is the dim values of one (token, cache head).  DIM / 16 lanes hold it,
// 16 values (32 bytes, 16 codes) each, two rows a thread at a time and six blocks
// an SM.  HBM bounds these kernels, so bytes in flight count, and few instructions
// a value: 46k tokens x 16 heads x 128 are read back from 8 bits to bf16 in 106 us
// (5.4 TB/s, 82% of the copy rate; with every value's range checked 117 us, with
// four rows a thread and four blocks 120 us, with 8 values a lane 158 us), 18k
// tokens x 8 heads x 128 bf16 are written in 24 us (4.7 TB/s, 71%; 27 us with the
// finite test on every value, or with infinities replaced on every row's path).  8 bits: the row's largest finite |x| comes from
// maxima of pairs and shuffles over its lanes; its exponent e is the
// least one with amax <= 448 * 2^e (448 = 1.75 * 2^8 is e4m3's largest value), so
// x * 2^-e is exact in f32 and the only rounding is the one to e4m3.  A power of
// two costs nothing against amax / 448 as a scale: e4m3's step is relative, only
// its smallest values come a binade nearer to zero, and the attention can apply
// it to exponents.  The places of a block's tokens are worked out once, in shared
// memory: the block counts the sequences that begin before its first token (one
// pass over cu_tokens, no chain of dependent loads), its tokens walk on from there.
#include <type_traits>

#include "cn_heads.cuh"

namespace cn {
namespace {

constexpr int kKvThreads = 256;
constexpr int kKvMaxTokens = 32;  // tokens of one block

struct KvArgs {
  BatchArgs b;
  void *ck, *cv;  // cache
  uint8_t *ke, *ve;
  void *hk, *hv;  // rows [tokens][heads][dim]
  long long k_token, k_head, v_token, v_head;
  int heads, per_block;
};

// Cache row (of head 0) of token t: page * heads * page rows + row, or -1: no such
// place (its row reads as zeros), or -2: t belongs to no sequence.  s: a sequence
// that begins at t or before (or -1).
__device__ __forceinline__ long long place_of(const KvArgs& a, long long t, int s) {
  if (s < 0) return -2;
  while (s < a.b.n_seqs && a.b.cu[s + 1] <= t) ++s;
  if (s >= a.b.n_seqs) return -2;
  const int pos = a.b.lengths[s] - a.b.cu[s + 1] + (int)t;
  if (pos < 0) return -1;
  const int page = page_of(a.b, s, pos);
  if (page < 0) return -1;
  return (((long long)page * a.heads) << a.b.page_shift) + (pos & ((1 << a.b.page_shift) - 1));
}

// The largest of v over groups of N neighbouring lanes.
template <int N>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Larger of pairs of 16-bit values (a NaN loses against a number).
template <typename T>
__device__ __forceinline__ uint32_t max_pairs(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t max_pairs<__half>(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <>
__device__ __forceinline__ uint32_t max_pairs<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// 16 values of a row to codes; every lane of the row gets the row's exponent byte.
template <typename T, int LANES>
__device__ __forceinline__ uint4 quantise16(const uint4 (&raw)[2], uint32_t* byte) {
  uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max_pairs<T>(top, w[i] & 0x7fff7fffu);
  const float2 two = Num<T>::unpack(top);
  float amax = group_max<LANES>(fmaxf(two.x, two.y));
  // (the warp decides together: group_max below is for all lanes)
  const bool infinite = __any_sync(0xffffffffu, isinf(amax));
  if (infinite) {  // the largest finite one then; infinities become NaN (not 448), the other values stay as they are
    constexpr uint32_t quiet = std::is_same_v<T, __half> ? 0x0200u : 0x0040u;
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = Num<T>::unpack(w[i]);
      amax = fmaxf(amax, fmaxf(isfinite(f.x) ? fabsf(f.x) : 0.f, isfinite(f.y) ? fabsf(f.y) : 0.f));
      w[i] |= (isinf(f.x) ? quiet : 0u) | (isinf(f.y) ? quiet << 16 : 0u);
    }
    amax = group_max<LANES>(amax);
  }
  // amax = 1.m * 2^k; 448 * 2^e >= amax  <=>  e >= k - 8, or k - 7 where 1.m > 1.75
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = amax > 0.f ? min(max(e, -48), 48) : 0;
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  *byte = (uint32_t)(e + 127);
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = Num<T>::unpack(w[i]);
    c[i] = floats_to_codes(f.x * inv, f.y * inv);
  }
  return make_uint4(c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | c[7] << 16);
}

// 8 codes to 8 values of T, times 2^(byte - 127).
template <typename T>
__device__ __forceinline__ uint4 expand8(const uint2& codes, uint32_t byte) {
  const uint32_t c[4] = {codes.x & 0xffffu, codes.x >> 16, codes.y & 0xffffu, codes.y >> 16};
  uint32_t w[4];
  if constexpr (std::is_same_v<T, __half>) {
    // 2^-24 .. 2^7: the power is an f16 number and no product is beyond f16 (448 * 2^7 < 65504); it is
    // rounded once, as from f32
    if (byte >= 103u && byte <= 134u) {
      const uint32_t p = byte >= 113u ? (byte - 112u) << 10 : 1u << (byte - 103u);
#pragma unroll
      for (int i = 0; i < 4; ++i) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(w[i]) : "r"(codes_to_h2(c[i])), "r"(p | p << 16));
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  const float scale = exp_byte(byte);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Num<__half>::unpack(codes_to_h2(c[i]));
    float a = f.x * scale, b = f.y * scale;
    if constexpr (std::is_same_v<T, __half>) {
      // finite values beyond f16 become its largest (fminf and fmaxf would make one of a NaN; bf16 holds all that
      // cn_kv_write's exponents can make)
      a = fabsf(a) > 65504.f ? copysignf(65504.f, a) : a;
      b = fabsf(b) > 65504.f ? copysignf(65504.f, b) : b;
    }
    w[i] = Num<T>::pack(a, b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// T: type of the rows.  CODED: 8-bit cache (else of type T too).  READ: cache -> rows.
template <typename T, int DIM, bool CODED, bool READ>
__global__ void __launch_bounds__(kKvThreads, 6) k_kv(const KvArgs a) {
  constexpr int LANES = DIM / 16;  // lanes of a row
  constexpr int RPB = kKvThreads / LANES;  // rows that the block takes at a time
  constexpr int U = 2;
  __shared__ long long place[kKvMaxTokens];
  __shared__ int began[kKvThreads / 32];
  pdl_trigger();
  pdl_wait();
  const long long t0 = (long long)blockIdx.x * a.per_block;
  const int nt = (int)min((long long)a.per_block, a.b.tokens - t0);
  int count = 0;  // sequences that begin at t0 or before (cu_tokens ascends)
  for (int i = threadIdx.x; i < a.b.n_seqs; i += kKvThreads) count += a.b.cu[i] <= t0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
  if ((threadIdx.x & 31) == 0) began[threadIdx.x >> 5] = count;
  __syncthreads();
  if (threadIdx.x < nt) {
    int s = -1;
#pragma unroll
    for (int w = 0; w < kKvThreads / 32; ++w) s += began[w];
    const long long t = t0 + threadIdx.x;
    // rows before the first sequence: one may begin behind t0
    if (s < 0 && a.b.cu[0] <= t) s = 0;
    place[threadIdx.x] = place_of(a, t, s);
  }
  __syncthreads();
  const int lane = threadIdx.x % LANES;
  const int rows = nt * a.heads * 2;  // [token][k or v][head]
  const uint32_t per_token = 2 * a.heads;
  for (int base = 0; base < rows; base += RPB * U) {
    uint4 x[U][2], c[U];
    uint32_t byte[U];
    long long at[U];
    T* row[U];
    bool v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = base + u * RPB + (int)threadIdx.x / LANES;
      at[u] = -2;
      byte[u] = 127;
      x[u][0] = x[u][1] = c[u] = make_uint4(0, 0, 0, 0);
      if (j < rows) {
        const uint32_t t = (uint32_t)j / per_token, r = (uint32_t)j - t * per_token;
        v[u] = r >= (uint32_t)a.heads;
        const int h = v[u] ? r - a.heads : r;
        at[u] = place[t];
        row[u] = static_cast<T*>(v[u] ? a.hv : a.hk) + (t0 + t) * (v[u] ? a.v_token : a.k_token) +
                 h * (v[u] ? a.v_head : a.k_head) + lane * 16;
        if (at[u] >= 0) {
          at[u] += (long long)h << a.b.page_shift;
          if constexpr (!READ) {
            x[u][0] = reinterpret_cast<const uint4*>(row[u])[0];
            x[u][1] = reinterpret_cast<const uint4*>(row[u])[1];
          } else if constexpr (CODED) {
            c[u] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(v[u] ? a.cv : a.ck) + at[u] * DIM + lane * 16);
            byte[u] = (v[u] ? a.ve : a.ke)[at[u]];
          } else {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(v[u] ? a.cv : a.ck) + at[u] * DIM + lane * 16);
            x[u][0] = p[0];
            x[u][1] = p[1];
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (READ) {
        if constexpr (CODED) {
          x[u][0] = expand8<T>(make_uint2(c[u].x, c[u].y), byte[u]);
          x[u][1] = expand8<T>(make_uint2(c[u].z, c[u].w), byte[u]);
        }
        if (at[u] >= -1) {
          reinterpret_cast<uint4*>(row[u])[0] = x[u][0];
          reinterpret_cast<uint4*>(row[u])[1] = x[u][1];
        }
      } else if constexpr (CODED) {
        c[u] = quantise16<T, LANES>(x[u], &byte[u]);  // all lanes: it shuffles
        if (at[u] >= 0) {
          *reinterpret_cast<uint4*>(static_cast<uint8_t*>(v[u] ? a.cv : a.ck) + at[u] * DIM + lane * 16) = c[u];
          if (lane == 0) (v[u] ? a.ve : a.ke)[at[u]] = (uint8_t)byte[u];
        }
      } else if (at[u] >= 0) {
        uint4* p = reinterpret_cast<uint4*>(static_cast<T*>(v[u] ? a.cv : a.ck) + at[u] * DIM + lane * 16);
        p[0] = x[u][0];
        p[1] = x[u][1];
      }
    }
  }
}

template <typename T, bool READ>
cudaError_t kv_launch(const KvArgs& a, int dim, bool coded, cudaStream_t s) {
  const dim3 grid((unsigned)((a.b.tokens + a.per_block - 1) / a.per_block)), block(kKvThreads);
  if (dim == 128)
    return coded ? launch_ex(k_kv<T, 128, true, READ>, grid, block, 0, s, true, a)
                 : launch_ex(k_kv<T, 128, false, READ>, grid, block, 0, s, true, a);
  return coded ? launch_ex(k_kv<T, 64, true, READ>, grid, block, 0, s, true, a)
               : launch_ex(k_kv<T, 64, false, READ>, grid, block, 0, s, true, a);
}

int kv_call(const char* who, bool read, const cn_kv_cache* cache, const cn_kv_batch* batch, const cn_heads* k,
            const cn_heads* v, long long tokens, void* stream) {
  int r;
  if ((r = check_cache(who, cache)) || (r = check_batch(who, batch, cache)) || (r = check_heads(who, "k", k, tokens, read)) ||
      (r = check_heads(who, "v", v, tokens, read)))
    return r;
  if (k->dtype != v->dtype || k->dtype == CN_F32 || (cache->dtype != CN_E4M3 && cache->dtype != k->dtype)) {
    set_last_error("%s: k (dtype %d) and v (%d) are alike, f16 or bf16, and a 16-bit cache (%d) has their dtype", who,
                   k->dtype, v->dtype, cache->dtype);
    return CN_ERR_ARG;
  }
  if (k->heads != cache->heads || v->heads != cache->heads || k->dim != cache->dim || v->dim != cache->dim) {
    set_last_error("%s: k (%d x %d), v (%d x %d) and the cache (%d x %d) differ in heads or dim", who, k->heads, k->dim,
                   v->heads, v->dim, cache->heads, cache->dim);
    return CN_ERR_ARG;
  }
  if (tokens < 0 || tokens > INT32_MAX) {
    set_last_error("%s: %lld tokens", who, tokens);
    return CN_ERR_ARG;
  }
  if (tokens == 0 || batch->n_seqs == 0) return 0;
  DataDevice dev;
  const void* all[] = {cache->k, cache->v, k->data, v->data, batch->cu_tokens, batch->lengths};
  for (const void* p : all)
    if ((r = dev.use(who, p))) return r;
  if (batch->table_width && (r = dev.use(who, batch->table))) return r;
  if (cache->dtype == CN_E4M3 && ((r = dev.use(who, cache->k_exp)) || (r = dev.use(who, cache->v_exp)))) return r;
  KvArgs a;
  a.b = batch_args(cache, batch, tokens);
  a.ck = cache->k;
  a.cv = cache->v;
  a.ke = cache->k_exp;
  a.ve = cache->v_exp;
  a.hk = k->data;
  a.hv = v->data;
  a.k_token = k->token_stride;
  a.k_head = k->head_stride;
  a.v_token = v->token_stride;
  a.v_head = v->head_stride;
  a.heads = cache->heads;
  // Enough blocks for all SMs several times over, each with enough rows to be worth its search.
  a.per_block = (int)min((long long)kKvMaxTokens, max(1ll, tokens / (148 * 16)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool coded = cache->dtype == CN_E4M3;
  cudaError_t e;
  if (k->dtype == CN_F16)
    e = read ? kv_launch<__half, true>(a, cache->dim, coded, s) : kv_launch<__half, false>(a, cache->dim, coded, s);
  else
    e = read ? kv_launch<__nv_bfloat16, true>(a, cache->dim, coded, s)
             : kv_launch<__nv_bfloat16, false>(a, cache->dim, coded, s);
  return launch_status(who, e);
}

}  // namespace
}  // namespace cn

extern "C" int cn_kv_write(const cn_kv_cache* cache, const cn_kv_batch* batch, const cn_heads* k, const cn_heads* v,
                           long long tokens, void* stream) {
  return cn::kv_call("cn_kv_write", false, cache, batch, k, v, tokens, stream);
}

extern "C" int cn_kv_read(const cn_kv_cache* cache, const cn_kv_batch* batch, const cn_heads* k_out,
                          const cn_heads* v_out, long long tokens, void* stream) {
  return cn::kv_call("cn_kv_read", true, cache, batch, k_out, v_out, tokens, stream);
}
