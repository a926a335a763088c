// Rotary positions: out = x with the first rot values of every head turned by
// the token's angle, one read and one write of each value.
//
// Pair i of a token at position p turns by p * f_i radians.  Far positions make
// angles of 10^6 radians and more, whose f32 ulp is a visible angle, so the
// product is taken in f64 as a number of turns, reduced to [-1/2, 1/2] there,
// and only then goes to f32 (sincospif of twice the turns).  A block does this
// once per (token, pair) for all heads of its tokens: cos and sin (times
// `magnitude`) lie in shared memory, and each thread then turns vectors of up
// to 16 bytes: 8 neighbours (4 pairs) of the interleaved layout, or the same V
// places of both halves of the half layout, V the largest power of two that
// divides rot / 2.  HBM bounds it, and warps rather than loads a thread keep it
// busy: eight blocks an SM with one vector (pair) a thread in flight move 16384 x
// 40 heads x 128 bf16 in 65 us (5.2 TB/s); four vectors a thread, at 62 registers
// and four blocks, take 95 us.  An odd rot / 2 leaves vectors of one value, for the
// copied places too: 54 of 128 values turned take 223 us.
#include "cn_heads.cuh"

namespace cn {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxTokens = 4;  // tokens of one block

struct RopeArgs {
  const void* x;
  void* out;
  long long x_token, x_head, o_token, o_head;  // strides in elements
  long long tokens;
  const long long* pos;
  const double* freq;
  int heads, dim, rot, per_block;
  int copy;  // the values behind rot are copied (out is not x)
  float magnitude;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V: elements of a vector.  PAIRED: interleaved pairs (V even).
template <typename T, int V, bool PAIRED>
__global__ void __launch_bounds__(kRopeThreads, 8) k_rope(const RopeArgs a) {
  __shared__ float2 turn[kRopeMaxTokens][128];  // (cos, sin) of pair i
  pdl_trigger();
  pdl_wait();
  const long long t0 = (long long)blockIdx.x * a.per_block;
  const int nt = (int)min((long long)a.per_block, a.tokens - t0);
  const int half = a.rot >> 1;
  for (int j = threadIdx.x; j < nt * half; j += kRopeThreads) {
    const int t = j / half, i = j - t * half;
    const double turns = (double)a.pos[t0 + t] * a.freq[i] * 0.15915494309189533577;
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    turn[t][i] = make_float2(c * a.magnitude, s * a.magnitude);
  }
  __syncthreads();
  const int turned = PAIRED ? (a.rot + V - 1) / V : half / V;         // vectors of a head with a turned pair
  const int plain = !a.copy ? 0 : a.dim / V - (PAIRED ? turned : 2 * turned);  // vectors behind them
  const int per_head = turned + plain;
  const int per_token = per_head * a.heads;
  using P = Pack<T, V>;
  for (uint32_t j = threadIdx.x; j < (uint32_t)(nt * per_token); j += kRopeThreads) {
    const uint32_t t = j / (uint32_t)per_token, r = j - t * per_token;
    const uint32_t h = r / (uint32_t)per_head, v = r - h * per_head;
    const T* x = static_cast<const T*>(a.x) + (t0 + t) * a.x_token + h * a.x_head;
    T* o = static_cast<T*>(a.out) + (t0 + t) * a.o_token + h * a.o_head;
    const bool turn_it = v < (uint32_t)turned;
    const int at = (PAIRED || turn_it ? v : v + turned) * V;
    P p = *reinterpret_cast<const P*>(x + at);
    if (turn_it) {
      if constexpr (PAIRED) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const int i = (at + e) >> 1;
          if (i < half) {
            const float2 cs = turn[t][i];
            const float p0 = to_f32(p.v[e]), p1 = to_f32(p.v[e + 1]);
            p.v[e] = from_f32<T>(p0 * cs.x - p1 * cs.y);
            p.v[e + 1] = from_f32<T>(p1 * cs.x + p0 * cs.y);
          }
        }
      } else {
        P q = *reinterpret_cast<const P*>(x + half + at);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 cs = turn[t][at + e];
          const float p0 = to_f32(p.v[e]), p1 = to_f32(q.v[e]);
          p.v[e] = from_f32<T>(p0 * cs.x - p1 * cs.y);
          q.v[e] = from_f32<T>(p1 * cs.x + p0 * cs.y);
        }
        *reinterpret_cast<P*>(o + half + at) = q;
      }
    }
    *reinterpret_cast<P*>(o + at) = p;
  }
}

template <typename T>
cudaError_t rope_launch(const RopeArgs& a, bool paired, cudaStream_t s) {
  constexpr int W = 16 / sizeof(T);  // elements of 16 bytes
  const dim3 grid((unsigned)((a.tokens + a.per_block - 1) / a.per_block)), block(kRopeThreads);
  if (paired) return launch_ex(k_rope<T, W, true>, grid, block, 0, s, true, a);
  const int half = a.rot / 2;
  if (half % W == 0) return launch_ex(k_rope<T, W, false>, grid, block, 0, s, true, a);
  if (half % 4 == 0) return launch_ex(k_rope<T, 4, false>, grid, block, 0, s, true, a);
  if (half % 2 == 0) return launch_ex(k_rope<T, 2, false>, grid, block, 0, s, true, a);
  return launch_ex(k_rope<T, 1, false>, grid, block, 0, s, true, a);
}

}  // namespace
}  // namespace cn

extern "C" int cn_rope(const cn_heads* x, const cn_heads* out, long long tokens, const long long* positions,
                       const double* inv_freq, int rot_dim, int interleaved, float magnitude, void* stream) {
  using namespace cn;
  const char* who = "cn_rope";
  int r;
  if ((r = check_heads(who, "x", x, tokens, false)) || (r = check_heads(who, "out", out, tokens, true))) return r;
  if (x->dtype != out->dtype || x->heads != out->heads || x->dim != out->dim) {
    set_last_error("%s: x and out differ in dtype, heads or dim", who);
    return CN_ERR_ARG;
  }
  if (rot_dim < 2 || rot_dim % 2 || rot_dim > x->dim) {
    set_last_error("%s: rot_dim %d of heads of %d values (even, 2 to dim)", who, rot_dim, x->dim);
    return CN_ERR_ARG;
  }
  if (x->data == out->data && ((tokens > 1 && x->token_stride != out->token_stride) ||
                               (x->heads > 1 && x->head_stride != out->head_stride))) {
    set_last_error("%s: out starts where x does but has other strides", who);
    return CN_ERR_ARG;
  }
  if (tokens < 0 || tokens > INT32_MAX || (!positions && tokens > 0) || !inv_freq || reinterpret_cast<uintptr_t>(positions) % 8 ||
      reinterpret_cast<uintptr_t>(inv_freq) % 8) {
    set_last_error("%s: tokens out of range, or positions or inv_freq missing or not 8-byte aligned", who);
    return CN_ERR_ARG;
  }
  if (tokens == 0) return 0;
  DataDevice dev;
  if ((r = dev.use(who, x->data)) || (r = dev.use(who, out->data)) || (r = dev.use(who, positions)) ||
      (r = dev.use(who, inv_freq)))
    return r;
  RopeArgs a;
  a.x = x->data;
  a.out = out->data;
  a.x_token = x->token_stride;
  a.x_head = x->head_stride;
  a.o_token = out->token_stride;
  a.o_head = out->head_stride;
  a.tokens = tokens;
  a.pos = positions;
  a.freq = inv_freq;
  a.heads = x->heads;
  a.dim = x->dim;
  a.rot = rot_dim;
  a.per_block = tokens >= 4096 ? kRopeMaxTokens : 1;
  a.copy = x->data != out->data;
  a.magnitude = magnitude;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool paired = interleaved != 0;
  return launch_status(who, x->dtype == CN_F16    ? rope_launch<__half>(a, paired, s)
                            : x->dtype == CN_BF16 ? rope_launch<__nv_bfloat16>(a, paired, s)
                                                  : rope_launch<float>(a, paired, s));
}
