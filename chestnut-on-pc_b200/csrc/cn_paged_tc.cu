// Attention over the paged cache for sequences of many query rows: tcgen05.
//
// A tile is 256 query rows (new tokens x the heads of a group) of one sequence
// and cache head, as two halves of 128 that share every block of 128 keys.
// S = Q K^T and O += P V both run on tcgen05.mma with M = 128; S, P and O live in
// tensor memory (columns 0..127 and 128..255: S of the halves, P written over it
// as 16-bit pairs; 256.. and 384..: O), so the weights never pass through shared
// memory: P is the A operand of the second product from tensor memory.
// A block's S comes as two products of 64 keys.  While a half's threads are in
// the softmax of one, the tensor core adds the other one's P V and computes its
// next S; with one S of 128 keys a half, each block paid softmax, hand-over and
// both products one after the other.  A tile whose tokens fill one half at most
// gives its odd blocks of keys to the other half (`dual`), which joins its sums
// in the end.
// 8192 tokens, causal, 32 heads over 8, 128 bf16: 585 us, 940 TFLOP/s, 56% of the
// cuBLAS burst rate (at 950 W, near the power cap; 1040 TFLOP/s in short runs).
// The tensor pipe is 48% busy.  Per 128 keys of 256 rows an SM spends ~4200
// clocks; the products need 2560 of them (S with N = 64 is bound by shared
// memory), the exponentials 2048, and taking either away shortens a block by a
// tenth: what is left is the chain scores - maximum - exponentials - P - product.
// 16 x 64 tokens over 640 to 4032, 16 heads x 128 f16: 102 us, 3.2 TB/s.
//   warpgroups 0, 1: softmax of a half, one thread a row, a row's 64 scores in
//                    registers: no shuffles
//   warpgroup 2:     loads.  A 16-bit cache comes by TMA, a box a page, in the
//                    128-byte swizzle that the tensor core reads; of an 8-bit one
//                    the threads hold the codes of the next K and V block in
//                    registers and store them as f16 (exact) in that swizzle
//   warp 15:         works out the parts ahead of the others (ring of two)
//   warps 12, 13:    issue the products of a half each, so that one half's wait
//                    never holds up the other
// The running maximum is raised only when a block's exceeds it by 2^8 (the sums
// stay exact, the weights are just up to 256): O is rescaled in tensor memory by
// the row's own thread then, which is rare after the first blocks.
// Keys and rows at the edge (tail, causal diagonal, window) are masked in
// registers.  V rows there that do not exist are zeroed in shared memory, and
// rows with NaN or infinities, which 0 * inf would carry into rows that do not
// see them, leave the product and are added by the threads whose row sees them.
// An 8-bit cache's powers of two: K's goes to its scores (2^ek * scale of each key).
// V's goes into its f16 rows, relative to the largest that the part has met: e4m3
// codes times 2^-15 .. 2^7 are exact, so the weights are those of the softmax alone
// and no row's size takes bits of another's.  (With V's power in the weights' exponent
// a row 2^26 larger than the others took them all.)  Rows outside those 22 powers
// leave the product like rows that are not finite.
#include <type_traits>
#include "cn_paged.cuh"

namespace cn {

namespace {

constexpr int kManyRows = 256;
constexpr int kManyKeys = 128;
constexpr int kManyThreads = 512;
// The maximum may be exceeded by 2^Lazy before it is raised; weights are relative to it times 2^-Top.
// f16 weights are 2^15 at most then, normal numbers down to 2^-23 of the maximum's and numbers down to
// 2^-33; bf16 ones have f32's exponents.
template <typename M>
struct ManyTop {
  static constexpr bool F16 = std::is_same_v<M, __half>;
  static constexpr float Lazy = F16 ? 6.f : 8.f, Top = F16 ? 9.f : 0.f;
};
// 8-bit cache: a row of V goes to f16 times 2^(7 - d), d how many powers of two its own is below the
// largest so far.  That is exact down to d = 22 (codes x 2^-15); rows below do not go through the tensor
// core, nor do those above kByteTop: the largest so far counts within what cn_kv_write makes.
constexpr int kSpread = 22, kByteLow = 79, kByteTop = 175;

// Registers of the warpgroups (softmax, loads, products): their sum is 4 x 128, what the block is
// launched with.  setmaxnreg.dec to more than 128 would be an illegal instruction.  Over an 8-bit
// cache the loads hold two blocks' codes: with 96 registers they spilled (dim 128, chunks of up to
// 701 tokens: a third more time).
template <bool CODED>
struct ManyRegs {
  static constexpr int Softmax = CODED ? 160 : 192;
  static constexpr int Load = CODED ? 128 : 64;
  static constexpr int Mma = 64;
  static_assert(2 * Softmax + Load + Mma == 512 && Softmax >= 128 && Load <= 128 && Mma <= 128, "register split");
};

template <int DIM>
struct Many {
  static constexpr int Sub = 128 * 128;            // 128 rows x 64 values of 16 bits
  static constexpr int Tile = DIM / 64 * Sub;      // 128 rows
  static constexpr int QBytes = 2 * Tile;
  static constexpr int Stages = DIM == 128 ? 2 : 4;  // of K, and of V; even: see ManyPart::dual
  static constexpr size_t Smem = 1024 + QBytes + 2 * Stages * Tile;
};

// A wait knows the parity of a phase, so it is right only where the phase before the awaited one has
// ended already (else it passes at once) and where the one behind it cannot end before the wait is
// over.  The second holds everywhere because a stage is given back by its waiting threads alone.  The
// first:
//   within a part, and from a part that is not dual to any other: an issuing thread waits for the K, V
//     and fix of every block in turn, and a stage's phase ends before its block is used again;
//   within a dual part, and from one to the next: a half's blocks have stages of its own (n % 2 = half);
//   from a dual part to one that is not: the other half's stages come up, whose last phases this half
//     has not waited for.  qempty tells of them: a half gives it in a dual part when it has its last
//     scores (its K was there) and has seen its last V (and fix), and every part begins with a wait for
//     qfull, which follows both halves' qempty.  (Given with the last scores, as in the other parts, it
//     would leave the other half's last V on its way: this half's wait for the stage's next V would pass
//     at once, and the product read what lies there.)
//   softmax warps: they wait for a block's scores before its V and fix, and the scores were issued after
//     all that their issuing thread had waited for; the halves of a dual part meet at `joined`, behind
//     their last products.
struct ManyBars {
  uint64_t kfull[4], kempty[4], vfull[4], vempty[4], vfix[4];  // stages
  uint64_t sfull[2][2], pfull[2][2];                           // [half][64 keys of a block]
  uint64_t odone[2][2];                                        // its product with V is added to O
  uint64_t asked[4];                                           // stages: V of an edge block is on its way
  uint64_t qfull, qempty;
  uint64_t told[2], heard[2];                                  // parts: worked out, read by all
  uint64_t joined;                                             // both halves' sums of a dual part are out
  uint64_t drain[2];
  uint32_t tmem;
};

// The part of a tile that a CTA works on.
struct ManyPart {
  int lo;          // position of the tile's unit 0
  int j0, j1;      // blocks of 128 keys, from lo
  int a[2], b[2];  // those that the halves take part in
  int hi;          // keys behind it no row sees
  int i0, i1;      // blocks that every row sees whole; the others are at the edge
  int tok0, toks;  // tokens of the sequence
  int seq, head, seq_tok0, past, len;
  int whole, first_part;  // the whole tile; its beginning
  int dual;               // the tile's tokens fill one half at most: the other one takes every second block of keys
  int live;               // 0: no further part
};

__device__ __forceinline__ ManyPart many_part(const PagedArgs& a, const PagedSeq& q, int s, int head, int tile, int u0,
                                              int u1, int units) {
  ManyPart p;
  p.seq = s;
  p.head = head;
  p.seq_tok0 = q.tok0;
  p.past = q.past;
  p.len = q.len;
  p.whole = u0 == 0 && u1 == units;
  p.first_part = u0 == 0;
  p.live = 1;
  p.tok0 = tile * a.tile_tokens;
  p.toks = paged_tokens(a, q, tile);
  paged_range<kManyKeys>(a, q, p.tok0, p.toks, &p.lo, &p.hi);
  p.j0 = u0;
  p.j1 = min(u1, max((p.hi - p.lo + kManyKeys - 1) / kManyKeys, u0));
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    p.a[t] = p.b[t] = p.j1;
    const int n = min(p.toks - t * a.half_tokens, a.half_tokens);
    if (n > 0 && p.j1 > p.j0) {
      int lo, hi;
      paged_range<kManyKeys>(a, q, p.tok0 + t * a.half_tokens, n, &lo, &hi);
      if (hi > lo) {
        p.a[t] = max(p.j0, (lo - p.lo) / kManyKeys);
        p.b[t] = min(p.j1, (hi - p.lo + kManyKeys - 1) / kManyKeys);
        if (p.b[t] < p.a[t]) p.a[t] = p.b[t] = p.j1;
      }
    }
  }
  p.dual = p.toks <= a.half_tokens && p.b[0] - p.a[0] >= 2;
  if (p.dual) {
    p.a[1] = p.a[0];
    p.b[1] = p.b[0];
  }
  const int first_pos = q.past + p.tok0, last_pos = first_pos + p.toks - 1;
  const int all_hi = first_pos < 0 ? 0 : a.causal ? min(q.len, first_pos + 1) : q.len;
  const int all_lo = a.window > 0 ? max(last_pos - a.window + 1, 0) : 0;
  p.i0 = max(all_lo - p.lo + kManyKeys - 1, 0) / kManyKeys;
  p.i1 = max(all_hi - p.lo, 0) / kManyKeys;
  return p;
}

// Whether some row of the tile does not see all of block j.
__device__ __forceinline__ bool many_edge(const ManyPart& p, int j) {
  return j < p.i0 || j >= p.i1;
}

// Bounded wait on the critical path: the limit goes by the SM's clock (%globaltimer
// takes about as long to read as a whole block's products).
constexpr long long kManyWaitClocks = 4000000000ll;  // ~2 s
__device__ __forceinline__ bool many_wait1(uint64_t* bar, uint32_t parity, int code) {
  if (__builtin_expect(mbar_try_wait(bar, parity), 1)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity))
    if (clock64() - t0 > kManyWaitClocks) {
      set_dev_error(code);
      return false;
    }
  return true;
}
// A warp's wait: the same answer for all its lanes.
__device__ __forceinline__ bool many_wait(uint64_t* bar, uint32_t parity, int code) {
  return __all_sync(0xffffffffu, many_wait1(bar, parity, code));
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
      "%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// Waits for this warp's tensor-memory loads.  r passes through it, so that nothing of r is read before.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
// Pairs of f32: one instruction for two values.
__device__ __forceinline__ uint64_t pair2(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ uint64_t pair2(float lo, float hi) { return pair2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float2 unpair2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {  // waits too
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(r) : "r"(taddr) : "memory");
  return r;
}

// The products of the issuing thread.  A shared-memory descriptor's high word is
// the same for all operands here; its low word counts 16-byte steps, so the k
// steps are additions to it (umma_desc_sw128 anew for each costs more than the
// product itself takes).
constexpr uint32_t kDescHi = (1024u >> 4) | 1u << 14 | 2u << 29;  // 8-row groups 1024 B apart, version 1, 128-byte swizzle
__device__ __forceinline__ uint32_t desc_lo(const void* p, uint32_t lbo_bytes) {
  return (smem_u32(p) >> 4) | (lbo_bytes >> 4) << 16;
}
// 64 bytes of a thread's own row; in whole 32-byte sectors where the row allows.
__device__ __forceinline__ void st_row64(void* p, const uint32_t* w, bool wide) {
  if (wide) {
#pragma unroll
    for (int i = 0; i < 16; i += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<uint8_t*>(p) + i * 4),
                   "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]),
                   "r"(w[i + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p) + i * 4) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
}

// D[tmem] (+)= A[smem] * B[smem]^T, 16-bit operands.
template <bool ADD>
__device__ __forceinline__ void tc_mma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %4};\n\t"
      "setp.ne.u32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(kDescHi), "n"(ADD ? 1 : 0)
      : "memory");
}
// D[tmem] += A[tmem] * B[smem].
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "setp.eq.u32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "n"(kDescHi)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

template <typename M>
__device__ __forceinline__ constexpr uint32_t many_idesc(int n, bool b_mn_major) {
  constexpr uint32_t f = std::is_same_v<M, __nv_bfloat16> ? 1u : 0u;  // operand format, both alike
  return umma_idesc_f16(n, b_mn_major) | (f << 7) | (f << 10);
}

template <typename M>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  constexpr uint32_t e = std::is_same_v<M, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

// Codes of a block of keys, 16 a piece, piece lt + 128 i of the loading thread lt, to f16 rows in the
// 128-byte swizzle.  V's rows are multiplied by a power of two or left out (see kSpread), by their
// exponent bytes (a lane of the warp has those of four keys) and the largest of those.
template <int DIM, bool IS_V, int PT>
__device__ __forceinline__ void many_put(const uint4 (&c)[PT], uint8_t* to, int lt, uint32_t bytes, int top) {
  constexpr int PR = DIM / 16;  // pieces of a row
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int row = (lt + 128 * i) / PR, piece = (lt + 128 * i) % PR;
    uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w}, f = 0;
    if constexpr (IS_V) {
      const int byte = (__shfl_sync(0xffffffffu, bytes, row >> 2) >> (8 * (row & 3))) & 0xff;
      const int k = min(max(byte - top, -kSpread), 0) + 7;
      f = (k > -15 ? (uint32_t)(k + 15) << 10 : 0x0200u) * 0x10001u;  // 2^k twice
      if (byte < top - kSpread || byte > top) w[0] = w[1] = w[2] = w[3] = 0;
    }
    uint32_t h[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      h[2 * e] = codes_to_h2(w[e] & 0xffffu);
      h[2 * e + 1] = codes_to_h2(w[e] >> 16);
    }
    if constexpr (IS_V) {
#pragma unroll
      for (int e = 0; e < 8; ++e) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(h[e]) : "r"(f));
    }
    uint8_t* base = to + (piece >> 2) * (128 * 128) + row * 128;
    const int ch = (piece & 3) * 2;
    *reinterpret_cast<uint4*>(base + ((ch ^ (row & 7)) * 16)) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(base + (((ch + 1) ^ (row & 7)) * 16)) = make_uint4(h[4], h[5], h[6], h[7]);
  }
}

// T: q and out (and a 16-bit cache).
template <typename T, int DIM, bool CODED>
__global__ void __launch_bounds__(kManyThreads, 1)
    k_paged_many(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const PagedArgs a) {
  using L = Many<DIM>;
  using M = std::conditional_t<CODED, __half, T>;
  using R = ManyRegs<CODED>;
  extern __shared__ uint8_t many_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(many_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;
  uint8_t* sk = smem + L::QBytes;
  uint8_t* sv = sk + L::Stages * L::Tile;
  __shared__ PagedScratch<kManyThreads> sc;
  __shared__ ManyBars bar;
  __shared__ ManyPart parts[2];
  __shared__ float2 join_ml[2][2][128];                 // (m, l) of a dual part's halves (such parts in turn)
  __shared__ uint32_t bad[L::Stages][4];                        // V rows of an edge block that are not finite
  // 8-bit cache, of each pair of keys: {scale 2^ek, scale 2^ek'}, as deep again as K's ring (a
  // block's softmax reads them when its K's stage is free already); of a block: what V lacks in shared
  // memory, as a power of two and as 2^-that (below zero: rows left the product)
  __shared__ __align__(16) float kscale[CODED ? 2 * L::Stages : 1][CODED ? 64 : 1][2];
  __shared__ float2 vrest[L::Stages];
  __shared__ float qpow[2][CODED ? kManyRows : 1];      // power of two that a row of Q was divided by (parts in turn)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < L::Stages; ++i) {
      mbar_init(&bar.kfull[i], CODED ? 128 : 1);
      mbar_init(&bar.vfull[i], CODED ? 128 : 1);
      mbar_init(&bar.kempty[i], 2);
      mbar_init(&bar.vempty[i], 2);
      mbar_init(&bar.vfix[i], 128);
      mbar_init(&bar.asked[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.drain[i], 1);
      mbar_init(&bar.told[i], 1);
      mbar_init(&bar.heard[i], 14);  // 8 softmax warps, 4 of the loads, 2 of the products
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bar.sfull[i][h], 1);
        mbar_init(&bar.pfull[i][h], 128);
        mbar_init(&bar.odone[i][h], 1);
      }
    }
    mbar_init(&bar.joined, 256);
    mbar_init(&bar.qfull, 128);
    mbar_init(&bar.qempty, 2);
    fence_barrier_init();
    if (a.q_map) tma_prefetch_desc(&tm_q);
    if constexpr (!CODED) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
  }
  if (warp == 14) {
    tmem_alloc(&bar.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem;
  pdl_trigger();
  pdl_wait();
  paged_find<kManyKeys, kManyThreads>(a, blockIdx.x, &sc);
  if (tid == 0) a.cuts[blockIdx.x] = sc.cut[0];
  // Every role walks the same parts: the next one, false at the end (or where the wait was given up).
  uint32_t np_read = 0;
  ManyPart p;
  auto next_part = [&]() {
    const uint32_t i = np_read & 1;
    if (!many_wait1(&bar.told[i], (np_read >> 1) & 1, 1)) return false;
    p = parts[i];
    ++np_read;
    return p.live != 0;
  };
  // its copy in shared memory may be written anew (a warp's lane, or its only thread)
  auto part_read = [&]() { mbar_arrive(&bar.heard[(np_read - 1) & 1]); };

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R::Softmax));
    const int t = warp >> 2, r = tid & 127;
    const int my_i = div_by(r, a.group, a.group_mul), my_h = r - my_i * a.group;  // token of the half, query head
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * 128;
    // so far: blocks of this half, blocks and parts of the CTA; fixes: phase bit of a stage
    uint32_t ns = 0, nb = 0, np = 0, fixes = 0, duals = 0;
    bool ok = true;
    while (ok) {
      if (!__all_sync(0xffffffffu, next_part())) break;
      __syncwarp();
      if (lane == 0) part_read();
      const int tok = (p.dual ? 0 : t * a.half_tokens) + my_i;  // of the tile
      const bool live = my_i < a.half_tokens && tok < p.toks;
      const int pos = live ? p.past + p.tok0 + tok : -1;
      const int see_hi = pos < 0 ? 0 : a.causal ? min(p.len, pos + 1) : p.len;
      const int see_lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
      float m = -INFINITY, l = 0.f;
      const int ja = t ? p.a[1] : p.a[0], jb = t ? p.b[1] : p.b[0];
      if (ja < jb) {
        uint32_t z[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = 0u;
#pragma unroll
        for (int c = 0; c < DIM; c += 32) tmem_st32(to + c, z);
        tmem_st_wait();
      }
      float rs = 1.f;
      const uint32_t ns0 = ns;
      // 64 keys of block j; EDGE: some row of the tile does not see all of the block.  Two copies of
      // the code: what edges need, between the lines of the common path, slows it by a tenth.
      auto step = [&](auto edge_block, int j, int h) {
        constexpr bool EDGE = decltype(edge_block)::value;
        const uint32_t n = nb + j - p.j0, st = n % L::Stages;
        if (!many_wait(&bar.sfull[t][h], ns & 1, 3)) return false;
        tc_fence_after();
        const uint32_t th = ts + h * 64;
        if constexpr (EDGE) {
          if (h == 0 && (!CODED || many_edge(p, j))) {  // its V is in order, and what lies beside it
            if (!many_wait(&bar.vfix[st], (fixes >> st) & 1, 2)) return false;
          }
        }
        if constexpr (CODED) {
          if (h == 0) {
            if constexpr (std::is_same_v<T, __nv_bfloat16>) rs = qpow[np & 1][(p.dual ? 0 : t * 128) + r];
            // (an inner block has been asked for rows that left the product: its V is there)
            if (EDGE && !many_wait(&bar.vfull[st], (n / L::Stages) & 1, 1)) return false;
          }
        }
        uint32_t s0[32], s1[32];
        tmem_ld32(th, s0);
        tmem_ld32(th + 32, s1);
        tmem_ld_wait32(s0);
        tmem_ld_wait32(s1);
        if constexpr (CODED) {
          const uint64_t rs2 = pair2(rs, rs);
          auto to_powers = [&](uint32_t* y, int c0) {
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              const uint64_t ks = *reinterpret_cast<const uint64_t*>(kscale[n % (2 * L::Stages)][(h * 64 + c0 + c) / 2]);
              uint64_t v = pair2(y[c], y[c + 1]);
              if constexpr (std::is_same_v<T, __nv_bfloat16>) v = mul2(v, rs2);
              const float2 f = unpair2(mul2(v, ks));
              y[c] = __float_as_uint(f.x);
              y[c + 1] = __float_as_uint(f.y);
            }
          };
          to_powers(s0, 0);
          to_powers(s1, 32);
        }
        if constexpr (EDGE) {  // what a row does not see (last: a masked key's powers may be no numbers)
          const int k0 = p.lo + j * kManyKeys + h * 64, clo = see_lo - k0, chi = see_hi - k0;
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            if (c < clo || c >= chi) s0[c] = 0xff800000u;
            if (c + 32 < clo || c + 32 >= chi) s1[c] = 0xff800000u;
          }
        }
        float mx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(s0[i]);
#pragma unroll
        for (int c = 4; c < 28; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], __uint_as_float(s0[c + i]), __uint_as_float(s0[c + 4 + i]));
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], __uint_as_float(s0[28 + i]), __uint_as_float(s1[i]));
#pragma unroll
        for (int c = 4; c < 28; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], __uint_as_float(s1[c + i]), __uint_as_float(s1[c + 4 + i]));
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = fmaxf(mx[i], __uint_as_float(s1[28 + i]));
        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        float rest = 0.f;
        if constexpr (CODED) top += rest = vrest[st].x;
        else top *= a.scale;
        const bool raise = top > m + ManyTop<M>::Lazy || (m == -INFINITY && top > -INFINITY);
        const uint32_t odd = EDGE ? bad[st][2 * h] | bad[st][2 * h + 1] : 0u;
        const bool begun = ns > ns0 || h > 0;  // there are sums in O
        const bool any = __any_sync(0xffffffffu, raise);
        if (__builtin_expect(begun && (any || odd), 0)) {  // O stands still once the product before this one is added
          if (!many_wait(&bar.odone[t][h ^ 1], (ns + h + 1) & 1, 3)) return false;
          tc_fence_after();
        }
        if (__builtin_expect(any, 0)) {
          const float c = raise ? (m == -INFINITY ? 0.f : exp2_approx(m - top)) : 1.f;
          if (raise) m = top;
          l *= c;
          if (begun) {
#pragma unroll 1
            for (int d = 0; d < DIM; d += 32) {
              uint32_t o[32];
              tmem_ld32(to + d, o);
              tmem_ld_wait32(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * c);
              tmem_st32(to + d, o);
            }
          }
        }
        const float sub = m == -INFINITY ? 0.f : ManyTop<M>::Top - m;
        if (EDGE && odd) {
          // rows of V that left the product: for the rows that see them, from the cache itself
          tmem_st_wait();
#pragma unroll 1
          for (int c = 0; c < 64; ++c) {
            if (!((bad[st][2 * h + (c >> 5)] >> (c & 31)) & 1u)) continue;
            float w = __uint_as_float(tmem_ld1(th + c));
            const int key = p.lo + j * kManyKeys + h * 64 + c;
            const int page = page_of(a.b, p.seq, key);
            if (page < 0) continue;  // its V is zeros
            const bool see = key >= see_lo && key < see_hi;
            const long long vr = (((long long)page * a.heads + p.head) << a.b.page_shift) + (key & ((1 << a.b.page_shift) - 1));
            if constexpr (CODED)  // (its own power of two in place of the block's)
              w = exp2_approx(fmaf(w * rs, kscale[n % (2 * L::Stages)][(h * 64 + c) >> 1][c & 1], (float)((int)a.v_exp[vr] - 127)) + sub);
            else
              w = exp2_approx(fmaf(w, a.scale, sub));
#pragma unroll 1
            for (int d = 0; d < DIM; d += 32) {
              uint32_t o[32];
              tmem_ld32(to + d, o);
              tmem_ld_wait32(o);
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float2 v;
                if constexpr (CODED)
                  v = Num<__half>::unpack(codes_to_h2(*reinterpret_cast<const uint16_t*>(static_cast<const uint8_t*>(a.v) + vr * DIM + d + i)));
                else
                  v = Num<T>::unpack(*reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.v) + vr * DIM + d + i));
                if (see) {
                  o[i] = __float_as_uint(fmaf(w, v.x, __uint_as_float(o[i])));
                  o[i + 1] = __float_as_uint(fmaf(w, v.y, __uint_as_float(o[i + 1])));
                }
              }
              tmem_st32(to + d, o);
            }
            tmem_st_wait();
          }
        }
        uint64_t sum[2] = {0ull, 0ull};
        const uint64_t scale2 = pair2(CODED ? 1.f : a.scale, CODED ? 1.f : a.scale), sub2 = pair2(sub + rest, sub + rest);
        uint32_t pk[32];
        // 16 values at a time: independent of one another, so that the exponentials follow each other closely
        auto weigh = [&](const uint32_t* y, uint32_t* w) {
#pragma unroll
          for (int c = 0; c < 32; c += 16) {
            float2 e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint64_t v = pair2(y[c + 2 * i], y[c + 2 * i + 1]);
              e[i] = unpair2(CODED ? add2(v, sub2) : fma2(v, scale2, sub2));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              e[i].x = exp2_approx(e[i].x);
              e[i].y = exp2_approx(e[i].y);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint64_t v = pair2(e[i].x, e[i].y);
              sum[i & 1] = add2(v, sum[i & 1]);
              w[c / 2 + i] = Num<M>::pack(e[i].x, e[i].y);
            }
          }
        };
        weigh(s0, pk);
        tmem_st16(th, pk);
        weigh(s1, pk + 16);
        tmem_st16(th + 16, pk + 16);
        const float2 sums = unpair2(add2(sum[0], sum[1]));
        if constexpr (CODED) l = fmaf(sums.x + sums.y, fabsf(vrest[st].y), l);
        else l += sums.x + sums.y;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bar.pfull[t][h]);
        return true;
      };
      // a dual part's blocks by their stages: even ones are half 0's
      auto own = [&](int j) { return j >= ja && j < jb && (!p.dual || ((nb + j - p.j0) & 1) == t); };
      // blocks [i0, i1) are not at the edge
      const int i0 = min(max(p.i0, ja), jb), i1 = min(max(p.i1, i0), jb);
      // 8-bit cache: rows of V left the product (see kSpread), which is the edge's path too.  V is waited
      // for behind the block's scores, as everywhere: see ManyBars.
      auto left = [&](int j) {
        const uint32_t n = nb + j - p.j0, st = n % L::Stages;
        ok = many_wait(&bar.sfull[t][0], ns & 1, 3) && many_wait(&bar.vfull[st], (n / L::Stages) & 1, 1);
        return ok && vrest[st].y < 0.f;
      };
#pragma unroll 1
      for (int j = p.j0; j < p.j1 && ok; ++j) {
        if (j < i0 || j >= i1 || (CODED && own(j) && left(j))) {
          if (own(j) && ok) {
#pragma unroll 1
            for (int h = 0; h < 2 && ok; ++h) ok = step(std::true_type(), j, h);
            ++ns;
          }
          if (many_edge(p, j)) fixes ^= 1u << ((nb + j - p.j0) % L::Stages);
          continue;
        }
#pragma unroll 1
        for (; j < i1 && ok; ++j) {
          if (!own(j)) continue;
          // (written out where the code is short: 3% for a long prompt; over an 8-bit cache it costs 4%)
          if constexpr (!CODED) {
            ok = step(std::false_type(), j, 0) && step(std::false_type(), j, 1);
          } else {
            if (left(j)) break;
#pragma unroll 1
            for (int h = 0; h < 2 && ok; ++h) ok = step(std::false_type(), j, h);
          }
          ++ns;
        }
        --j;
      }
      nb += p.j1 - p.j0;
      np += p.j1 > p.j0;
      if (!ok) break;
      // ---- out, or this part's sums
      const long long slot = 2ll * blockIdx.x + p.first_part;
      if (ja < jb) {
        ok = many_wait(&bar.odone[t][1], (ns - 1) & 1, 3);
        if (!ok) break;
        tc_fence_after();
      }
      int d0 = 0, d1 = DIM;  // the columns that this half writes out
      float c = 1.f, c2 = 0.f;
      const float4* theirs = nullptr;
      if (p.dual) {
        // Each half hands the other one its sums of the other one's columns (through L2: the
        // rings are full already of the next part) and joins its own.
        float4* mine = reinterpret_cast<float4*>(a.part_x) +
                       (((long long)blockIdx.x * 2 + (duals & 1)) * 2 + t) * (DIM / 8) * 128 + r;
#pragma unroll 1
        for (int d = 0; d < DIM / 2; d += 32) {
          uint32_t o[32];
          tmem_ld32(to + (t ^ 1) * (DIM / 2) + d, o);
          tmem_ld_wait32(o);
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            mine[(d + i) / 4 * 128] = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
        }
        join_ml[duals & 1][t][r] = make_float2(m, l);
        mbar_arrive(&bar.joined);
        ok = many_wait(&bar.joined, duals & 1, 3);
        if (!ok) break;
        const float2 ml = join_ml[duals & 1][t ^ 1][r];
        theirs = reinterpret_cast<const float4*>(a.part_x) +
                 (((long long)blockIdx.x * 2 + (duals & 1)) * 2 + (t ^ 1)) * (DIM / 8) * 128 + r;
        ++duals;
        const float top = fmaxf(m, ml.x);
        c = m == -INFINITY ? 0.f : exp2_approx(m - top);
        c2 = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top);
        l = l * c + ml.y * c2;
        m = top;
        d0 = t * (DIM / 2);
        d1 = d0 + DIM / 2;
      }
      const float inv = m == -INFINITY ? 0.f : 1.f / l;
      T* out = static_cast<T*>(a.out) + (long long)(p.seq_tok0 + p.tok0 + tok) * a.o_token +
               (long long)(p.head * a.group + my_h) * a.o_head;
      const int pr = (p.dual ? 0 : t * 128) + r;
      const bool wide = (reinterpret_cast<uintptr_t>(out) & 31) == 0;
#pragma unroll 1
      for (int d = d0; d < d1; d += 32) {
        uint32_t o[32];
        if (ja < jb) {
          tmem_ld32(to + d, o);
          tmem_ld_wait32(o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (p.dual) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 x = __ldcg(theirs + (d - d0 + i) / 4 * 128);
            o[i] = __float_as_uint(fmaf(x.x, c2, __uint_as_float(o[i]) * c));
            o[i + 1] = __float_as_uint(fmaf(x.y, c2, __uint_as_float(o[i + 1]) * c));
            o[i + 2] = __float_as_uint(fmaf(x.z, c2, __uint_as_float(o[i + 2]) * c));
            o[i + 3] = __float_as_uint(fmaf(x.w, c2, __uint_as_float(o[i + 3]) * c));
          }
        }
        if (live) {
          if (p.whole) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              w[i] = Num<T>::pack(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
            st_row64(out + d, w, wide);
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(a.part_o + ((slot * (DIM / 4) + (d + i) / 4) * kManyRows + pr) * 4) =
                  make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
      if (live && !p.whole && d0 == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * kManyRows + pr) * 2) = make_float2(m, l);
      tc_fence_before();  // the next part's zeros and products come after these loads
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------ loads
    if constexpr (R::Load < 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::Load));
    const int lt = tid - 256;
    uint32_t nb = 0, np = 0, edges = 0;  // blocks, parts with blocks so far; phase bits of `asked`
    bool ok = true;
    const int shift = a.b.page_shift, page_rows = 1 << shift;
    const int box_rows = min(page_rows, kManyKeys);
    while (ok) {
      if (!__all_sync(0xffffffffu, next_part())) break;
      __syncwarp();
      if (lane == 0) part_read();
      if (p.j0 >= p.j1) continue;
      const int blocks = p.j1 - p.j0;
      // pages that end in front of it are not looked up: no row sees them, and they may be given up already
      const int from = a.window > 0 ? p.past + p.tok0 - a.window + 1 : 0;

      // 16-bit cache: a warp asks for the blocks of K and another one for those of V (whose stages
      // come free later: one warp for both held K back), a lane for a page.  The pages of a block are
      // looked up while the one before it is on its way.
      auto look_up = [&](int j) {
        const int k0 = p.lo + j * kManyKeys;
        const int boxes = (min(kManyKeys, p.hi - k0) + box_rows - 1) / box_rows;
        if (j >= p.j1 || lane >= boxes) return -1;
        // no page, or one outside the cache: the one behind its last, which TMA fills with zeros
        const int key = k0 + lane * box_rows, page = key + box_rows > from ? page_of(a.b, p.seq, key) : -1;
        return page < 0 ? (int)a.b.pages : page;
      };
      auto fetch = [&](int j, int page, uint32_t n, const CUtensorMap* map, uint8_t* ring, uint64_t* full, uint64_t* empty) {
        const uint32_t st = n % L::Stages;
        if (n >= L::Stages && !many_wait(&empty[st], ((n / L::Stages) & 1) ^ 1, 2)) return false;
        const uint32_t pages = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) mbar_arrive_expect_tx(&full[st], pages * box_rows * DIM * 2);
        __syncwarp();
        if (page >= 0) {
          const int y = p.head * page_rows + ((p.lo + j * kManyKeys + lane * box_rows) & (page_rows - 1));
#pragma unroll
          for (int d = 0; d < DIM / 64; ++d)
            tma_load_3d(ring + st * L::Tile + d * L::Sub + lane * box_rows * 128, map, &full[st], d * 64, y, page);
        }
        return true;
      };
      // 8-bit cache: a thread's codes of block j, 16 a piece; piece lt + 128 i
      constexpr int PR = DIM / 16;                 // pieces of a row
      constexpr int PT = CODED ? 128 * PR / 128 : 1;  // pieces of a thread
      // (the pages of a block: lane l has that of keys 16 l .. 16 l + 15)
      auto pages = [&](int j) {
        const int key = p.lo + j * kManyKeys + lane * 16;
        return j < p.j1 && lane < 8 && key < p.hi && key + 16 > from ? page_of(a.b, p.seq, key) : -1;
      };
      auto hold = [&](int j, int page, const void* cache, uint4 (&c)[PT]) {
        const int k0 = p.lo + j * kManyKeys;
#pragma unroll
        for (int i = 0; i < PT; ++i) {
          const int r = (lt + 128 * i) / PR, at = __shfl_sync(0xffffffffu, page, r >> 4);
          c[i] = make_uint4(0, 0, 0, 0);
          if (at >= 0 && k0 + r < p.hi) {
            const long long kr = (((long long)at * a.heads + p.head) << shift) + ((k0 + r) & (page_rows - 1));
            c[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(cache) + kr * DIM + ((lt + 128 * i) % PR) * 16);
          }
        }
      };
      // their exponent bytes: a thread's key lt of K; of V every warp has all, four keys a lane
      auto byte_of = [&](int j, int page, int r, const uint8_t* exps) {
        return exps + ((((long long)page * a.heads + p.head) << shift) + ((p.lo + j * kManyKeys + r) & (page_rows - 1)));
      };
      auto hold_ek = [&](int j, int page) -> uint32_t {
        const int at = __shfl_sync(0xffffffffu, page, lt >> 4);
        return at < 0 || p.lo + j * kManyKeys + lt >= p.hi ? 127u : *byte_of(j, at, lt, a.k_exp);
      };
      auto hold_ev = [&](int j, int page) -> uint32_t {
        const int at = __shfl_sync(0xffffffffu, page, lane >> 2);
        return at < 0 ? 0x7f7f7f7fu : *reinterpret_cast<const uint32_t*>(byte_of(j, at, 4 * lane, a.v_exp));
      };

      uint4 ck[PT], cv[PT];
      uint32_t ek = 0, ev = 0;
      int v_top = kByteLow;  // the largest exponent byte of V so far that some row sees
      int page = -1;
      if constexpr (CODED) {
        page = pages(p.j0);
        hold(p.j0, page, a.k, ck);
        ek = hold_ek(p.j0, page);
        hold(p.j0, page, a.v, cv);
        ev = hold_ev(p.j0, page);
        page = pages(p.j0 + 1);
      } else {
        if (warp == 8) {
          ok = fetch(p.j0, look_up(p.j0), nb, &tm_k, sk, bar.kfull, bar.kempty);
          page = look_up(p.j0 + 1);
        } else if (warp == 9) {
          page = look_up(p.j0);
        }
      }

      // ---- Q: 128 or 256 rows, swizzled
      if (np > 0 && ok) ok = many_wait(&bar.qempty, (np - 1) & 1, 2);
      ++np;
      const int qrows = p.toks > a.half_tokens ? 256 : 128;
      constexpr int CH = DIM / 8;  // 16-byte pieces of a row
      auto q_src = [&](int i) {
        const int r = (i / CH) & 127, in = div_by(r, a.group, a.group_mul);
        const int tok = min((i / CH >> 7) * a.half_tokens + in, p.toks - 1);  // rows of no token: any
        return static_cast<const T*>(a.q) + (long long)(p.seq_tok0 + p.tok0 + tok) * a.q_token +
               (long long)(p.head * a.group + r - in * a.group) * a.q_head + (i % CH) * 8;
      };
      auto q_dst = [&](int i) {
        const int r = i / CH, ch = i % CH;
        return sq + (r >> 7) * L::Tile + (ch >> 3) * L::Sub + (r & 127) * 128 + (((ch & 7) ^ (r & 7)) * 16);
      };
      if constexpr (CODED && std::is_same_v<T, __nv_bfloat16>) {
        // to f16 by the row's power of two (see cn_paged.cu); CH lanes hold a row
#pragma unroll 1
        for (int i0 = lt; i0 < qrows * CH; i0 += 128 * 4) {
          uint4 w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x)
            w[x] = *reinterpret_cast<const uint4*>(q_src(i0 + x * 128));
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int i = i0 + x * 128;
            uint32_t v[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
            float mx = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = Num<T>::unpack(v[e]);
              mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
#pragma unroll
            for (int o = CH / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const uint32_t eb = min(max(__float_as_uint(mx) >> 23, 16u), 238u);
            const float by = __uint_as_float((254u + 13u - eb) << 23);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = Num<T>::unpack(v[e]);
              v[e] = Num<__half>::pack(f.x * by, f.y * by);
            }
            *reinterpret_cast<uint4*>(q_dst(i)) = make_uint4(v[0], v[1], v[2], v[3]);
            if (i % CH == 0) qpow[(np - 1) & 1][i / CH] = __uint_as_float((eb - 13u) << 23);
          }
        }
      } else if (a.q_map) {
        // a box is a half: half_tokens tokens x the group's heads x 64 values.  What of it belongs to
        // no token of this part are other rows, whose results nobody reads.
        if (lt == 0) {
          mbar_arrive_expect_tx(&bar.qfull, (uint32_t)(qrows / 128 * a.half_tokens * a.group * DIM * 2));
          for (int t = 0; t < qrows / 128; ++t)
#pragma unroll
            for (int d = 0; d < DIM / 64; ++d)
              tma_load_3d(sq + t * L::Tile + d * L::Sub, &tm_q, &bar.qfull, d * 64, p.head * a.group,
                          p.seq_tok0 + p.tok0 + t * a.half_tokens);
        }
      } else {
#pragma unroll 4
        for (int i = lt; i < qrows * CH; i += 128) cp_async16(q_dst(i), q_src(i));
        cp_async_wait_all();
      }
      fence_proxy_async_smem();
      if (lt != 0 || !a.q_map) mbar_arrive(&bar.qfull);

      // ---- blocks
      for (int i = 0; i < blocks && ok; ++i) {
        const int j = p.j0 + i;
        const uint32_t n = nb + i, st = n % L::Stages;
        const bool edge = many_edge(p, j);
        uint32_t left = 0;  // 8-bit cache: this warp's rows of V that are not in the product
        if constexpr (CODED) {
          // K waits for its stage alone: in a dual part the products of the block whose V lies two
          // before wait for this K
          if (n >= L::Stages) ok = many_wait(&bar.kempty[st], ((n / L::Stages) & 1) ^ 1, 2);
          if (!ok) break;
          many_put<DIM, false>(ck, sk + st * L::Tile, lt, 0, 0);
          kscale[n % (2 * L::Stages)][lt >> 1][lt & 1] = exp_byte(ek) * a.scale;
          fence_proxy_async_smem();
          mbar_arrive(&bar.kfull[st]);
          if (i + 1 < blocks) {
            hold(j + 1, page, a.k, ck);
            ek = hold_ek(j + 1, page);
          }
          // the largest power of two of V so far that some row sees: the block's, and each row's way to f16
          const int k0 = p.lo + j * kManyKeys;
          int top = 0, low = 255;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = k0 + 4 * lane + e, byte = (ev >> (8 * e)) & 0xff;
            if (key >= from && key < p.hi) {
              top = max(top, byte);
              low = min(low, byte);
            }
          }
          v_top = max(v_top, __reduce_max_sync(0xffffffffu, min(top, kByteTop)));
          if (n >= L::Stages) ok = many_wait(&bar.vempty[st], ((n / L::Stages) & 1) ^ 1, 2);
          if (!ok) break;
          many_put<DIM, true>(cv, sv + st * L::Tile, lt, ev, v_top);
          // rows that left the product: of all 128 keys, then this warp's 32
          const bool any = __any_sync(0xffffffffu, top > v_top || low < v_top - kSpread);
          if (any) {
            const int mine = (__shfl_sync(0xffffffffu, ev, lt >> 2) >> (8 * (lt & 3))) & 0xff;
            left = __ballot_sync(0xffffffffu, k0 + lt >= from && k0 + lt < p.hi && (mine < v_top - kSpread || mine > v_top));
          }
          if (lane == 0) bad[st][warp - 8] = left;
          if (lt == 0) vrest[st] = make_float2((float)(v_top - 7 - 127), copysignf(inverse_exp_byte(v_top - 7), any ? -1.f : 1.f));
          fence_proxy_async_smem();
          mbar_arrive(&bar.vfull[st]);
          if (i + 1 < blocks) {
            hold(j + 1, page, a.v, cv);
            ev = hold_ev(j + 1, page);
          }
          page = pages(j + 2);
        } else {
          if (warp == 8) {
            if (i + 1 < blocks) ok = fetch(j + 1, page, n + 1, &tm_k, sk, bar.kfull, bar.kempty);
            page = look_up(j + 2);
          } else if (warp == 9) {
            ok = fetch(j, page, n, &tm_v, sv, bar.vfull, bar.vempty);
            page = look_up(j + 1);
          }
        }
        if (edge && ok) {
          // The other warps come here ahead of the one that asks for V, or after it has gone on: a
          // parity tells a phase from the next one only.  So the word that V is asked for goes by
          // stage: a stage's next block waits for this fix, that is, for all four warps.
          if constexpr (!CODED) {
            if (lt == 32) mbar_arrive(&bar.asked[st]);
            ok = __all_sync(0xffffffffu, mbar_wait(&bar.asked[st], (edges >> st) & 1, 2));  // asleep: it can take long
            edges ^= 1u << st;
            if (!ok) break;
          }
          ok = many_wait(&bar.vfull[st], (n / L::Stages) & 1, 1);
          if (!ok) break;
          const int key = p.lo + j * kManyKeys + lt;
          uint8_t* vr = sv + st * L::Tile + lt * 128;
          bool odd = false;
          if (key < p.len && key < p.hi) {
#pragma unroll
            for (int d = 0; d < DIM / 64; ++d)
#pragma unroll 4
              for (int c = 0; c < 8; ++c) {
                const uint4 w = *reinterpret_cast<const uint4*>(vr + d * L::Sub + ((c + lt) & 7) * 16);
                odd |= not_finite2<M>(w.x) | not_finite2<M>(w.y) | not_finite2<M>(w.z) | not_finite2<M>(w.w);
              }
          }
          if (odd || key >= p.len || key >= p.hi) {
#pragma unroll
            for (int d = 0; d < DIM / 64; ++d)
#pragma unroll 4
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(vr + d * L::Sub + ((c + lt) & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          const uint32_t bits = __ballot_sync(0xffffffffu, odd);
          if (lane == 0) bad[st][warp - 8] = bits | left;
          fence_proxy_async_smem();
          mbar_arrive(&bar.vfix[st]);
        }
      }
      nb += blocks;
    }
    if (!ok && !CODED && lane == 0) {  // given up: the copies in flight land before the block ends
      const unsigned long long t0 = global_ns();
      while (global_ns() - t0 < 100000000ull) {
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::Mma));
    if (warp < 14 && elect_one()) {
      // ------------------------------------------------------------ products
      constexpr uint32_t id_s = many_idesc<M>(64, false), id_o = many_idesc<M>(DIM, true);
      const int t = warp - 12;
      uint32_t nb = 0, np = 0, ns = 0, fixes = 0;
      bool ok = true;
      const uint32_t q_lo0 = desc_lo(sq, 16), k_lo = desc_lo(sk, 16), v_lo = desc_lo(sv, L::Sub);
      const uint32_t d_s = tmem + t * 128, d_o = tmem + 256 + t * 128;
      // S of keys h * 64 .. of a block: rows h * 64 .. of the K tile
      auto scores = [&](uint32_t q_lo, int h, uint32_t st) {
        const uint32_t ka = k_lo + st * (L::Tile >> 4) + h * (64 * 128 >> 4);
        tc_mma_ss<false>(d_s + h * 64, q_lo, ka, id_s);
#pragma unroll
        for (int k = 1; k < DIM / 16; ++k) {
          const uint32_t off = ((k >> 2) * L::Sub + (k & 3) * 32) >> 4;
          tc_mma_ss<true>(d_s + h * 64, q_lo + off, ka + off, id_s);
        }
        tc_commit(&bar.sfull[t][h]);
      };
      // O += P V of those keys
      auto sums = [&](int h, uint32_t st) {
        const uint32_t va = v_lo + st * (L::Tile >> 4) + h * (64 * 128 >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_ts(d_o, d_s + h * 64 + k * 8, va + k * (2048 >> 4), id_o);
        tc_commit(&bar.odone[t][h]);
      };
      auto stage = [](uint32_t n) { return n % L::Stages; };
      auto phase = [](uint32_t n) { return (n / L::Stages) & 1; };
      auto v_there = [&](int j, uint32_t n) {
        if (!many_wait1(&bar.vfull[stage(n)], phase(n), 1)) return false;
        return !many_edge(p, j) || many_wait1(&bar.vfix[stage(n)], (fixes >> stage(n)) & 1, 1);
      };
      while (ok && next_part()) {
        part_read();
        if (p.j0 >= p.j1) continue;
        const int ja = t ? p.a[1] : p.a[0], jb = t ? p.b[1] : p.b[0];
        const uint32_t q_lo = q_lo0 + (p.dual ? 0 : t * (L::Tile >> 4));
        ok = many_wait1(&bar.qfull, np & 1, 1);
        if (!ok) break;
        ++np;
        if (p.dual) {
          // this half's blocks: every second one, in stages that are this half's alone (it gives
          // both halves' word that they are free)
          int j = p.j0 + ((nb + t) & 1);
          uint32_t n = nb + j - p.j0;
          for (int i = p.j0; i < p.j1; ++i)  // fix phases of the other half's blocks
            if (many_edge(p, i) && ((i - j) & 1)) fixes ^= 1u << stage(nb + i - p.j0);
          ok = many_wait1(&bar.kfull[stage(n)], phase(n), 1);
          if (!ok) break;
          tc_fence_after();
          scores(q_lo, 0, stage(n));
          scores(q_lo, 1, stage(n));
          tc_commit(&bar.kempty[stage(n)]);
          tc_commit(&bar.kempty[stage(n)]);
#pragma unroll 1
          for (; j < p.j1; j += 2, n += 2) {
            ok = v_there(j, n);
            if (!ok) break;
            if (many_edge(p, j)) fixes ^= 1u << stage(n);
            const bool again = j + 2 < p.j1;
            // Q is free once the last scores are there, but the word waits for this half's last V as
            // well: see ManyBars
            if (!again) tc_commit(&bar.qempty);
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              ok = many_wait1(&bar.pfull[t][h], ns & 1, 3);
              if (ok && again && h == 0) ok = many_wait1(&bar.kfull[stage(n + 2)], phase(n + 2), 1);
              if (!ok) break;
              tc_fence_after();
              sums(h, stage(n));
              if (again) scores(q_lo, h, stage(n + 2));
            }
            if (!ok) break;
            ++ns;
            if (again) {
              tc_commit(&bar.kempty[stage(n + 2)]);
              tc_commit(&bar.kempty[stage(n + 2)]);
            }
            tc_commit(&bar.vempty[stage(n)]);
            tc_commit(&bar.vempty[stage(n)]);
          }
          if (!ok) break;
        } else {
          ok = many_wait1(&bar.kfull[stage(nb)], phase(nb), 1);
          if (!ok) break;
          tc_fence_after();
          if (ja == p.j0 && ja < jb) {
            scores(q_lo, 0, stage(nb));
            scores(q_lo, 1, stage(nb));
          }
          tc_commit(&bar.kempty[stage(nb)]);
          if (p.j1 == p.j0 + 1) tc_commit(&bar.qempty);
#pragma unroll 1
          for (int j = p.j0; j < p.j1; ++j) {
            const uint32_t n = nb + j - p.j0;
            ok = v_there(j, n);
            if (many_edge(p, j)) fixes ^= 1u << stage(n);
            if (ok && j + 1 < p.j1) ok = many_wait1(&bar.kfull[stage(n + 1)], phase(n + 1), 1);
            if (!ok) break;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              if (j >= ja && j < jb) {
                ok = many_wait1(&bar.pfull[t][h], ns & 1, 3);
                if (!ok) break;
                tc_fence_after();
                sums(h, stage(n));
              }
              if (j + 1 >= ja && j + 1 < jb) scores(q_lo, h, stage(n + 1));
            }
            if (!ok) break;
            ns += j >= ja && j < jb;
            if (j + 1 < p.j1) {
              tc_commit(&bar.kempty[stage(n + 1)]);
              if (j + 2 == p.j1) tc_commit(&bar.qempty);
            }
            tc_commit(&bar.vempty[stage(n)]);
          }
          if (!ok) break;
        }
        nb += p.j1 - p.j0;
      }
      // the last products and their arrivals end before the block does
      tc_commit(&bar.drain[t]);
      many_wait1(&bar.drain[t], 0, 3);
    }
    if (warp == 15 && lane == 0) {
      // ------------------------------------------------------------ parts
      long long at = sc.cut[0].start, first = sc.cut[0].first;
      const long long end = sc.cut[1].start;
      int s = sc.cut[0].seq, head = sc.cut[0].head, tile = sc.cut[0].tile;
      bool more = at < end, ok = true;
      PagedSeq q = {};
      if (more) q = paged_seq(a, s);
      for (uint32_t n = 0; ok; ++n) {
        ManyPart next;
        next.live = 0;
        if (more) {
          const int units = paged_blocks<kManyKeys>(a, q, tile);
          next = many_part(a, q, s, head, tile, paged_block_at(a, at, first, units), paged_block_at(a, end, first, units), units);
          first += units + a.extra;
          at = first;
        }
        if (n >= 2) ok = many_wait1(&bar.heard[n & 1], ((n >> 1) & 1) ^ 1, 2);
        if (!ok) break;
        parts[n & 1] = next;
        mbar_arrive(&bar.told[n & 1]);
        if (!more) break;
        more = at < end && paged_next(a, &q, &s, &head, &tile);
      }
    }
    __syncwarp();
  }
  // Every product's result was waited for by the softmax that used it; the others (a give-up) end here.
  tc_fence_before();
  __syncthreads();
  if (warp == 14) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace
}  // namespace cn
