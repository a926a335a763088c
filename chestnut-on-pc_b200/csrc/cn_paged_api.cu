// Attention over the paged cache: choice of the launches, workspace, entry points.
#include <cmath>

#include "cn_paged.cuh"

namespace cn {
namespace {

// Workspace of one launch: the cuts, then the parts.
struct PagedSpace {
  size_t o, ml, x, bytes;
};
PagedSpace paged_space(int ctas, int rows, int dim) {
  PagedSpace s;
  s.o = ((size_t)(ctas + 1) * sizeof(PagedCut) + 255) / 256 * 256;
  s.ml = s.o + (size_t)2 * ctas * rows * dim * 4;
  s.x = s.ml + ((size_t)2 * ctas * rows * 2 * 4 + 255) / 256 * 256;
  s.bytes = s.x + (rows == kManyRows ? (size_t)ctas * 4 * 128 * (dim / 2) * 4 : 0);
  return s;
}

int sm_count(int dev) {
  static int count[64];
  if (dev < 0 || dev >= 64) return 148;
  if (!count[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
      cudaGetLastError();
      return 148;
    }
    count[dev] = n;
  }
  return count[dev];
}

constexpr int kFewCtas = 3 * 148;  // three CTAs an SM over an 8-bit cache, two over a 16-bit one

constexpr int kManyCtas = 148;

template <typename T, int DIM, bool CODED>
cudaError_t few_launch(const PagedArgs& a, int dev, cudaStream_t s) {
  static unsigned long long ready = 0;
  if (dev >= 64 || !(ready & (1ull << dev))) {
    const cudaError_t e = cudaFuncSetAttribute(k_paged_few<T, DIM, CODED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)Few<DIM, CODED>::Smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready |= 1ull << dev;
  }
  return launch_ex(k_paged_few<T, DIM, CODED>, dim3(a.ctas), dim3(kFewThreads), Few<DIM, CODED>::Smem, s, true, a);
}

template <typename T, int DIM, bool CODED>
cudaError_t many_launch(const PagedArgs& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, int dev,
                        cudaStream_t s) {
  static unsigned long long ready = 0;
  if (dev >= 64 || !(ready & (1ull << dev))) {
    cudaFuncAttributes at;
    cudaError_t e = cudaFuncGetAttributes(&at, k_paged_many<T, DIM, CODED>);
    // the warpgroups share out 4 x 128 registers: a block launched with fewer would wait for ever
    if (e == cudaSuccess && at.numRegs != 128) e = cudaErrorInvalidKernelImage;
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(k_paged_many<T, DIM, CODED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)Many<DIM>::Smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready |= 1ull << dev;
  }
  return launch_ex(k_paged_many<T, DIM, CODED>, dim3(a.ctas), dim3(kManyThreads), Many<DIM>::Smem, s, true, tq, tk, tv, a);
}

// One call: the launches for few and for many rows (each where it may find work).
struct PagedCall {
  PagedArgs few, many;
  bool do_few, do_many;
  int merge_few, merge_many;  // blocks of the merge
  CUtensorMap tq, tk, tv;
};

template <typename T, int DIM, bool CODED>
cudaError_t paged_launch(const PagedCall& c, int dev, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (c.do_few) e = few_launch<T, DIM, CODED>(c.few, dev, s);
  if (e == cudaSuccess && c.do_many) e = many_launch<T, DIM, CODED>(c.many, c.tq, c.tk, c.tv, dev, s);
  if (e == cudaSuccess && c.merge_few + c.merge_many)
    e = launch_ex(k_paged_merge<T, DIM>, dim3(c.merge_few + c.merge_many), dim3(256), 0, s, true, c.few, c.many, c.merge_few);
  return e;
}

template <typename T>
cudaError_t paged_dispatch(const PagedCall& c, int dim, bool coded, int dev, cudaStream_t s) {
  if (dim == 128) return coded ? paged_launch<T, 128, true>(c, dev, s) : paged_launch<T, 128, false>(c, dev, s);
  return coded ? paged_launch<T, 64, true>(c, dev, s) : paged_launch<T, 64, false>(c, dev, s);
}

// A 16-bit cache as [pages][heads * page rows][dim], boxes of up to 128 rows of a page x 64 values.
int paged_map(CUtensorMap* m, const cn_kv_cache* c, const void* base) {
  const uint64_t d[3] = {(uint64_t)c->dim, (uint64_t)c->heads * c->page, (uint64_t)c->pages};
  const uint64_t st[2] = {(uint64_t)c->dim * 2, (uint64_t)c->heads * c->page * c->dim * 2};
  const uint32_t b[3] = {64, (uint32_t)(c->page < kManyKeys ? c->page : kManyKeys), 1};
  return encode(m, c->dtype == CN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, d,
                st, b, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The queries as [tokens][heads][dim], boxes of one half of a tile.  Strides of 0 (rows that are
// the same memory) are left to the kernel's own loads.
bool paged_q_map(CUtensorMap* m, const cn_heads* q, long long tokens, int group, int half_tokens) {
  if ((q->heads > 1 && q->head_stride == 0) || (tokens > 1 && q->token_stride == 0)) return false;
  const uint64_t row = (uint64_t)q->dim * 2;
  const uint64_t d[3] = {(uint64_t)q->dim, (uint64_t)q->heads, (uint64_t)tokens};
  const uint64_t st[2] = {q->heads > 1 ? (uint64_t)q->head_stride * 2 : row, tokens > 1 ? (uint64_t)q->token_stride * 2 : row};
  if (st[0] >= 1ull << 40 || st[1] >= 1ull << 40) return false;
  const uint32_t b[3] = {64, (uint32_t)group, (uint32_t)half_tokens};
  return encode(m, q->dtype == CN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, q->data, d, st,
                b, CU_TENSOR_MAP_SWIZZLE_128B) == 0;
}

// sizes_only: q's rows need no memory yet.
int paged_check(const char* who, const cn_kv_cache* cache, const cn_kv_batch* batch, const cn_heads* q,
                long long tokens, bool sizes_only) {
  int r;
  if ((r = check_cache(who, cache)) || (r = check_batch(who, batch, cache)) ||
      (r = check_heads(who, "q", q, sizes_only ? 0 : tokens, false)))
    return r;
  if (q->dtype == CN_F32 || (cache->dtype != CN_E4M3 && cache->dtype != q->dtype)) {
    set_last_error("%s: q has dtype %d, the cache %d (q f16 or bf16, a 16-bit cache the same)", who, q->dtype, cache->dtype);
    return CN_ERR_ARG;
  }
  if (q->dim != cache->dim || q->heads % cache->heads) {
    set_last_error("%s: %d query heads of %d values over %d cache heads of %d", who, q->heads, q->dim, cache->heads,
                   cache->dim);
    return CN_ERR_ARG;
  }
  if (q->heads / cache->heads > 128) {
    set_last_error("%s: %d query heads read one cache head (at most 128)", who, q->heads / cache->heads);
    return CN_ERR_ARG;
  }
  if (tokens < 0 || tokens > (1ll << 30) / (q->heads / cache->heads)) {
    set_last_error("%s: %lld tokens (tokens x query heads of a cache head: at most 2^30)", who, tokens);
    return CN_ERR_ARG;
  }
  return 0;
}

}  // namespace
}  // namespace cn

extern "C" int cn_paged_attention_workspace(const cn_kv_cache* cache, const cn_kv_batch* batch, const cn_heads* q,
                                            long long tokens, size_t* bytes) {
  using namespace cn;
  const char* who = "cn_paged_attention_workspace";
  if (!bytes) {
    set_last_error("%s: bytes is NULL", who);
    return CN_ERR_ARG;
  }
  const int r = paged_check(who, cache, batch, q, tokens, true);
  if (r) return r;
  *bytes = paged_space(kFewCtas, kFewRows, cache->dim).bytes + paged_space(kManyCtas, kManyRows, cache->dim).bytes;
  return 0;
}

extern "C" int cn_paged_attention(const cn_kv_cache* cache, const cn_kv_batch* batch, const cn_heads* q,
                                  const cn_heads* out, long long tokens, float scale, int causal, int window,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  using namespace cn;
  const char* who = "cn_paged_attention";
  int r = paged_check(who, cache, batch, q, tokens, false);
  if (r || (r = check_heads(who, "out", out, tokens, true))) return r;
  if (out->dtype != q->dtype || out->heads != q->heads || out->dim != q->dim) {
    set_last_error("%s: q and out differ in dtype, heads or dim", who);
    return CN_ERR_ARG;
  }
  if (window < 0 || (window > 0 && !causal)) {
    set_last_error("%s: window %d (a window needs causal)", who, window);
    return CN_ERR_ARG;
  }
  if (!(scale > 0.f) || std::isinf(scale)) {
    set_last_error("%s: scale %g (positive and finite)", who, (double)scale);
    return CN_ERR_ARG;
  }
  const PagedSpace few = paged_space(kFewCtas, kFewRows, cache->dim), many = paged_space(kManyCtas, kManyRows, cache->dim);
  if (tokens > 0 &&
      (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < few.bytes + many.bytes)) {
    set_last_error("%s: workspace of %zu bytes, 256-byte aligned, is needed (%zu given)", who, few.bytes + many.bytes,
                   workspace_bytes);
    return CN_ERR_ARG;
  }
  if (tokens == 0 || batch->n_seqs == 0) return 0;
  DataDevice dev;
  const void* all[] = {cache->k, cache->v, q->data, out->data, batch->cu_tokens, batch->lengths, workspace};
  for (const void* p : all)
    if ((r = dev.use(who, p))) return r;
  if (batch->table_width && (r = dev.use(who, batch->table))) return r;
  const bool coded = cache->dtype == CN_E4M3;
  if (coded && ((r = dev.use(who, cache->k_exp)) || (r = dev.use(who, cache->v_exp)))) return r;
  PagedArgs a;
  a.b = batch_args(cache, batch, tokens);
  a.q = q->data;
  a.out = out->data;
  a.q_token = q->token_stride;
  a.q_head = q->head_stride;
  a.o_token = out->token_stride;
  a.o_head = out->head_stride;
  a.k = cache->k;
  a.v = cache->v;
  a.k_exp = cache->k_exp;
  a.v_exp = cache->v_exp;
  a.heads = cache->heads;
  a.group = q->heads / cache->heads;
  a.group_mul = a.group == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / (uint32_t)a.group);
  a.scale = scale * 1.44269504088896340736f;
  a.causal = causal != 0;
  a.window = min(window, 1 << 30);  // positions end below it
  // Sequences of up to 16 rows go to the kernel for few rows, the others to the
  // tensor-core one.  How long each is, only the device knows; a launch that cannot
  // find work is left out.  So is one that costs more than it can give: the first
  // kernel takes any sequence in tiles of 16 rows, each of which reads the context
  // from L2, and a second launch that finds nothing costs 11 us (64 tokens of 64
  // clips over 1000 each, 16 heads x 128 f16: 93 us, with it 105).  It takes all
  //  - where no sequence can have more than 128 rows, however the tokens are spread
  //    (two 64-token frames over 300 / 1000 / 4000 / 16000 tokens: 19 / 25 / 47 / 132
  //    us; both kernels: 26 / 33 / 46 / 82);
  //  - where none has if each sequence has a token or more, as in a step of one token
  //    a clip, and the rows are 512 at most.  Where sequences are empty and one has
  //    all the tokens, that costs (64 slots, a 64-token frame in one, 4 heads a group,
  //    over the same lengths: 21 / 26 / 49 / 123 us; both: 25 / 28 / 37 / 52), and
  //    beyond 512 rows more than it saves.
  const long long rows = tokens * a.group;
  const bool short_all = rows <= 128, short_likely = (tokens - batch->n_seqs + 1) * a.group <= 128 && rows <= 512;
  const bool steps = batch->n_seqs > 1 && a.group <= kFewRows && (short_all || short_likely);
  PagedCall c;
  memset(&c, 0, sizeof(c));
  c.do_few = batch->n_seqs > 1 ? a.group <= kFewRows : rows <= kFewRows;
  c.do_many = !(steps || rows <= kFewRows);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const long long cap = (long long)batch->table_width * cache->page;
  if (c.do_few) {
    PagedArgs& f = c.few = a;
    f.rows_min = 1;
    f.rows_max = c.do_many ? kFewRows : INT32_MAX;
    f.ctas = min((coded ? 3 : 2) * sm_count(dev.device()), kFewCtas);
    f.tile_tokens = f.half_tokens = kFewRows / a.group;
    f.min_units = f.snap = 4;
    f.extra = 1;
    f.cuts = reinterpret_cast<PagedCut*>(w);
    f.part_o = reinterpret_cast<float*>(w + few.o);
    f.part_ml = reinterpret_cast<float*>(w + few.ml);
    if (cap > (long long)f.snap * kFewKeys) c.merge_few = f.ctas - 1;  // else no tile is ever cut
  }
  if (c.do_many) {
    PagedArgs& m = c.many = a;
    m.rows_min = c.do_few ? kFewRows + 1 : 1;
    m.rows_max = INT32_MAX;
    m.ctas = min(sm_count(dev.device()), kManyCtas);
    m.half_tokens = kManyRows / 2 / a.group;
    m.tile_tokens = 2 * m.half_tokens;
    m.min_units = m.snap = 2;
    m.extra = 2;
    w += few.bytes;
    m.cuts = reinterpret_cast<PagedCut*>(w);
    m.part_o = reinterpret_cast<float*>(w + many.o);
    m.part_ml = reinterpret_cast<float*>(w + many.ml);
    m.part_x = reinterpret_cast<float*>(w + many.x);
    if (cap > (long long)m.snap * kManyKeys) c.merge_many = (m.ctas - 1) * (kManyRows / kManyMergeRows);
    // (bf16 rows over an 8-bit cache are scaled to f16 on their way)
    m.q_map = !(coded && q->dtype == CN_BF16) && paged_q_map(&c.tq, q, tokens, m.group, m.half_tokens);
    if (!coded && (paged_map(&c.tk, cache, cache->k) || paged_map(&c.tv, cache, cache->v))) return CN_ERR_CUDA;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return launch_status(who, q->dtype == CN_F16 ? paged_dispatch<__half>(c, cache->dim, coded, dev.device(), s)
                                               : paged_dispatch<__nv_bfloat16>(c, cache->dim, coded, dev.device(), s));
}
