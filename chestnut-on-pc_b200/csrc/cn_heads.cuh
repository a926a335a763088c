// What the temporal-context kernels share: checks of their descriptors, the
// call's device, row loads and stores of 16-bit types, and the 8-bit rows of
// the cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "../../include/chestnut.h"
#include "cn_common.cuh"
#include "cn_gemm.cuh"

namespace cn {

// Device error word: a page table entry names no page of the cache, or a
// position lies past the table.
constexpr int kErrPage = 6;

// Runs a call on the GPU that holds its data and puts the current device back.
// Every pointer handed to use() has to be memory of that one GPU.
class DataDevice {
 public:
  ~DataDevice() {
    if (switched_) cudaSetDevice(before_);
  }
  int use(const char* who, const void* p) {
    cudaPointerAttributes at;
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_last_error("%s: %s", who, cudaGetErrorString(e));
      return CN_ERR_CUDA;
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) {
      set_last_error("%s: a pointer is not device memory", who);
      return CN_ERR_ARG;
    }
    if (device_ < 0) {
      device_ = at.device;
      if (cudaGetDevice(&before_) != cudaSuccess || (before_ != device_ && cudaSetDevice(device_) != cudaSuccess)) {
        set_last_error("%s: device %d cannot be used", who, device_);
        return CN_ERR_CUDA;
      }
      switched_ = before_ != device_;
    } else if (at.type == cudaMemoryTypeDevice && at.device != device_) {
      set_last_error("%s: its pointers lie on devices %d and %d", who, device_, at.device);
      return CN_ERR_ARG;
    }
    return 0;
  }
  int device() const { return device_; }

 private:
  int device_ = -1, before_ = 0;
  bool switched_ = false;
};

inline int launch_status(const char* who, cudaError_t e) {
  if (e == cudaSuccess) return 0;
  cudaGetLastError();
  set_last_error("%s: launch failed: %s", who, cudaGetErrorString(e));
  return CN_ERR_CUDA;
}

inline int dtype_bytes(int dtype) { return dtype == CN_F32 ? 4 : dtype == CN_E4M3 ? 1 : 2; }

inline bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// Checks of a [tokens][heads][dim] view; `written`: no two of its rows may overlap.  Without tokens it
// needs no memory (an empty tensor has no address).
inline int check_heads(const char* who, const char* name, const cn_heads* h, long long tokens, bool written) {
  if (!h || (!h->data && tokens > 0)) {
    set_last_error("%s: %s is missing", who, name);
    return CN_ERR_ARG;
  }
  if (h->dtype != CN_F16 && h->dtype != CN_BF16 && h->dtype != CN_F32) {
    set_last_error("%s: %s has dtype %d", who, name, h->dtype);
    return CN_ERR_ARG;
  }
  if (h->heads < 1 || h->heads > 65535 || h->dim < 8 || h->dim > 256 || h->dim % 8) {
    set_last_error("%s: %s has %d heads of %d values (1 to 65535 heads, dim a multiple of 8 up to 256)", who, name,
                   h->heads, h->dim);
    return CN_ERR_ARG;
  }
  const int size = dtype_bytes(h->dtype);
  const long long ts = h->token_stride, hs = h->head_stride;
  if (misaligned16(h->data) || ts < 0 || hs < 0 || (ts * size) % 16 || (hs * size) % 16) {
    set_last_error("%s: %s: data and strides must be multiples of 16 bytes, strides not negative", who, name);
    return CN_ERR_ARG;
  }
  if (written) {
    // the dimension with the smaller stride holds whole rows, the other one whole runs of it
    bool apart = true;
    if (tokens > 1 && h->heads > 1)
      apart = hs <= ts ? hs >= h->dim && ts >= (h->heads - 1) * hs + h->dim
                       : ts >= h->dim && hs >= (tokens - 1) * ts + h->dim;
    else if (tokens > 1)
      apart = ts >= h->dim;
    else if (h->heads > 1)
      apart = hs >= h->dim;
    if (!apart) {
      set_last_error("%s: rows of %s overlap", who, name);
      return CN_ERR_ARG;
    }
  }
  return 0;
}

inline int check_cache(const char* who, const cn_kv_cache* c) {
  if (!c || !c->k || !c->v) {
    set_last_error("%s: the cache is missing", who);
    return CN_ERR_ARG;
  }
  const bool coded = c->dtype == CN_E4M3;
  if (c->dtype != CN_F16 && c->dtype != CN_BF16 && !coded) {
    set_last_error("%s: the cache has dtype %d", who, c->dtype);
    return CN_ERR_ARG;
  }
  if (coded != (c->k_exp != nullptr) || coded != (c->v_exp != nullptr)) {
    set_last_error("%s: k_exp and v_exp belong to an e4m3 cache, and to no other", who);
    return CN_ERR_ARG;
  }
  if ((c->dim != 64 && c->dim != 128) || c->heads < 1 || c->heads > 65535 || c->page < 16 || c->page > 256 ||
      (c->page & (c->page - 1)) || c->pages < 1 || c->pages > INT32_MAX) {
    set_last_error("%s: cache of %lld pages x %d heads x %d rows x %d values (dim 64 or 128; page 16, 32, 64, 128 or 256)",
                   who, c->pages, c->heads, c->page, c->dim);
    return CN_ERR_ARG;
  }
  if (misaligned16(c->k) || misaligned16(c->v) || misaligned16(c->k_exp) || misaligned16(c->v_exp)) {
    set_last_error("%s: the cache's buffers must be 16-byte aligned", who);
    return CN_ERR_ARG;
  }
  return 0;
}

inline int check_batch(const char* who, const cn_kv_batch* b, const cn_kv_cache* c) {
  if (!b || b->n_seqs < 0 || b->n_seqs > 65535 || b->table_width < 0 || b->table_stride < 0 ||
      (b->n_seqs > 0 && (!b->cu_tokens || !b->lengths || (b->table_width > 0 && !b->table)))) {
    set_last_error("%s: the batch is missing or malformed (at most 65535 sequences)", who);
    return CN_ERR_ARG;
  }
  if ((long long)b->table_width * c->page > (1ll << 30)) {
    set_last_error("%s: contexts of %d pages x %d rows exceed 2^30 tokens", who, b->table_width, c->page);
    return CN_ERR_ARG;
  }
  return 0;
}

// ---- element types
template <typename T>
struct Num;
template <>
struct Num<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Num<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// 2^(byte - 127) of a row's exponent byte; the bytes that cn_kv_write makes are 79 .. 175.
__device__ __forceinline__ float exp_byte(uint32_t byte) { return __uint_as_float(byte << 23); }
// 2^(127 - byte), finite for every byte: a masked key's weight, 0, is multiplied by it, and its byte
// may be anything (255 is no power that a row can have: 0 then).
__device__ __forceinline__ float inverse_exp_byte(uint32_t byte) { return __uint_as_float((254u - min(byte, 254u)) << 23); }

// Two e4m3 codes (low byte first) to two f16 values: exact, e4m3 is a subset of f16.
__device__ __forceinline__ uint32_t codes_to_h2(uint32_t codes16) {
  uint32_t r;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(r) : "r"(codes16));
  return r;
}
// Two f32 to two e4m3 codes: nearest, ties to even, beyond 448 to 448, NaN to NaN.
__device__ __forceinline__ uint32_t floats_to_codes(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b16 c;\n\tcvt.rn.satfinite.e4m3x2.f32 c, %2, %1;\n\tcvt.u32.u16 %0, c;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}

// ---- where a token's row lies
struct BatchArgs {
  const int *cu, *lengths, *table;
  int n_seqs, table_width, page_shift;
  long long table_stride, pages, tokens;
};

inline BatchArgs batch_args(const cn_kv_cache* c, const cn_kv_batch* b, long long tokens) {
  BatchArgs a;
  a.cu = b->cu_tokens;
  a.lengths = b->lengths;
  a.table = b->table;
  a.n_seqs = b->n_seqs;
  a.table_width = b->table_width;
  a.page_shift = __builtin_ctz((unsigned)c->page);
  a.table_stride = b->table_stride;
  a.pages = c->pages;
  a.tokens = tokens;
  return a;
}

// The batch's arrays are read with plain loads: the kernel may start (programmatic
// dependent launch) while the call before still writes them, so they are not
// read-only for its whole life.

// Page number of position pos (not negative) of sequence s, or -1 with the error word set.
__device__ __forceinline__ int page_of(const BatchArgs& a, int s, int pos) {
  const int i = pos >> a.page_shift;
  const int p = i < a.table_width ? a.table[s * a.table_stride + i] : -1;
  if (p < 0 || p >= a.pages) {
    set_dev_error(kErrPage);
    return -1;
  }
  return p;
}

}  // namespace cn
