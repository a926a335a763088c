"""Kernel-level entry points (device pointers), mirroring the reference's
per-kernel A/B harnesses (``bench_r62.py``, ``bench_alu.py``): the same
kernel launched on caller-provided buffers."""
import ctypes
import math

from . import _lib
from ._lib import check, lib

DTYPES = {"f16": 0, "bf16": 1, "f32": 2, "e4m3": 3}  # CN_F16 ... CN_E4M3


def gemm_wmma_f16(A, B, C, M, N, K, b_kmajor, bn=0, splits=0, stream=None):
    """C[M][N] += A[M][K] * B (device pointers); WMMA semantics D = C + A*B."""
    check(lib().cn_gemm_wmma_f16(A, B, C, M, N, K, int(b_kmajor), bn, splits, stream), "cn_gemm_wmma_f16")


def reduce_rows_f16(x, w, out, rows, length, chunks_per_row=0, stream=None):
    """out[r] = sum_i x[r][i] * w[i] (device pointers)."""
    check(lib().cn_reduce_rows_f16(x, w, out, rows, length, chunks_per_row, stream), "cn_reduce_rows_f16")


def border_gather_s2(act, G, B, H, W, C, out, stream=None):
    check(lib().cn_border_gather_s2(act, G, B, H, W, C, out, stream), "cn_border_gather_s2")


def warp_frames(frame, big_frame, tfm, big_tfm, width, height, stride, y_height, uv_height, out,
                model_w=512, model_h=256, stream=None):
    """Road + wide NV12 frames (device pointers) -> model input u8[2,6,model_h/2,model_w/2]
    at device pointer out.  tfm / big_tfm: 3x3 inverse transforms (anything numpy
    turns into 9 float32 values, row-major)."""
    import numpy as np
    m0 = np.ascontiguousarray(np.asarray(tfm, np.float32).reshape(9))
    m1 = np.ascontiguousarray(np.asarray(big_tfm, np.float32).reshape(9))
    check(lib().cn_warp_frames(frame, big_frame, m0.ctypes.data, m1.ctypes.data, width, height, stride, y_height,
                               uv_height, model_w, model_h, out, stream), "cn_warp_frames")


# ---- temporal context: rotary positions, paged K/V cache, attention ----------


def heads(ptr, dtype, n_heads, dim, token_stride=None, head_stride=None):
    """Rows [tokens][n_heads][dim] at device pointer ptr; strides in elements (default: contiguous)."""
    hs = dim if head_stride is None else head_stride
    return _lib.cn_heads(ptr, DTYPES[dtype], n_heads, dim, n_heads * dim if token_stride is None else token_stride, hs)


def kv_cache(k, v, dtype, pages, page, n_heads, dim, k_exp=None, v_exp=None):
    """A paged cache over device buffers k, v [pages][n_heads][page][dim]; dtype "f16", "bf16" or
    "e4m3" (then k_exp, v_exp: u8 [pages][n_heads][page], each row's power of two + 127)."""
    return _lib.cn_kv_cache(k, v, k_exp, v_exp, DTYPES[dtype], n_heads, dim, page, pages)


def kv_batch(n_seqs, cu_tokens, lengths, table, table_width, table_stride=None):
    """Device i32 arrays: cu_tokens [n_seqs + 1] (rows of the new tokens), lengths [n_seqs] (tokens of
    each context, the new ones included), table [n_seqs][table_width] (page numbers)."""
    return _lib.cn_kv_batch(n_seqs, cu_tokens, lengths, table, table_width,
                            table_width if table_stride is None else table_stride)


def rope_frequencies(rot_dim, base=10000.0, factor=1.0, scaling=None, context=None, low=1.0, high=32.0):
    """(inv_freq f64[rot_dim / 2], magnitude) for rope().  scaling=None: base^(-2i / rot_dim).  For a
    context `factor` times as long: "linear" divides every frequency by factor; "base" raises the base to
    base * factor^(rot_dim / (rot_dim - 2)), which leaves the fastest pair and slows the slowest by factor;
    "parts" goes by the turns that a pair makes in the `context` tokens of the unscaled model: over `high`
    it stays, under `low` it is divided by factor, between them it is blended, and magnitude is
    0.1 ln(factor) + 1."""
    import numpy as np
    if rot_dim < 2 or rot_dim % 2 or base <= 0 or factor <= 0:
        raise ValueError("rope_frequencies: rot_dim even and positive, base and factor positive")
    if scaling == "base":
        if rot_dim < 4:
            raise ValueError("rope_frequencies: scaling='base' needs rot_dim of 4 or more")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = float(base) ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
    if scaling in (None, "base"):
        return freq, 1.0
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling != "parts" or not context or high <= low:
        raise ValueError("rope_frequencies: scaling is None, 'linear', 'base' or 'parts' (with context, low < high)")
    keep = np.clip((context * freq / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
    return freq * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0


def rope(x, out, tokens, positions, inv_freq, rot_dim, interleaved=False, magnitude=1.0, stream=None):
    """Turns the first rot_dim values of every head of x (heads()) by its token's position into out (may be x).
    positions: device i64 [tokens]; inv_freq: device f64 [rot_dim / 2] (rope_frequencies)."""
    check(lib().cn_rope(x, out, tokens, positions, inv_freq, rot_dim, int(interleaved), magnitude, stream), "cn_rope")


def kv_write(cache, batch, k, v, tokens, stream=None):
    """Writes the new tokens' rows into the cache (8 bits: quantised row by row)."""
    check(lib().cn_kv_write(cache, batch, k, v, tokens, stream), "cn_kv_write")


def kv_read(cache, batch, k_out, v_out, tokens, stream=None):
    """Reads the new tokens' rows back from the cache."""
    check(lib().cn_kv_read(cache, batch, k_out, v_out, tokens, stream), "cn_kv_read")


def paged_attention_workspace(cache, batch, q, tokens):
    """Bytes of device memory that paged_attention needs for these sizes."""
    n = ctypes.c_size_t(0)
    check(lib().cn_paged_attention_workspace(cache, batch, q, tokens, ctypes.byref(n)), "cn_paged_attention_workspace")
    return n.value


def paged_attention(cache, batch, q, out, tokens, scale, causal, window, workspace, workspace_bytes, stream=None):
    """out[i] = softmax over the visible keys of (scale * q[i] . k) times v, for the batch's new tokens."""
    check(lib().cn_paged_attention(cache, batch, q, out, tokens, scale, int(causal), int(window), workspace,
                                   workspace_bytes, stream), "cn_paged_attention")


def synchronize(device=0):
    check(lib().cn_device_synchronize(device), "cn_device_synchronize")


def device_error():
    c = ctypes.c_int(0)
    check(lib().cn_device_error(ctypes.byref(c)), "cn_device_error")
    return c.value
