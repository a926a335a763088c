"""Rotary positions, the paged K/V cache and the attention over it, against their formulas in 64 bits.

Tolerances are counted from the formulas.  u(t) = finfo(t).eps / 2 is the largest relative error of one rounding to
type t of a normal number; below smallest_normal the type's numbers are smallest_normal * eps apart, so a rounding there
is off by half of that, tiny(t), in absolute terms (f16: 2^-14 * 2^-10 / 2 = 2^-25); every output is rounded once, and what comes before it is held in f32 (u32 = 2^-24):

* rope: cos and sin are f32 (sincospif is within 2 ulp, the angle's turns are rounded once: pi * u32 absolute), then
  two products and a sum: |error| <= u(t) |out| + tiny(t) + 8 u32 (|a| + |b|) |magnitude|.
* kv_write / kv_read: exact but for the one rounding, so codes and values are equal to the formula's.
* attention: a score is a sum of dim products in f32, |ds| <= (dim + 4) u32 S with S = scale * sum |q k|; a weight is
  off by a factor within 2 ds (its own score's and the maximum's error), 2^-21 of exp2 and n u32 of the sum; it enters
  the product with V rounded to 16 bits, u(16) of itself, or 2^-25 of the largest contribution where it is so small
  that f16 has no normal number for it (the running maximum is a weight of 1).
"""
import ctypes
import math

import numpy as np
import pytest

from chestnut_b200 import _lib, kernels

torch = pytest.importorskip("torch")

CN_ERR_ARG = -2
U32 = 2.0 ** -24
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def u(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2


def tiny(dtype):
    t = torch.finfo(TYPES[dtype])
    return t.smallest_normal * t.eps / 2


# ------------------------------------------------------------------ plain forms (numpy / torch on the CPU, 64 bits)


def e4m3_values():
    """The 127 finite values from 0 to 448, in the order of their codes."""
    c = np.arange(127)
    return np.where(c < 8, (c % 8) / 8 * 2.0 ** -6, (1 + (c % 8) / 8) * 2.0 ** (c // 8 - 7.0))


def quantise(x):
    """f64 [..., dim] -> (codes u8, exponent bytes u8), by the definition."""
    val = e4m3_values()
    a = np.abs(x)
    fin = np.where(np.isfinite(a), a, 0.0)
    amax = fin.max(-1, keepdims=True)
    e = np.full(amax.shape, -48)
    for k in range(-48, 48):
        e = np.where(amax > 448.0 * 2.0 ** k, k + 1, e)
    e = np.where(amax == 0, 0, e)
    y = np.minimum(fin * 2.0 ** -e.astype(float), 448.0)
    hi = np.clip(np.searchsorted(val, y), 0, 126)
    lo = np.clip(hi - 1, 0, 126)
    up, down = val[hi] - y, y - val[lo]
    code = np.where(up < down, hi, np.where(up > down, lo, np.where(hi % 2 == 0, hi, lo)))
    code = np.where(val[hi] == y, hi, code)
    code = np.where(np.isfinite(x), code, 0x7f) | (np.signbit(x).astype(int) << 7)
    return code.astype(np.uint8), (e[..., 0] + 127).astype(np.uint8)


def expand(codes, exps):
    val = np.append(e4m3_values(), np.nan)
    v = val[codes & 0x7f] * np.where(codes & 0x80, -1.0, 1.0)
    return v * 2.0 ** (exps.astype(float) - 127)[..., None]


def attention(q, k, v, pos, length, scale, causal, window):
    """One sequence in f64: q [n, hq, d], k, v [length, hk, d].  Returns (out, bound parts)."""
    n, hq, d = q.shape
    hk = k.shape[1]
    out, wv, err, small = (np.zeros((n, hq, d)) for _ in range(4))
    for i in range(n):
        hi = min(length, pos[i] + 1) if causal else (length if pos[i] >= 0 else 0)
        lo = max(0, pos[i] - window + 1) if window else 0
        if hi <= lo:
            continue
        for h in range(hq):
            kk, vv = k[lo:hi, h // (hq // hk)], v[lo:hi, h // (hq // hk)]
            s = kk @ q[i, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            big = (np.abs(kk) @ np.abs(q[i, h]) * abs(scale)).max()
            out[i, h] = w @ vv
            wv[i, h] = w @ np.abs(vv)
            err[i, h] = 2 * (d + 4) * U32 * big + 2.0 ** -21 + (hi - lo) * U32
            small[i, h] = 2 * (hi - lo) * 2.0 ** -25 * (w * np.abs(vv).max(-1)).max()
    return out, wv, err, small


# ------------------------------------------------------------------ CPU: refusals, formulas


def _heads(ptr=0x10000, dtype="f16", h=8, d=64, ts=None, hs=None):
    return kernels.heads(ptr, dtype, h, d, ts, hs)


def _cache(dtype="f16", pages=4, page=16, h=8, d=64, exps=None, **kw):
    e = dtype == "e4m3" if exps is None else exps
    return kernels.kv_cache(kw.get("k", 0x20000), kw.get("v", 0x30000), dtype, pages, page, h, d,
                            *([0x40000, 0x50000] if e else []))


def _batch(n=2, width=4, cu=0x60000, lens=0x70000, table=0x80000, stride=None):
    return kernels.kv_batch(n, cu, lens, table, width, stride)


@pytest.mark.parametrize("args", [
    dict(x=_heads(dtype="f32", d=64), out=_heads(d=64)),                     # types differ
    dict(out=_heads(h=7)), dict(out=_heads(d=128)),                          # shapes differ
    dict(rot=0), dict(rot=7), dict(rot=66), dict(rot=-2),                    # rot_dim
    dict(x=_heads(ptr=0)), dict(out=_heads(ptr=None)), dict(pos=None), dict(freq=None),
    dict(pos=0x10004), dict(freq=0x10004),                                   # 8-byte alignment
    dict(x=_heads(ptr=0x10008)), dict(x=_heads(ts=513)), dict(x=_heads(hs=68)), dict(x=_heads(ts=-512)),
    dict(out=_heads(ts=0)), dict(out=_heads(hs=0)), dict(out=_heads(ts=256)),  # rows of out overlap
    dict(x=_heads(d=60), out=_heads(d=60)), dict(x=_heads(d=264), out=_heads(d=264)),
    dict(x=_heads(h=0), out=_heads(h=0)), dict(tokens=-1), dict(tokens=1 << 31),
    dict(out=_heads(ptr=0x10000, ts=1024)),                                  # in place with other strides
    dict(x=kernels._lib.cn_heads(0x10000, 3, 8, 64, 512, 64), out=kernels._lib.cn_heads(0x10000, 3, 8, 64, 512, 64)),
])
def test_rope_refuses(args):
    a = dict(x=_heads(), out=_heads(ptr=0x90000), tokens=16, pos=0x20000, freq=0x30000, rot=64) | args
    rc = _lib.lib().cn_rope(a["x"], a["out"], a["tokens"], a["pos"], a["freq"], a["rot"], 0, 1.0, None)
    assert rc == CN_ERR_ARG and _lib.lib().cn_last_error().startswith(b"cn_rope")


CACHE_FAULTS = [
    dict(cache=_cache("f32")), dict(cache=_cache(k=None)), dict(cache=_cache(v=0)), dict(cache=_cache(k=0x20008)),
    dict(cache=_cache("e4m3", exps=False)), dict(cache=_cache("f16", exps=True)),
    dict(cache=_cache(page=8)), dict(cache=_cache(page=48)), dict(cache=_cache(page=512)), dict(cache=_cache(pages=0)),
    dict(cache=_cache(d=96)), dict(cache=_cache(h=0)),
    dict(batch=_batch(n=-1)), dict(batch=_batch(n=65536)), dict(batch=_batch(cu=None)), dict(batch=_batch(lens=None)),
    dict(batch=_batch(table=None)), dict(batch=_batch(width=-1)), dict(batch=_batch(stride=-1)),
    dict(batch=_batch(width=1 << 27)),
]


@pytest.mark.parametrize("args", CACHE_FAULTS + [
    dict(k=_heads(h=4)), dict(v=_heads(d=128)), dict(k=_heads(dtype="bf16")), dict(k=_heads(dtype="f32"), v=_heads(dtype="f32")),
    dict(k=_heads(dtype="bf16"), v=_heads(dtype="bf16")), dict(k=_heads(ptr=None)), dict(tokens=-1),
    dict(tokens=1 << 31), dict(v=_heads(ptr=0x10008)), dict(v=_heads(hs=63)),
])
@pytest.mark.parametrize("name", ["cn_kv_write", "cn_kv_read"])
def test_kv_refuses(name, args):
    a = dict(cache=_cache(), batch=_batch(), k=_heads(), v=_heads(ptr=0x90000), tokens=16) | args
    rc = getattr(_lib.lib(), name)(a["cache"], a["batch"], a["k"], a["v"], a["tokens"], None)
    assert rc == CN_ERR_ARG and _lib.lib().cn_last_error().startswith(name.encode())


def test_kv_read_refuses_overlapping_outputs():
    rc = _lib.lib().cn_kv_read(_cache(), _batch(), _heads(), _heads(ptr=0x90000, ts=64), 16, None)
    assert rc == CN_ERR_ARG and b"overlap" in _lib.lib().cn_last_error()


@pytest.mark.parametrize("args", CACHE_FAULTS + [
    dict(q=_heads(h=12)), dict(q=_heads(h=4)), dict(q=_heads(d=128), out=_heads(d=128)), dict(out=_heads(h=16)),
    dict(q=_heads(dtype="bf16"), out=_heads(dtype="bf16")), dict(q=_heads(dtype="f32"), out=_heads(dtype="f32")),
    dict(out=_heads(dtype="bf16")), dict(window=-1), dict(window=4, causal=0), dict(out=_heads(ts=64)),
    dict(q=_heads(h=1032), out=_heads(h=1032)), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan),
    dict(work=None), dict(work=0xa0010), dict(bytes=1000), dict(tokens=-1), dict(tokens=(1 << 30) + 1),
])
def test_attention_refuses(args):
    a = dict(cache=_cache(), batch=_batch(), q=_heads(), out=_heads(ptr=0x90000), tokens=16, causal=1, window=0,
             work=0xa0000, bytes=1 << 40, scale=0.125) | args
    rc = _lib.lib().cn_paged_attention(a["cache"], a["batch"], a["q"], a["out"], a["tokens"], a["scale"], a["causal"],
                                       a["window"], a["work"], a["bytes"], None)
    assert rc == CN_ERR_ARG and _lib.lib().cn_last_error().startswith(b"cn_paged_attention")


def test_missing_descriptors_are_refused():
    L = _lib.lib()
    assert L.cn_rope(None, None, 1, 8, 8, 64, 0, 1.0, None) == CN_ERR_ARG
    assert L.cn_kv_write(None, None, None, None, 1, None) == CN_ERR_ARG
    assert L.cn_kv_read(_cache(), None, _heads(), _heads(), 1, None) == CN_ERR_ARG
    assert L.cn_paged_attention(_cache(), _batch(), None, None, 1, 1.0, 0, 0, None, 0, None) == CN_ERR_ARG
    assert L.cn_paged_attention_workspace(_cache(), _batch(), _heads(), 4, None) == CN_ERR_ARG
    n = ctypes.c_size_t()
    assert L.cn_paged_attention_workspace(_cache(), _batch(), _heads(h=12), 4, ctypes.byref(n)) == CN_ERR_ARG
    assert L.cn_paged_attention_workspace(_cache(), _batch(), _heads(), 4, ctypes.byref(n)) == 0 and n.value > 0


def test_nothing_to_do_is_no_error():
    """No tokens or no sequences: returns at once, without a GPU."""
    L = _lib.lib()
    assert L.cn_rope(_heads(), _heads(), 0, 0x20000, 0x30000, 64, 0, 1.0, None) == 0
    assert L.cn_kv_write(_cache(), _batch(), _heads(), _heads(), 0, None) == 0
    assert L.cn_kv_write(_cache(), _batch(n=0, cu=None, lens=None, table=None), _heads(), _heads(), 5, None) == 0
    assert L.cn_paged_attention(_cache(), _batch(), _heads(), _heads(), 0, 1.0, 0, 0, None, 0, None) == 0


def test_rope_frequencies():
    f, m = kernels.rope_frequencies(8, base=100.0)
    assert np.allclose(f, [1, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-15) and m == 1.0
    g, m = kernels.rope_frequencies(8, base=100.0, factor=4.0, scaling="linear")
    assert np.allclose(g, f / 4, rtol=1e-15) and m == 1.0
    g, m = kernels.rope_frequencies(8, base=100.0, factor=4.0, scaling="base")
    assert g[0] == 1.0 and math.isclose(g[-1], f[-1] / 4, rel_tol=1e-12) and m == 1.0
    g, m = kernels.rope_frequencies(64, factor=4.0, scaling="parts", context=4096)
    f, _ = kernels.rope_frequencies(64)
    turns = 4096 * f / (2 * math.pi)
    assert np.array_equal(g[turns >= 32], f[turns >= 32]) and np.allclose(g[turns <= 1], f[turns <= 1] / 4)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and np.all(g[mid] < f[mid]) and np.all(g[mid] > f[mid] / 4)
    assert math.isclose(m, 0.1 * math.log(4) + 1)
    for bad in (dict(rot_dim=7), dict(rot_dim=8, scaling="other"), dict(rot_dim=8, scaling="parts"),
                dict(rot_dim=2, scaling="base"), dict(rot_dim=8, factor=0.0)):
        with pytest.raises(ValueError):
            kernels.rope_frequencies(**bad)


def test_the_quantisers_definition():
    """Hand-worked rows of the 64-bit form that the kernels are held to."""
    codes, exps = quantise(np.array([[448.0, 1.0, -0.5, 0.0], [449.0, 448.0, 2.0, 0.0], [0.0, 0.0, -0.0, 0.0],
                                     [np.inf, 3.5, np.nan, -1.0]]))
    assert exps.tolist() == [127, 128, 127, 127 - 7]
    val = expand(codes, exps)
    assert val[0].tolist() == [448, 1, -0.5, 0] and val[1, 1] == 448 and val[1, 0] == 448  # 224.5 -> 224 * 2
    assert np.isnan(val[3, 0]) and np.isnan(val[3, 2]) and val[3, 1] == 3.5 and val[3, 3] == -1


# ------------------------------------------------------------------ GPU

gpu = pytest.mark.gpu


def handle(t, dtype):
    return kernels.heads(t.data_ptr(), dtype, t.shape[1], t.shape[2], t.stride(0), t.stride(1))


def stream():
    return torch.cuda.current_stream().cuda_stream


@gpu
@pytest.mark.parametrize("tokens,h,dim,rot,inter,dtype", [
    (1, 1, 64, 64, False, "f16"), (64, 32, 128, 128, False, "f16"), (64, 32, 128, 128, True, "f16"),
    (7, 3, 64, 64, True, "bf16"), (5, 5, 128, 64, False, "bf16"), (5, 2, 128, 56, False, "f16"),
    (9, 4, 128, 54, False, "f16"), (9, 4, 64, 52, False, "bf16"), (9, 4, 64, 30, True, "bf16"),
    (3, 2, 64, 2, False, "f32"), (3, 2, 64, 2, True, "f32"), (17, 5, 256, 256, False, "f32"),
    (17, 5, 8, 8, True, "f32"), (33, 6, 128, 44, False, "f32"), (5000, 3, 64, 64, False, "f16"),
    (4099, 2, 128, 96, True, "bf16"),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_rope_against_64_bits(tokens, h, dim, rot, inter, dtype, in_place):
    g = torch.Generator().manual_seed(tokens * 131 + rot)
    x = torch.randn(tokens, h + 2, dim, generator=g).to(TYPES[dtype])
    pos = torch.randint(-1000, 2000000, (tokens,), generator=g)
    pos[0] = 0 if tokens == 1 else 2000003
    freq, mag = kernels.rope_frequencies(rot, factor=8.0, scaling="parts", context=4096)
    d = x.cuda()
    view = d[:, 1:1 + h]                                    # heads inside a wider row
    out = view if in_place else torch.full((h, tokens, dim), 7.0, device="cuda", dtype=TYPES[dtype]).transpose(0, 1)
    d_pos, d_freq = pos.cuda(), torch.from_numpy(freq).cuda()
    kernels.rope(handle(view, dtype), handle(out, dtype), tokens, d_pos.data_ptr(), d_freq.data_ptr(), rot, inter, mag,
                 stream())
    torch.cuda.synchronize()
    got = out.cpu().double().numpy()
    ref = x[:, 1:1 + h].double().numpy().copy()
    ang = pos.double().numpy()[:, None, None] * freq
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    xa, xb = ref[..., a].copy(), ref[..., b].copy()
    ref[..., a] = mag * (xa * np.cos(ang) - xb * np.sin(ang))
    ref[..., b] = mag * (xb * np.cos(ang) + xa * np.sin(ang))
    tol = u(dtype) * np.abs(ref) + tiny(dtype)
    slop = 8 * U32 * mag * (np.abs(xa) + np.abs(xb))
    tol[..., a] += slop
    tol[..., b] += slop
    assert np.all(np.abs(got - ref) <= tol), np.max(np.abs(got - ref) - tol)
    assert np.array_equal(got[..., rot:], ref[..., rot:])
    assert torch.equal(d[:, 0].cpu(), x[:, 0]) and torch.equal(d[:, 1 + h].cpu(), x[:, 1 + h])  # the heads beside them
    assert in_place or torch.equal(d.cpu(), x)


def make(dtype, cache, dim, page, hk, group, new, past, seed=0, spare=3, fill=float("nan"), tail_rows=2):
    """Random sequences in a cache whose unused places hold `fill`.  Everything on the CPU and on the GPU."""
    g = torch.Generator().manual_seed(seed + 7 * len(new) + dim + page)
    n = len(new)
    length = [a + b for a, b in zip(new, past)]
    used = [max(0, -(-v // page)) for v in length]
    width = max(max(used), 1)
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((n, width + 1), -5, dtype=torch.int32)       # entries that no sequence uses name no page
    for s in range(n):
        for i in range(used[s]):
            table[s, i] = order.pop()
    st = dict(dtype=dtype, cache=cache, dim=dim, page=page, hk=hk, group=group, new=new, past=past, length=length,
              total=sum(new), width=width, pages=pages, table=table)
    rows = sum(new) + tail_rows
    st["qkv"] = torch.randn(rows, hk * group + 2 * hk, dim, generator=g).to(TYPES[dtype])
    st["ctx"] = {}
    for name in "kv":
        body = torch.full((pages, hk, page, dim), fill).to(TYPES[dtype] if cache != "e4m3" else torch.float32)
        exps = None
        if cache == "e4m3":
            codes = np.full(body.shape, 0x7f if math.isnan(fill) else 0, np.uint8)
            exps = np.full(body.shape[:3], 127, np.uint8)
        ctx = []
        for s in range(n):
            L = max(length[s], 0)
            x = torch.randn(L, hk, dim, generator=g) * (0.25 + 4 * torch.rand(L, hk, 1, generator=g) ** 4)
            if cache == "e4m3":
                c, e = quantise(x.double().numpy())
                for p in range(L):
                    codes[table[s, p // page], :, p % page] = c[p]
                    exps[table[s, p // page], :, p % page] = e[p]
                ctx.append(expand(c, e))
            else:
                x = x.to(TYPES[dtype])
                for p in range(L):
                    body[table[s, p // page], :, p % page] = x[p]
                ctx.append(x.double().numpy())
        st["ctx"][name] = ctx
        st[name] = (torch.from_numpy(codes) if cache == "e4m3" else body).cuda()
        st[name + "_exp"] = torch.from_numpy(exps).cuda() if exps is not None else None
    st["d_table"] = table.cuda()
    st["d_cu"] = torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32).cuda()
    st["d_len"] = torch.tensor(length, dtype=torch.int32).cuda()
    st["d_qkv"] = st["qkv"].cuda()
    return st


def descriptors(st):
    exps = [t.data_ptr() for t in (st["k_exp"], st["v_exp"])] if st["cache"] == "e4m3" else []
    return (kernels.kv_cache(st["k"].data_ptr(), st["v"].data_ptr(), st["cache"], st["pages"], st["page"], st["hk"],
                             st["dim"], *exps),
            kernels.kv_batch(len(st["new"]), st["d_cu"].data_ptr(), st["d_len"].data_ptr(), st["d_table"].data_ptr(),
                             st["width"], st["d_table"].shape[1]))


def attend(st, out=None, causal=True, window=0, scale=None, work=None):
    cache, batch = descriptors(st)
    hq = st["hk"] * st["group"]
    q = st["d_qkv"][:, :hq]
    if out is None:
        out = torch.full((q.shape[0], hq, st["dim"]), 7.0, device="cuda", dtype=q.dtype)
    h = handle(q, st["dtype"])
    nb = kernels.paged_attention_workspace(cache, batch, h, q.shape[0])
    if work is None:
        work = torch.full((max(nb, 1),), 0xff, device="cuda", dtype=torch.uint8)  # its content is of no matter
    kernels.paged_attention(cache, batch, h, handle(out, st["dtype"]), q.shape[0],
                            st["dim"] ** -0.5 if scale is None else scale, causal, window, work.data_ptr(), nb, stream())
    return out


def check_attention(st, out, causal=True, window=0, scale=None, ctx=None):
    scale = st["dim"] ** -0.5 if scale is None else scale
    got = out.cpu().double().numpy()
    hq = st["hk"] * st["group"]
    row = 0
    ctx = ctx or st["ctx"]
    for s, (n, p) in enumerate(zip(st["new"], st["past"])):
        q = st["qkv"][row:row + n, :hq].double().numpy()
        ref, wv, err, small = attention(q, ctx["k"][s], ctx["v"][s], p + np.arange(n), max(p + n, 0), scale, causal, window)
        tol = tiny(st["dtype"]) + u(st["dtype"]) * np.abs(ref) + (u("f16" if st["cache"] == "e4m3" else st["dtype"]) + err) * wv + small
        bad = ~(np.abs(got[row:row + n] - ref) <= tol * (1 + u(st["dtype"])))
        assert not bad.any(), (s, np.argwhere(bad)[:4].tolist(), got[row:row + n][bad][:4], ref[bad][:4], tol[bad][:4])
        row += n
    assert np.all(got[row:] == 7.0)  # rows behind the last sequence


SHAPES = [
    # dtype, cache, dim, page, cache heads, group, new, past, causal, window
    ("f16", "f16", 64, 16, 1, 1, [1], [0], True, 0),
    ("f16", "f16", 128, 16, 2, 1, [1], [1000], True, 0),
    ("bf16", "bf16", 128, 64, 2, 4, [1, 1, 1, 1], [50, 0, 1, 700], True, 0),
    ("f16", "e4m3", 128, 32, 2, 1, [1, 3, 4, 2], [1200, 63, 64, 65], True, 0),
    ("bf16", "e4m3", 128, 64, 2, 2, [1, 5], [129, 300], True, 0),
    ("bf16", "e4m3", 64, 16, 3, 5, [2, 1], [31, 400], True, 0),
    ("f16", "e4m3", 64, 128, 2, 3, [5, 1, 40], [0, 500, 90], True, 33),
    ("f16", "f16", 128, 64, 2, 1, [64, 64], [640, 0], False, 0),
    ("bf16", "bf16", 64, 32, 1, 8, [33, 1, 17], [15, 260, 16], True, 0),
    ("f16", "f16", 64, 16, 2, 7, [1, 0, 3, 0], [100, 40, 0, 0], True, 0),
    ("bf16", "bf16", 128, 256, 1, 1, [300], [0], True, 0),
    ("f16", "f16", 128, 16, 1, 2, [200], [57], True, 100),
    ("bf16", "e4m3", 128, 16, 1, 3, [130], [200], False, 0),
    ("f16", "f16", 64, 64, 1, 1, [4, 1], [300, 0], True, 1),
    ("f16", "e4m3", 128, 64, 1, 16, [1, 20], [2049, 111], True, 700),
    ("bf16", "bf16", 64, 16, 2, 1, [5, 6], [-3, -6], True, 0),          # tokens before position 0 see nothing
    ("f16", "f16", 128, 16, 1, 1, [5, 2], [-3, -2], False, 0),
    ("f16", "e4m3", 64, 16, 2, 2, [257, 129, 1], [0, 127, 3000], True, 0),
]


@gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:6])) + f"-{s[6]}+{s[7]}".replace(" ", ""))
def test_attention_against_64_bits(shape):
    dtype, cache, dim, page, hk, group, new, past, causal, window = shape
    st = make(dtype, cache, dim, page, hk, group, new, past)
    out = attend(st, causal=causal, window=window)
    check_attention(st, out, causal, window)
    assert kernels.device_error() == 0
    again = attend(st, causal=causal, window=window)
    assert torch.equal(out, again)


LARGE = [
    # dtype, cache, dim, page, cache heads, group, new, past, causal, window
    ("bf16", "bf16", 128, 64, 2, 3, [700, 64, 1, 0, 17], [0, 3000, 5000, 10, 900], True, 0),  # both kernels, one merge
    ("f16", "f16", 128, 16, 1, 1, [64], [20000], False, 0),        # one tile of one half over every CTA
    ("f16", "f16", 128, 256, 1, 1, [1], [30000], True, 0),         # one row in hundreds of parts
    ("f16", "e4m3", 64, 32, 1, 2, [1, 2], [40000, 3], True, 0),
    ("f16", "e4m3", 64, 128, 2, 3, [1500, 300], [0, 2000], True, 333),
    ("bf16", "e4m3", 128, 64, 1, 4, [513], [1111], True, 0),
    ("bf16", "bf16", 64, 64, 1, 128, [1, 3], [700, 40], True, 0),  # the largest group
    ("f16", "f16", 64, 16, 1, 40, [1, 1, 9], [5000, 0, 77], True, 0),
    ("f16", "e4m3", 128, 16, 2, 20, [2, 1], [300, 4000], True, 1000),
    ("f16", "f16", 128, 128, 4, 1, [2048], [0], True, 0),
    ("bf16", "bf16", 64, 32, 3, 5, [255, 256, 257], [129, 127, 128], True, 128),
    ("f16", "f16", 128, 64, 1, 1, [129, 128, 127, 1], [640, 64, 0, 0], False, 0),
    ("f16", "f16", 64, 16, 2, 2, [1] * 300 + [40], list(range(300)) + [1000], True, 0),
    # tiles of one half over several blocks of keys an SM, each cache and dim
    ("f16", "e4m3", 128, 64, 4, 3, list(range(17, 42)), [459] * 25, True, 0),
    ("bf16", "e4m3", 128, 16, 8, 1, [40] * 16, [900 + 61 * i for i in range(16)], False, 0),
    ("bf16", "bf16", 128, 64, 4, 3, list(range(17, 42)), [459] * 25, True, 0),
    ("f16", "e4m3", 64, 64, 8, 3, list(range(17, 42)), [1459] * 25, True, 700),
    ("f16", "f16", 64, 64, 8, 3, list(range(17, 42)), [1459] * 25, True, 0),
    # many blocks at the edge one after the other, of all stages
    ("f16", "f16", 64, 32, 4, 3, [701, 5, 300, 64, 400], [0, 5000, 2000, 700, 3000], True, 500),
    ("bf16", "bf16", 128, 32, 4, 1, [701, 5, 300, 64, 400], [0, 5000, 2000, 700, 3000], True, 300),
    ("f16", "f16", 128, 16, 4, 2, [500, 130, 257], [0, 1000, 5], True, 120),
    ("f16", "f16", 64, 64, 8, 1, [900, 33], [50, 700], True, 64),
]


@gpu
@pytest.mark.parametrize("shape", LARGE, ids=lambda s: "-".join(map(str, s[:6])) + f"-{len(s[6])}seqs-{max(s[6])}-{max(s[7])}")
def test_attention_over_long_contexts(shape):
    """Cut tiles, merges, halves that share a tile's keys: against 64 bits on the GPU, sequence by sequence."""
    dtype, cache, dim, page, hk, group, new, past, causal, window = shape
    g = torch.Generator(device="cuda").manual_seed(7)
    n, hq = len(new), hk * group
    length = [a + b for a, b in zip(new, past)]
    used = [-(-v // page) for v in length]
    pages, width = sum(used) + 2, max(used)
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s in range(n):
        table[s, : used[s]] = order[at:at + used[s]]
        at += used[s]
    body, exps, wide = {}, {}, {}
    for m in "kv":
        x = torch.randn(pages, hk, page, dim, generator=g, device="cuda") * (0.3 + 3 * torch.rand(pages, hk, page, 1, generator=g, device="cuda") ** 3)
        if cache == "e4m3":
            part, e = torch.frexp(x.abs().amax(-1))
            e = e - 9 + (part > 0.875).int()
            power = lambda k: ((k + 127) << 23).view(torch.float32)[..., None]  # noqa: E731
            codes = (x * power(-e)).to(torch.float8_e4m3fn)
            wide[m] = codes.double() * power(e).double()
            body[m], exps[m] = codes.view(torch.uint8), (e + 127).to(torch.uint8)
        else:
            body[m], exps[m] = x.to(TYPES[dtype]), None
            wide[m] = body[m].double()
    q = torch.randn(sum(new) + 1, hq, dim, generator=g, device="cuda").to(TYPES[dtype])
    st = dict(dtype=dtype, cache=cache, dim=dim, page=page, hk=hk, group=group, new=new, past=past, pages=pages, width=width,
              k=body["k"], v=body["v"], k_exp=exps["k"], v_exp=exps["v"], d_table=table, d_qkv=q,
              d_cu=torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32).cuda(), d_len=torch.tensor(length, dtype=torch.int32).cuda())
    out = attend(st, causal=causal, window=window)
    assert kernels.device_error() == 0
    assert torch.equal(out, attend(st, causal=causal, window=window))
    row = 0
    for s in range(n):
        keys = torch.arange(length[s], device="cuda")
        k, v = (wide[m][table[s].long()[keys // page], :, keys % page] for m in "kv")  # [keys, hk, dim]
        pos = past[s] + torch.arange(new[s], device="cuda")[:, None]
        for h in range(hq):
            kk, vv = k[:, h // group], v[:, h // group]
            qq = q[row:row + new[s], h].double()
            a = qq @ kk.T * dim ** -0.5
            if causal:
                a[keys > pos] = -math.inf
            if window:
                a[keys <= pos - window] = -math.inf
            w = torch.softmax(a, -1)
            big = (qq.abs() @ kk.abs().T * dim ** -0.5).amax(-1, keepdim=True)
            err = 2 * (dim + 4) * U32 * big + 2.0 ** -21 + length[s] * U32
            tol = tiny(dtype) + u(dtype) * (w @ vv).abs() + (u("f16" if cache == "e4m3" else dtype) + err) * (w @ vv.abs()) \
                + 2 * length[s] * 2.0 ** -25 * (w * vv.abs().amax(-1)).amax(-1, keepdim=True)
            off = (out[row:row + new[s], h].double() - w @ vv).abs() - tol * (1 + u(dtype))
            assert new[s] == 0 or off.max() <= 0, (s, h, off.max())
        row += new[s]
    assert torch.all(out[row:] == 7.0)


@gpu
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_attention_many_sequences_and_scale(cache):
    """More sequences than a block has threads, lengths from none to a few pages, another scale."""
    n = 1100
    new = [(s * 7) % 3 for s in range(n)]
    past = [(s * 37) % 90 for s in range(n)]
    st = make("f16", cache, 64, 16, 1, 2, new, past)
    check_attention(st, attend(st, scale=0.5), scale=0.5)


@gpu
@pytest.mark.parametrize("dtype,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3")])
@pytest.mark.parametrize("new,past,window", [([4], [40], 0), ([3, 2], [30, 200], 20), ([150], [20], 0), ([90], [200], 64)])
def test_what_a_row_does_not_see_has_no_influence(dtype, cache, new, past, window):
    """NaN and infinities in later tokens, and in front of the window, stay out of the rows that do not see them;
    rows that do see them are not finite."""
    st = make(dtype, cache, 64, 16, 2, 2, new, past)
    L, n = st["length"][0], new[0]
    for p, x in ((L - 1, math.nan), (L - 2, math.inf)):
        at, r = int(st["table"][0, p // 16]), p % 16
        for name in "kv":
            if cache == "e4m3":
                st[name][at, :, r, 5] = 0x7f
            else:
                st[name][at, :, r, 5] = x
            st["ctx"][name][0][p, :, 5] = math.nan
    if window:
        for p in range(0, max(0, past[0] - window + 1)):  # in front of every row's window
            at, r = int(st["table"][0, p // 16]), p % 16
            st["v"][at, :, r] = 0x7f if cache == "e4m3" else math.inf
            st["k"][at, :, r] = 0x7f if cache == "e4m3" else -math.inf
    out = attend(st, window=window)
    got = out.cpu().double().numpy()
    assert not np.isfinite(got[n - 1]).any()
    clean = dict(st, new=[n - 2] + new[1:], past=past)  # the rows that see neither
    q = st["qkv"]
    rows = list(range(n - 2)) + list(range(n, sum(new)))
    sub = dict(clean, qkv=q[rows])
    with np.errstate(invalid="ignore"):
        check_attention(sub, torch.cat([out[rows], torch.full_like(out[:1], 7.0)]), window=window,
                        ctx={m: [c[: st["length"][s] - (2 if s == 0 else 0)] for s, c in enumerate(st["ctx"][m])] for m in "kv"})


@gpu
def test_rows_that_see_a_value_beyond_all_others_get_it():
    """An infinite V in the newest key: rows that see it are infinite in that place alone."""
    st = make("f16", "f16", 64, 16, 1, 1, [3], [20])
    p = st["length"][0] - 1
    st["v"][int(st["table"][0, p // 16]), 0, p % 16, 9] = math.inf
    got = attend(st).cpu()
    assert torch.isfinite(got[:2]).all() and got[2, 0, 9] == math.inf
    rest = [i for i in range(64) if i != 9]
    assert torch.isfinite(got[2, 0, rest]).all()


@gpu
def test_attention_layouts_streams_and_in_place():
    """q as a view of a packed row and out as [heads][tokens][dim]; out = q; another stream than the current one."""
    st = make("bf16", "bf16", 128, 32, 2, 3, [7, 1], [100, 33], tail_rows=0)
    ref = attend(st)
    check_attention(st, ref)
    t = torch.empty(6, 8, 128, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    assert torch.equal(attend(st, out=t), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = attend(st)
    side.synchronize()
    assert torch.equal(other, ref)
    assert torch.equal(attend(st, out=st["d_qkv"][:, :6]), ref)


@gpu
def test_a_captured_step_replays_with_new_lengths():
    """rope, write and attention captured once; the arrays that hold lengths and pages change between replays."""
    hk, group, dim, page = 2, 2, 128, 16
    st = make("f16", "e4m3", dim, page, hk, group, [1, 1, 1], [40, 0, 200], fill=0.0, tail_rows=0)
    full = st["length"]
    freq, _ = kernels.rope_frequencies(dim)
    d_freq, d_pos = torch.from_numpy(freq).cuda(), torch.tensor(full).cuda() - 1
    hq = hk * group
    cache, batch = descriptors(st)
    turned = torch.empty_like(st["d_qkv"])
    out = torch.zeros(3, hq, dim, device="cuda", dtype=torch.float16)
    q = handle(turned[:, :hq], "f16")
    nb = kernels.paged_attention_workspace(cache, batch, q, 3)
    work = torch.empty(nb, device="cuda", dtype=torch.uint8)

    def step():
        turned.copy_(st["d_qkv"])
        kernels.rope(handle(turned[:, :hq + hk], "f16"), handle(turned[:, :hq + hk], "f16"), 3, d_pos.data_ptr(),
                     d_freq.data_ptr(), dim, False, 1.0, stream())
        kernels.kv_write(cache, batch, handle(turned[:, hq:hq + hk], "f16"), handle(turned[:, hq + hk:], "f16"), 3, stream())
        kernels.paged_attention(cache, batch, q, handle(out, "f16"), 3, dim ** -0.5, True, 0, work.data_ptr(), nb, stream())

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens in (full, [20, 1, 199], [33, 1, 64]):
        st["d_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        d_pos.copy_(torch.tensor(lens) - 1)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert replayed.abs().sum() > 0
        out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, replayed)


@gpu
def test_pages_shared_and_repeated():
    """Two sequences with the same first pages, and one whose table names a page twice."""
    st = make("f16", "f16", 64, 16, 1, 2, [1, 1], [70, 70], tail_rows=0)
    st["table"][1, :3] = st["table"][0, :3]
    st["table"][0, 3] = st["table"][0, 1]
    st["d_table"].copy_(st["table"])
    for m in "kv":
        body = st[m].cpu().double().numpy()
        st["ctx"][m] = [np.stack([body[st["table"][s, p // 16], :, p % 16] for p in range(71)]) for s in range(2)]
    check_attention(st, attend(st))


@gpu
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_pages_outside_the_cache_are_reported(cache):
    """A page number outside the cache, and lengths past the table: no access there, the error word says 6."""
    st = make("f16", cache, 64, 16, 1, 1, [1, 1], [70, 20], tail_rows=0)
    ref = attend(st)
    assert kernels.device_error() == 0
    for bad in (-1, st["pages"], 2 ** 31 - 1):
        st["d_table"][0, 2] = bad
        out = attend(st)
        torch.cuda.synchronize()
        assert kernels.device_error() == 6
        assert torch.equal(out[1], ref[1])  # the other sequence
    st["d_table"].copy_(st["table"])
    st["d_len"][0] = 16 * st["width"] + 1
    attend(st)
    torch.cuda.synchronize()
    assert kernels.device_error() == 6
    ks = torch.full((2, 1, 64), 3.0, device="cuda", dtype=torch.float16)
    c, b = descriptors(st)
    before = st["k"].clone()
    kernels.kv_write(c, b, handle(ks, "f16"), handle(ks, "f16"), 2, stream())
    torch.cuda.synchronize()
    assert kernels.device_error() == 6
    changed = (st["k"].view(torch.uint8) != before.view(torch.uint8)).flatten(1).any(1)  # bytes: unused rows are NaN
    changed = changed.nonzero().flatten().tolist()
    assert changed == [int(st["table"][1, 1])]
    kernels.kv_read(c, b, handle(ks, "f16"), handle(ks, "f16"), 2, stream())
    torch.cuda.synchronize()
    assert kernels.device_error() == 6 and torch.all(ks[0] == 0) and torch.all(ks[1] == 3)


def special_rows(dim, dtype):
    """Rows that quantisation can get wrong: zeros, ties, borders of the exponent, extremes, values that are not finite."""
    t = torch.finfo(TYPES[dtype])
    rows = [torch.zeros(dim), -torch.zeros(dim), torch.full((dim,), 448.0), torch.linspace(-448, 448, dim),
            torch.full((dim,), t.max), torch.full((dim,), t.smallest_normal), torch.full((dim,), t.tiny / 4),
            torch.linspace(-t.max, t.max, dim), 2.0 ** -torch.arange(dim).float().clamp(max=40),
            1.0 + torch.arange(dim) / 16, 17.0 + torch.arange(dim) / 2, torch.arange(dim).float() * 3.5]
    for x in (math.inf, -math.inf, math.nan):
        r = torch.randn(dim)
        r[3] = x
        rows.append(r)
    rows.append(torch.full((dim,), math.nan))
    for k in (-20, -3, 0, 5, 7):
        for top in (1.75, 1.7578125, 1.75 - 2.0 ** -7, 1.0):
            r = torch.randn(dim).clamp(-1, 1) * 2.0 ** k
            r[7] = top * 2.0 ** k
            rows.append(r)
    if dtype == "bf16":
        rows += [torch.full((dim,), 1e30), torch.full((dim,), 3.3e38), torch.full((dim,), 1e-30), torch.full((dim,), 1e-40)]
    return torch.stack(rows).to(TYPES[dtype])


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_write_quantises_by_the_definition_and_reads_back(dtype, dim):
    rows = special_rows(dim, dtype)
    n, page, hk = len(rows), 16, 2
    k = torch.stack([rows, rows.flip(0)], 1)
    v = torch.stack([rows.roll(5, 0), -rows], 1)
    st = make(dtype, "e4m3", dim, page, hk, 1, [n], [5], fill=0.0)
    before = {m: st[m].clone() for m in ("k", "v", "k_exp", "v_exp")}
    c, b = descriptors(st)
    dk, dv = k.cuda(), v.cuda()
    kernels.kv_write(c, b, handle(dk, dtype), handle(dv, dtype), n, stream())
    back = [torch.full_like(dk, 9.0) for _ in "kv"]
    kernels.kv_read(c, b, handle(back[0], dtype), handle(back[1], dtype), n, stream())
    torch.cuda.synchronize()
    assert kernels.device_error() == 0
    for m, x, got in (("k", k, back[0]), ("v", v, back[1])):
        want_c, want_e = quantise(x.double().numpy())
        body, exps = before[m].cpu().numpy(), before[m + "_exp"].cpu().numpy()
        for i in range(n):
            p = 5 + i
            body[st["table"][0, p // page], :, p % page] = want_c[i]
            exps[st["table"][0, p // page], :, p % page] = want_e[i]
        have = st[m].cpu().numpy()
        zero = lambda z: np.where((z & 0x7f) == 0, 0, np.where((z & 0x7f) == 0x7f, 0x7f, z))  # noqa: E731 (signs of 0 and NaN)
        assert np.array_equal(zero(have), zero(body))
        assert np.array_equal(st[m + "_exp"].cpu().numpy(), exps)
        ref = torch.from_numpy(expand(want_c, want_e)).clamp(-torch.finfo(TYPES[dtype]).max, torch.finfo(TYPES[dtype]).max)
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=1e300), torch.nan_to_num(ref.to(TYPES[dtype]).double(), nan=1e300))


@gpu
@pytest.mark.parametrize("dtype,cache,dim,page,hk,new,past", [
    ("f16", "f16", 64, 16, 3, [5, 0, 1, 40], [0, 9, 31, 15]), ("bf16", "bf16", 128, 256, 1, [300, 1], [0, 0]),
    ("bf16", "e4m3", 64, 32, 5, [31, 2], [1, 64]), ("f16", "e4m3", 128, 64, 2, [2100, 100], [3, 0]),
    ("f16", "f16", 128, 16, 1, [6, 3], [-4, -3]), ("f16", "e4m3", 64, 16, 8, [17000], [0]),
])
def test_write_and_read_places(dtype, cache, dim, page, hk, new, past):
    """Every row lands in its place and nothing else changes; reading gives it back; rows of no sequence and rows
    before position 0 are left alone (reading: zeros)."""
    if sum(new) < 10000:
        st = make(dtype, cache, dim, page, hk, 1, new, past, fill=0.0)
    else:  # many tokens: no random context under them
        st = make(dtype, cache, dim, page, hk, 1, [1], [0], fill=0.0)
        pages = -(-sum(new) // page) + 3
        st |= dict(new=new, past=past, length=[new[0] + past[0]], total=sum(new), pages=pages, width=pages - 3)
        st["table"] = torch.randperm(pages)[None].int()
        st["d_table"], st["d_cu"], st["d_len"] = st["table"].cuda(), torch.tensor([0] + new).int().cuda(), torch.tensor(st["length"]).int().cuda()
        for m in "kv":
            st[m] = torch.zeros(pages, hk, page, dim, dtype=torch.uint8, device="cuda")
            st[m + "_exp"] = torch.full((pages, hk, page), 127, dtype=torch.uint8, device="cuda")
        st["qkv"] = torch.randn(sum(new) + 2, 3 * hk, dim).to(TYPES[dtype])
        st["d_qkv"] = st["qkv"].cuda()
    before = {m: st[m].cpu().clone() for m in "kv"}
    c, b = descriptors(st)
    rows = len(st["qkv"])
    k, v = st["d_qkv"][:, hk:2 * hk], st["d_qkv"][:, 2 * hk:]
    kernels.kv_write(c, b, handle(k, dtype), handle(v, dtype), rows, stream())
    back = torch.full((2, hk, rows, dim), 9.0, device="cuda", dtype=TYPES[dtype]).transpose(1, 2)
    kernels.kv_read(c, b, handle(back[0], dtype), handle(back[1], dtype), rows, stream())
    torch.cuda.synchronize()
    assert kernels.device_error() == 0
    for m, x, got in (("k", st["qkv"][:, hk:2 * hk], back[0].cpu()), ("v", st["qkv"][:, 2 * hk:], back[1].cpu())):
        want, have = before[m], st[m].cpu()
        if cache == "e4m3":
            codes, exps = quantise(x.double().numpy())
            x = torch.from_numpy(expand(codes, exps)).to(TYPES[dtype])
            codes = torch.from_numpy(codes)
        r = 0
        for s in range(len(new)):
            for i in range(new[s]):
                p = past[s] + i
                if p >= 0:
                    want[st["table"][s, p // page], :, p % page] = codes[r] if cache == "e4m3" else x[r]
                    assert torch.equal(got[r], x[r])
                else:
                    assert torch.all(got[r] == 0)
                r += 1
        assert torch.equal(have, want) if cache != "e4m3" else torch.equal(have & ~((have & 0x7f) == 0) * 0x80 | have & 0x7f, want & ~((want & 0x7f) == 0) * 0x80 | want & 0x7f)
        assert torch.all(got[r:] == 9.0)


@gpu
def test_cache_beyond_32_bits():
    """Pages whose values lie more than 2^32 bytes (and 2^31 values) into the cache."""
    dim, page, hk = 128, 64, 4
    pages = (1 << 31) // (hk * page * dim) + 40
    k = torch.zeros(pages, hk, page, dim, device="cuda", dtype=torch.float16)
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(3)
    new, past = [70], [0]
    qkv = torch.randn(70, 3 * hk, dim, generator=g).half()
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    st = dict(dtype="f16", cache="f16", dim=dim, page=page, hk=hk, group=1, new=new, past=past, length=[70], total=70,
              width=2, pages=pages, table=table, qkv=qkv, d_qkv=qkv.cuda(), k=k, v=v, d_table=table.cuda(),
              d_cu=torch.tensor([0, 70], dtype=torch.int32).cuda(), d_len=torch.tensor([70], dtype=torch.int32).cuda())
    c, b = descriptors(st)
    kernels.kv_write(c, b, handle(st["d_qkv"][:, hk:2 * hk], "f16"), handle(st["d_qkv"][:, 2 * hk:], "f16"), 70, stream())
    torch.cuda.synchronize()
    assert torch.equal(k[pages - 1, :, 5].cpu(), qkv[5, hk:2 * hk]) and torch.equal(v[pages - 2, :, 5].cpu(), qkv[69, 2 * hk:])
    ctx = {"k": [qkv[:, hk:2 * hk].double().numpy()], "v": [qkv[:, 2 * hk:].double().numpy()]}
    check_attention(st, attend(st), ctx=ctx)


@gpu
@pytest.mark.parametrize("dtype,cache,dim,page", [("f16", "e4m3", 128, 16), ("bf16", "bf16", 64, 32)])
def test_a_run_of_steps(dtype, cache, dim, page):
    """Clips as they are served: a first prompt, then frames of some tokens and of one, each turned by its positions,
    written and attended; the whole past is checked against the formulas in 64 bits of what was written."""
    hk, group, clips = 2, 2, 3
    hq = hk * group
    freq, _ = kernels.rope_frequencies(dim, factor=2.0, scaling="linear")
    d_freq = torch.from_numpy(freq).cuda()
    pages, width = 40, 12
    g = torch.Generator().manual_seed(5)
    table = torch.randperm(pages, generator=g)[: clips * width].view(clips, width).int()
    shape = (pages, hk, page, dim)
    coded = cache == "e4m3"
    st = dict(dtype=dtype, cache=cache, dim=dim, page=page, hk=hk, group=group, pages=pages, width=width, table=table, d_table=table.cuda())
    for m in "kv":
        st[m] = torch.full(shape, 0x7f, dtype=torch.uint8, device="cuda") if coded else torch.full(shape, math.nan, dtype=TYPES[dtype], device="cuda")
        st[m + "_exp"] = torch.zeros(shape[:3], dtype=torch.uint8, device="cuda") if coded else None
    past = [0] * clips
    ctx = {m: [np.zeros((0, hk, dim)) for _ in range(clips)] for m in "kv"}
    for new in ([20, 1, 33], [1, 1, 1], [4, 0, 17], [1, 1, 1], [0, 64, 2]):
        rows = sum(new)
        x = torch.randn(rows, hq + 2 * hk, dim, generator=g).to(TYPES[dtype])
        d = x.cuda()
        pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)])
        d_pos = pos.cuda()
        length = [n + p for n, p in zip(new, past)]
        st |= dict(new=new, past=list(past), length=length, d_cu=torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32).cuda(),
                   d_len=torch.tensor(length, dtype=torch.int32).cuda(), d_qkv=d)
        c, b = descriptors(st)
        kernels.rope(handle(d[:, :hq + hk], dtype), handle(d[:, :hq + hk], dtype), rows, d_pos.data_ptr(), d_freq.data_ptr(), dim, True, 1.0, stream())
        kernels.kv_write(c, b, handle(d[:, hq:hq + hk], dtype), handle(d[:, hq + hk:], dtype), rows, stream())
        out = attend(st)
        torch.cuda.synchronize()
        turned = d.cpu()
        # the turned rows, by the formula (a rounding apart), and what of them the cache holds
        z = x[:, :hq + hk].double().numpy()
        ang = pos.double().numpy()[:, None, None] * freq
        ref = np.empty_like(z)
        ref[..., 0::2] = z[..., 0::2] * np.cos(ang) - z[..., 1::2] * np.sin(ang)
        ref[..., 1::2] = z[..., 1::2] * np.cos(ang) + z[..., 0::2] * np.sin(ang)
        pair = np.repeat(np.abs(z[..., 0::2]) + np.abs(z[..., 1::2]), 2, -1)
        assert np.all(np.abs(turned[:, :hq + hk].double().numpy() - ref) <= u(dtype) * np.abs(ref) + tiny(dtype) + 8 * U32 * pair)
        st["qkv"] = turned
        r = 0
        for s in range(clips):
            for m, lo in (("k", hq), ("v", hq + hk)):
                y = turned[r:r + new[s], lo:lo + hk].double().numpy()
                ctx[m][s] = np.concatenate([ctx[m][s], expand(*quantise(y)) if coded else y])
            r += new[s]
        check_attention(st, out, ctx=ctx)
        past = length
    assert kernels.device_error() == 0


@gpu
@pytest.mark.parametrize("cache,dtype", [("f16", "f16"), ("e4m3", "bf16")])
def test_rows_before_the_first_sequence_and_repeated_queries(cache, dtype):
    """cu_tokens that begin behind row 0; queries whose tokens are one row in memory (token stride 0)."""
    st = make(dtype, cache, 64, 16, 2, 2, [40, 1], [30, 100], tail_rows=0)
    ref = attend(st)
    check_attention(st, ref)
    st["d_cu"] += 3
    shifted = torch.cat([st["d_qkv"][:3], st["d_qkv"], st["d_qkv"][:2]])
    moved = dict(st, d_qkv=shifted)
    out = attend(moved)
    assert torch.equal(out[3:-2], ref) and torch.all(out[:3] == 7.0) and torch.all(out[-2:] == 7.0)
    st["d_cu"] -= 3
    one = torch.randn(1, 4, 64, device="cuda").to(TYPES[dtype])
    same = dict(st, d_qkv=one.expand(41, 4, 64), qkv=one.expand(41, 4, 64).cpu())
    check_attention(same, attend(same))
    k = torch.full((46, 2, 64), 2.0, device="cuda", dtype=TYPES[dtype])
    st["d_cu"] += 3
    c, b = descriptors(st)
    back = torch.full_like(k, 9.0)
    kernels.kv_write(c, b, handle(k, dtype), handle(k, dtype), 46, stream())
    kernels.kv_read(c, b, handle(back, dtype), handle(back.clone(), dtype), 46, stream())
    assert torch.all(back[3:44] == 2.0) and torch.all(back[:3] == 9.0) and torch.all(back[44:] == 9.0)
    assert kernels.device_error() == 0


@gpu
def test_sequences_without_a_table():
    """Contexts of length 0 need no pages: zeros; a length without pages is reported."""
    q = torch.randn(3, 2, 64, device="cuda").half()
    cu, lens = torch.tensor([0, 2, 3], dtype=torch.int32).cuda(), torch.tensor([0, 0], dtype=torch.int32).cuda()
    k = torch.zeros(1, 2, 16, 64, device="cuda", dtype=torch.float16)
    cache = kernels.kv_cache(k.data_ptr(), k.data_ptr(), "f16", 1, 16, 2, 64)
    batch = kernels.kv_batch(2, cu.data_ptr(), lens.data_ptr(), None, 0)
    nb = kernels.paged_attention_workspace(cache, batch, handle(q, "f16"), 3)
    work, out = torch.empty(nb, device="cuda", dtype=torch.uint8), torch.ones_like(q)
    for length, code in ((0, 0), (5, 6)):
        lens.fill_(length)
        kernels.paged_attention(cache, batch, handle(q, "f16"), handle(out.fill_(1), "f16"), 3, 0.125, True, 0, work.data_ptr(), nb, stream())
        torch.cuda.synchronize()
        assert torch.all(out == 0) and kernels.device_error() == code


@gpu
def test_two_calls_at_once():
    """Two streams, each with a workspace of its own, over one cache."""
    st = make("f16", "f16", 128, 64, 2, 2, [90, 1, 5], [300, 2000, 0], tail_rows=0)
    ref = attend(st)
    check_attention(st, ref)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(side[i]):
                outs[i].append(attend(st))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs[0] + outs[1])


@gpu
def test_calls_without_torch():
    """A step on the package's own buffers, as a host without PyTorch makes it: packed q|k|v, 8-bit cache."""
    from chestnut_b200 import DeviceBuffer
    rs = np.random.default_rng(0)
    tokens, page, pages, width = 3, 64, 6, 3
    qkv = rs.standard_normal((tokens, 48, 128)).astype(np.float16)
    d_qkv = DeviceBuffer(qkv.nbytes).upload(qkv)
    k, v = (DeviceBuffer(pages * 16 * page * 128).zero() for _ in range(2))
    ke, ve = (DeviceBuffer(pages * 16 * page).zero() for _ in range(2))
    i32 = [DeviceBuffer(a.nbytes).upload(a) for a in (np.array([0, 1, 2, 3], np.int32), np.array([1, 1, 1], np.int32),
                                                      np.arange(9, dtype=np.int32).reshape(3, 3) % 6)]
    cache = kernels.kv_cache(k.ptr, v.ptr, "e4m3", pages, page, 16, 128, ke.ptr, ve.ptr)
    table = np.array([[0, 1, 2], [3, 4, 5], [5, 1, 1]], np.int32)
    i32[2].upload(table)
    batch = kernels.kv_batch(tokens, *(b.ptr for b in i32), width)
    q, kk, vv = (kernels.heads(d_qkv.ptr + i * 16 * 128 * 2, "f16", 16, 128, 48 * 128) for i in range(3))
    qk = kernels.heads(d_qkv.ptr, "f16", 32, 128, 48 * 128)
    freq, magnitude = kernels.rope_frequencies(128, factor=8.0, scaling="parts", context=4096)
    pos, d_freq = np.zeros(tokens, np.int64), DeviceBuffer(freq.nbytes).upload(freq)
    d_pos, d_out = DeviceBuffer(pos.nbytes).upload(pos), DeviceBuffer(tokens * 16 * 128 * 2)
    out = kernels.heads(d_out.ptr, "f16", 16, 128)
    work = DeviceBuffer(kernels.paged_attention_workspace(cache, batch, q, tokens))
    kernels.rope(qk, qk, tokens, d_pos.ptr, d_freq.ptr, 128, magnitude=magnitude)
    kernels.kv_write(cache, batch, kk, vv, tokens)
    kernels.paged_attention(cache, batch, q, out, tokens, 128 ** -0.5, True, 0, work.ptr, work.nbytes)
    kernels.synchronize()
    assert kernels.device_error() == 0
    # one key each: the output is the value that the cache holds
    want = expand(*quantise(qkv[:, 32:].astype(np.float64)))
    assert np.array_equal(d_out.download(np.float16, (tokens, 16, 128)), want.astype(np.float16))


@gpu
def test_host_pointers_are_refused():
    host = torch.zeros(16, 8, 64, dtype=torch.float16)
    dev = host.cuda()
    pos, freq = torch.zeros(16, dtype=torch.int64), torch.zeros(32, dtype=torch.float64)
    d_pos, d_freq = pos.cuda(), freq.cuda()
    L = _lib.lib()
    assert L.cn_rope(handle(host, "f16"), handle(dev, "f16"), 16, d_pos.data_ptr(), d_freq.data_ptr(), 64, 0, 1.0, None) == CN_ERR_ARG
    assert b"not device memory" in L.cn_last_error()
    assert L.cn_rope(handle(dev, "f16"), handle(dev, "f16"), 16, pos.data_ptr(), d_freq.data_ptr(), 64, 0, 1.0, None) == CN_ERR_ARG
