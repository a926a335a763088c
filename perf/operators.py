"""Measured cases of the temporal-context operators: rotary positions, the paged K/V cache (8 bits as it is
written, read back) and the attention of new tokens over that cache.

The heads are the frame models' own (16 x 128 and 8 x 64) and grouped variants of them; a frame brings 64 vision
tokens, a clip lasts up to 1,200 frames and up to 64 clips share a GPU.  `own` chooses between the plain form (torch,
32 bits) and the framework's kernels on the same inputs."""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
EXP_MIN, EXP_MAX, EXP_BIAS = -48, 48, 127  # the power-of-two scales of an 8-bit cache row


def listed():
    return [
        # one token of each of 64 clips: q and k heads of the 1B model turned in one call
        {"name": "rope step", "op": "rope", "tokens": 64, "heads": 32, "dim": 128, "rot": 128, "interleaved": False,
         "dtype": "f16", "far": 76800, "factor": 1.0},
        # a long first prompt in bf16, half of each head turned, interleaved pairs, frequencies scaled for 8x the context
        {"name": "rope prompt", "op": "rope", "tokens": 16384, "heads": 40, "dim": 128, "rot": 64, "interleaved": True,
         "dtype": "bf16", "far": 1000000, "factor": 8.0},
        # the step's K and V enter an 8-bit cache
        {"name": "write step e4m3", "op": "write", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 100, "past_hi": 4800,
         "q_heads": 16, "kv_heads": 16, "dim": 128, "page": 64, "dtype": "f16", "cache": "e4m3"},
        # whole prompts of eight clips, lengths all different
        {"name": "write prompts e4m3", "op": "write", "seqs": 8, "new_lo": 513, "new_hi": 4099, "past_lo": 0, "past_hi": 700,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "dtype": "bf16", "cache": "e4m3"},
        # the last frame's 64 tokens of one clip read back
        {"name": "read frame e4m3", "op": "read", "seqs": 1, "new_lo": 64, "new_hi": 64, "past_lo": 3000, "past_hi": 3000,
         "q_heads": 8, "kv_heads": 8, "dim": 64, "page": 16, "dtype": "f16", "cache": "e4m3"},
        # sixteen clips' whole contexts read back
        {"name": "read contexts e4m3", "op": "read", "seqs": 16, "new_lo": 1001, "new_hi": 4797, "past_lo": 0, "past_hi": 0,
         "q_heads": 16, "kv_heads": 16, "dim": 128, "page": 64, "dtype": "bf16", "cache": "e4m3"},
        # one token of one clip: the shortest call
        {"name": "attend one token", "op": "attend", "seqs": 1, "new_lo": 1, "new_hi": 1, "past_lo": 1000, "past_hi": 1000,
         "q_heads": 16, "kv_heads": 16, "dim": 128, "page": 16, "dtype": "f16", "cache": "f16", "causal": True, "window": 0},
        # one token of 64 clips of very different lengths, grouped heads
        {"name": "attend step ragged", "op": "attend", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 50, "past_hi": 8190,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "cache": "bf16", "causal": True, "window": 0},
        # a few tokens (1 to 4) of 48 clips over the 8-bit cache, one frame a token for 1,200 frames and more
        {"name": "attend step e4m3", "op": "attend", "seqs": 48, "new_lo": 1, "new_hi": 4, "past_lo": 1200, "past_hi": 4800,
         "q_heads": 16, "kv_heads": 16, "dim": 128, "page": 32, "dtype": "f16", "cache": "e4m3", "causal": True, "window": 0},
        # a frame's 64 vision tokens of 16 clips, free within the frame, over all frames before it
        {"name": "attend frame", "op": "attend", "seqs": 16, "new_lo": 64, "new_hi": 64, "past_lo": 640, "past_hi": 4032,
         "q_heads": 16, "kv_heads": 16, "dim": 128, "page": 64, "dtype": "f16", "cache": "f16", "causal": False, "window": 0},
        # a whole first prompt, causal, grouped heads
        {"name": "attend prompt", "op": "attend", "seqs": 1, "new_lo": 8192, "new_hi": 8192, "past_lo": 0, "past_hi": 0,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "dtype": "bf16", "cache": "bf16", "causal": True, "window": 0},
        # chunks of odd lengths over an 8-bit cache, heads of the 39M model in groups of three, a sliding window
        {"name": "attend chunks e4m3", "op": "attend", "seqs": 12, "new_lo": 5, "new_hi": 701, "past_lo": 0, "past_hi": 5000,
         "q_heads": 24, "kv_heads": 8, "dim": 64, "page": 32, "dtype": "f16", "cache": "e4m3", "causal": True, "window": 2500},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attend", "attend", "attend"])
    if op == "rope":
        dim, dtype = rng.choice([64, 128]), rng.choice(["f16", "bf16", "f32"])
        return {"op": op, "tokens": _log(rng, 1, 8192 if dtype == "f32" else 16384), "heads": rng.randint(1, 40), "dim": dim,
                "rot": rng.choice([dim, dim // 2, 2 * rng.randint(1, dim // 2)]), "interleaved": rng.random() < 0.5,
                "dtype": dtype, "far": _log(rng, 1000, 2000000), "factor": rng.choice([1.0, 4.0, 8.0])}
    top = max(work(c)["flops"] for c in listed()), max(work(c)["bytes"] for c in listed())
    while True:
        dtype = rng.choice(["f16", "bf16"])
        kv = rng.choice([1, 2, 4, 5, 8, 16])
        c = {"op": op, "seqs": _log(rng, 1, 64), "new_lo": 1, "new_hi": 1, "past_lo": 0, "past_hi": _log(rng, 1, 8000),
             "q_heads": kv * rng.choice([1, 1, 2, 3, 4, 7, 8]), "kv_heads": kv, "dim": rng.choice([64, 128]),
             "page": rng.choice([16, 32, 64, 128]), "dtype": dtype, "cache": rng.choice([dtype, "e4m3"])}
        c["past_lo"] = rng.choice([0, c["past_hi"] // 2, c["past_hi"]])
        if op != "attend" or rng.random() < 0.6:
            c["new_hi"] = _log(rng, 1, 8192 if op == "attend" else 4800)
            c["new_lo"] = rng.choice([1, max(1, c["new_hi"] // 2), c["new_hi"]])
        if op == "attend":
            c["causal"] = rng.random() < 0.75
            c["window"] = _log(rng, 1, 6000) if c["causal"] and rng.random() < 0.3 else 0
        w = work(c)
        reach = c["seqs"] * (c["new_hi"] + c["past_hi"])
        if w["flops"] <= top[0] and w["bytes"] <= top[1] and reach * c["kv_heads"] * c["dim"] * 4 <= 3e9 and (
                op != "attend" or reach * c["new_hi"] * c["q_heads"] * 4 <= 8.6e9):
            return c


def _spread(n, lo, hi, turn):
    """n whole numbers over lo..hi, both ends among them where n > 1, in no order."""
    if n == 1:
        return [hi]
    return [lo + round((hi - lo) * ((s * turn) % n) / (n - 1)) for s in range(n)]


def _turn(n, k):
    return next(t for t in range(max(1, n // k), 2 * n + 2) if math.gcd(t, n) == 1)


def _counts(case):
    """(new tokens, tokens before them) of each sequence."""
    n = case["seqs"]
    return (_spread(n, case["new_lo"], case["new_hi"], _turn(n, 3)), _spread(n, case["past_lo"], case["past_hi"], _turn(n, 2)))


def work(case):
    if case["op"] == "rope":
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": 2 * size * case["tokens"] * case["heads"] * case["dim"] + 8 * case["tokens"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    new, past = _counts(case)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    size, held = DTYPES[case["dtype"]].itemsize, d * DTYPES[case["cache"]].itemsize + (case["cache"] == "e4m3")
    if case["op"] != "attend":
        return {"bytes": 2 * sum(new) * hk * (d * size + held), "flops": 2 * sum(new) * hk * d}
    pairs = rows = 0
    for n, p in zip(new, past):
        if not case["causal"]:
            pairs, rows = pairs + n * (n + p), rows + n + p
            continue
        w = case["window"] or n + p
        full = max(0, min(n, n + p - w))  # tokens whose window is full: the last ones
        pairs += full * w + (n - full) * p + (n - full) * (n - full + 1) // 2
        rows += min(n + p, n + w - 1)
    return {"bytes": 2 * sum(new) * hq * d * size + 2 * rows * hk * held, "flops": 4 * d * hq * pairs}


def _frequencies(rot, factor, far):
    """Radians a token of each pair; scaled by parts where the context grows by `factor`: pairs that turn often stay,
    pairs that turn less than once are slowed by the factor, those between are blended."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if factor == 1.0:
        return f, 1.0
    turns = far / factor * f / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0, 1)
    return f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype, by=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(by).to(dtype)

    st = {"case": case}
    if case["op"] == "rope":
        freq, st["magnitude"] = _frequencies(case["rot"], case["factor"], case["far"])
        st["freq"] = freq.cuda()
        st["x"] = normal(case["tokens"], case["heads"], case["dim"])
        st["out"] = torch.empty_like(st["x"])
        st["pos"] = torch.randint(0, case["far"], (case["tokens"],), generator=g, device="cuda")
        return st
    new, past = _counts(case)
    n, hq, hk, d, page = case["seqs"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    length = [a + b for a, b in zip(new, past)]
    used = [-(-v // page) for v in length]
    pages, width = sum(used) + 3, max(used)
    st["new"] = torch.tensor(new, device="cuda")
    st["cu"] = torch.cat([st["new"].new_zeros(1), st["new"].cumsum(0)]).to(torch.int32)
    st["length"] = torch.tensor(length, device="cuda", dtype=torch.int32)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)  # pages lie in no order
    held = torch.arange(width, device="cuda")[None] < torch.tensor(used, device="cuda")[:, None]
    st["table"] = torch.zeros(n, width, device="cuda", dtype=torch.int32)
    st["table"][held] = order[: sum(used)]
    total = sum(new)
    st["qkv"] = normal(total, hq + 2 * hk, d)  # as the product before it leaves them: q, k and v heads in one row
    for name in ("k", "v"):
        if case["cache"] == "e4m3":
            codes = torch.empty(pages, hk, page, d, device="cuda", dtype=DTYPES["e4m3"])
            exps = torch.full((pages, hk, page), EXP_BIAS, device="cuda", dtype=torch.uint8)
            if case["op"] == "write":
                codes.view(torch.uint8).zero_()
            else:
                for p in range(0, pages, 256):
                    size = torch.rand(min(256, pages - p), hk, page, 1, generator=g, device="cuda") * 2 + 0.5  # rows differ in size
                    codes[p:p + 256], exps[p:p + 256] = _quantise(normal(min(256, pages - p), hk, page, d, dtype=torch.float32) * size)
            st[name], st[name + "_exp"] = codes, exps
        elif case["op"] == "write":
            st[name] = torch.zeros(pages, hk, page, d, device="cuda", dtype=DTYPES[case["cache"]])
        else:
            st[name] = torch.empty(pages, hk, page, d, device="cuda", dtype=DTYPES[case["cache"]])
            for p in range(0, pages, 256):
                st[name][p:p + 256] = normal(min(256, pages - p), hk, page, d, dtype=st[name].dtype)
    if case["op"] == "read":
        st["k_out"], st["v_out"] = (torch.empty(total, hk, d, device="cuda", dtype=dtype) for _ in "kv")
    if case["op"] == "attend":
        st["out"] = torch.empty(total, hq, d, device="cuda", dtype=dtype)
        st["scale"] = d ** -0.5
    return st


# ---- plain forms


def _power(e):
    """2.0 ** e in f32 for whole numbers e of a tensor, from its bits: exact."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """f32 rows to e4m3 codes and biased exponents: the least power of two that brings the row's largest value under 448."""
    amax = x.abs().amax(-1)
    part, e = torch.frexp(amax)
    e = torch.where(amax > 0, (e - 9 + (part > 0.875).int()).clamp(EXP_MIN, EXP_MAX), torch.zeros_like(e))
    codes = (x * _power(-e)[..., None]).clamp(-448.0, 448.0).to(DTYPES["e4m3"])
    return codes, (e + EXP_BIAS).to(torch.uint8)


def _places(st):
    """Sequence and position in its context of each new token."""
    seq = torch.repeat_interleave(torch.arange(len(st["new"]), device="cuda"), st["new"], output_size=len(st["qkv"]))
    at = torch.arange(len(st["qkv"]), device="cuda") - st["cu"].long()[seq]
    return seq, at, (st["length"].long() - st["new"])[seq] + at


def _rope(st):
    c, x = st["case"], st["x"].float()
    angle = st["pos"].double()[:, None] * st["freq"]
    cos, sin = (f(angle).float()[:, None] * st["magnitude"] for f in (torch.cos, torch.sin))
    rot, half = c["rot"], c["rot"] // 2
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if c["interleaved"] else (slice(0, half), slice(half, rot))
    out = x.clone()
    out[..., one] = x[..., one] * cos - x[..., two] * sin
    out[..., two] = x[..., two] * cos + x[..., one] * sin
    return out.to(st["x"].dtype)


def _write(st):
    c = st["case"]
    seq, _, pos = _places(st)
    page, row = st["table"][seq, pos // c["page"]].long(), pos % c["page"]
    got = []
    for name, first in (("k", c["q_heads"]), ("v", c["q_heads"] + c["kv_heads"])):
        x = st["qkv"][:, first:first + c["kv_heads"]]
        if c["cache"] == "e4m3":
            codes, exps = _quantise(x.float())
            st[name].view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
            st[name + "_exp"][page, :, row] = exps
            got += [st[name], st[name + "_exp"]]
        else:
            st[name][page, :, row] = x
            got.append(st[name])
    return got


def _read(st):
    c = st["case"]
    seq, _, pos = _places(st)
    page, row = st["table"][seq, pos // c["page"]].long(), pos % c["page"]
    got = []
    for name in ("k", "v"):
        x = st[name].view(torch.uint8)[page, :, row].view(st[name].dtype) if c["cache"] == "e4m3" else st[name][page, :, row]
        x = x.float()
        if c["cache"] == "e4m3":
            x = x * _power(st[name + "_exp"][page, :, row].int() - EXP_BIAS)[..., None]
        top = torch.finfo(st["qkv"].dtype).max
        got.append(x.clamp(-top, top).to(st["qkv"].dtype))
    return got


def _context(st, name):
    """The cache's rows of every sequence in order, f32 [seqs, kv heads, keys, dim]."""
    t = st["table"].long()
    x = st[name].view(torch.uint8)[t].view(st[name].dtype) if st["case"]["cache"] == "e4m3" else st[name][t]
    x = x.float()
    if st["case"]["cache"] == "e4m3":
        x = x * _power(st[name + "_exp"][t].int() - EXP_BIAS)[..., None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _attend(st):
    c = st["case"]
    seq, at, pos = _places(st)
    n, most, hq, hk, d = c["seqs"], int(c["new_hi"]), c["q_heads"], c["kv_heads"], c["dim"]
    q = torch.zeros(n, most, hq, d, device="cuda")
    q[seq, at] = st["qkv"][:, :hq].float()
    where = torch.full((n, most), -1, device="cuda", dtype=torch.long)
    where[seq, at] = pos
    k, v = _context(st, "k"), _context(st, "v")
    keys = torch.arange(k.shape[2], device="cuda")
    exists = keys < st["length"][:, None]
    seen = exists[:, None] & (where[..., None] >= 0)
    if c["causal"]:
        seen &= keys <= where[..., None]
    if c["window"]:
        seen &= keys > where[..., None] - c["window"]
    q = q.view(n, most, hk, hq // hk, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s = (q @ k.mT).mul_(st["scale"]).view(n, hk, hq // hk, most, -1)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill_(~exists[:, None, :, None], 0.0)
    o = (p.flatten(2, 3) @ v).view(n, hk, hq // hk, most, d) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(n, most, hq, d)[seq, at].to(st["qkv"].dtype)


# ---- the framework's calls


def _kernels():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "chestnut-on-pc_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from chestnut_b200 import kernels
    return kernels


def _descriptors(kernels, st):
    """What a program keeps beside its buffers: their descriptions, made once, and the attention's workspace."""
    c = st["case"]

    def heads(t):
        return kernels.heads(t.data_ptr(), c["dtype"], t.shape[1], t.shape[2], t.stride(0), t.stride(1))

    if c["op"] == "rope":
        return {"x": heads(st["x"]), "out": heads(st["out"])}
    hq, hk = c["q_heads"], c["kv_heads"]
    exps = [st[n].data_ptr() for n in ("k_exp", "v_exp")] if c["cache"] == "e4m3" else [None, None]
    own_ = {"cache": kernels.kv_cache(st["k"].data_ptr(), st["v"].data_ptr(), c["cache"], len(st["k"]), c["page"], hk, c["dim"], *exps),
            "batch": kernels.kv_batch(c["seqs"], st["cu"].data_ptr(), st["length"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1]),
            "q": heads(st["qkv"][:, :hq]), "k": heads(st["qkv"][:, hq:hq + hk]), "v": heads(st["qkv"][:, hq + hk:])}
    if c["op"] == "read":
        own_ |= {"k_out": heads(st["k_out"]), "v_out": heads(st["v_out"])}
    if c["op"] == "attend":
        own_["out"] = heads(st["out"])
        own_["bytes"] = kernels.paged_attention_workspace(own_["cache"], own_["batch"], own_["q"], len(st["qkv"]))
        own_["work"] = torch.empty(max(1, own_["bytes"]), device="cuda", dtype=torch.uint8)
    return own_


def run(state):
    c = state["case"]
    if not own:
        return {"rope": _rope, "write": _write, "read": _read, "attend": _attend}[c["op"]](state)
    kernels = _kernels()
    if "own" not in state:
        state["own"] = _descriptors(kernels, state)
    o, stream = state["own"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "rope":
        kernels.rope(o["x"], o["out"], c["tokens"], state["pos"].data_ptr(), state["freq"].data_ptr(), c["rot"],
                     c["interleaved"], state["magnitude"], stream)
        return state["out"]
    total = len(state["qkv"])
    if c["op"] == "write":
        kernels.kv_write(o["cache"], o["batch"], o["k"], o["v"], total, stream)
        return [state[n] for n in (("k", "k_exp", "v", "v_exp") if c["cache"] == "e4m3" else ("k", "v"))]
    if c["op"] == "read":
        kernels.kv_read(o["cache"], o["batch"], o["k_out"], o["v_out"], total, stream)
        return [state["k_out"], state["v_out"]]
    kernels.paged_attention(o["cache"], o["batch"], o["q"], o["out"], total, state["scale"], c["causal"], c["window"],
                            o["work"].data_ptr(), o["bytes"], stream)
    return state["out"]


# ---- the definitions in 64 bits, sequence by sequence


def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _codes64(x):
    """f64 rows [..., dim]: (values of the e4m3 codes, exponents), by comparison with all the type's values."""
    byte = torch.arange(127, device="cuda")
    part, up = (byte % 8).double(), byte // 8
    values = torch.where(byte < 8, part / 8 / 64, (1 + part / 8) * _power64(up - 7))  # 0 ... 448
    middle = (values[1:] + values[:-1]) / 2
    amax = x.abs().amax(-1, keepdim=True)
    powers = _power64(torch.arange(EXP_MIN, EXP_MAX + 1, device="cuda"))
    e = (amax > 448.0 * powers).sum(-1, keepdim=True).clamp(max=EXP_MAX - EXP_MIN) + EXP_MIN
    e = torch.where(amax > 0, e, 0)
    y = (x.abs() * _power64(-e)).clamp(max=448.0)
    below, above = torch.searchsorted(middle, y), torch.searchsorted(middle, y, right=True)
    pick = torch.where(below % 2 == 0, below, above)  # on a middle the two differ by one: the even code
    return values[pick] * torch.where(torch.signbit(x), -1.0, 1.0), e[..., 0] + EXP_BIAS


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        x, out = st["x"].double(), st["x"].double()
        pairs = torch.arange(case["rot"] // 2, device="cuda")
        one, two = (2 * pairs, 2 * pairs + 1) if case["interleaved"] else (pairs, pairs + case["rot"] // 2)
        turn = torch.polar(torch.full((1,), st["magnitude"], device="cuda", dtype=torch.float64), st["pos"].double()[:, None] * st["freq"][None])
        z = torch.complex(x[..., one], x[..., two]) * turn[:, None]
        out[..., one], out[..., two] = z.real, z.imag
        return out
    hq, hk, page = case["q_heads"], case["kv_heads"], case["page"]
    new, past = _counts(case)
    starts = [sum(new[:s]) for s in range(len(new) + 1)]
    table = st["table"].tolist()
    if case["op"] == "write":
        got = []
        for name, first in (("k", hq), ("v", hq + hk)):
            cache = st[name].double() if case["cache"] != "e4m3" else st[name].view(torch.uint8).double()  # all zero but in what is written
            exps = torch.full(cache.shape[:3], EXP_BIAS, device="cuda", dtype=torch.uint8)
            for s, (n, p) in enumerate(zip(new, past)):
                x = st["qkv"][starts[s]:starts[s + 1], first:first + hk].double()
                if case["cache"] == "e4m3":
                    x, e = _codes64(x)
                pos = torch.arange(p, p + n, device="cuda")
                at = torch.tensor(table[s], device="cuda")[pos // page]
                cache[at, :, pos % page] = x
                if case["cache"] == "e4m3":
                    exps[at, :, pos % page] = e.to(torch.uint8)
            got += [cache, exps] if case["cache"] == "e4m3" else [cache]
        return got

    def rows(name, s, lo, hi):
        pos = torch.arange(lo, hi, device="cuda")
        at = torch.tensor(table[s], device="cuda")[pos // page]
        if case["cache"] != "e4m3":
            return st[name][at, :, pos % page].double()
        x = st[name].view(torch.uint8)[at, :, pos % page].view(DTYPES["e4m3"]).double()
        return x * _power64(st[name + "_exp"][at, :, pos % page].int() - EXP_BIAS)[..., None]

    if case["op"] == "read":
        return [torch.cat([rows(name, s, p, p + n) for s, (n, p) in enumerate(zip(new, past))]) for name in "kv"]
    out = torch.zeros(starts[-1], hq, case["dim"], device="cuda", dtype=torch.float64)
    for s, (n, p) in enumerate(zip(new, past)):
        k, v = rows("k", s, 0, n + p), rows("v", s, 0, n + p)
        keys = torch.arange(n + p, device="cuda")
        for h in range(hq):
            for r in range(0, n, 4096):
                pos = torch.arange(p + r, p + min(n, r + 4096), device="cuda")[:, None]
                a = st["qkv"][starts[s] + r:starts[s] + min(n, r + 4096), h].double() @ k[:, h // (hq // hk)].T * st["scale"]
                if case["causal"]:
                    a[keys > pos] = -math.inf
                if case["window"]:
                    a[keys <= pos - case["window"]] = -math.inf
                out[starts[s] + r:starts[s] + min(n, r + 4096), h] = torch.softmax(a, -1) @ v[:, h // (hq // hk)]
    return out
