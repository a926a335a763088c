"""Rotary positions, the paged K/V cache and the attention over it at their edges: what lies in places that no row
sees, pages that are given up or do not exist, rows of very different sizes, empty calls.  Plain forms, tolerances and
their derivation: test_temporal_ops.py."""
import math

import numpy as np
import pytest

from chestnut_b200 import _lib, kernels

torch = pytest.importorskip("torch")

import test_temporal_ops as ops  # noqa: E402

gpu = pytest.mark.gpu


ALTERNATING = [
    # dtype, dim, page, cache heads, group, (new, length) of each sequence: contexts in whole blocks of 128 keys
    ("f16", 128, 64, 8, 1, [(64, 640), (256, 512), (128, 256), (20, 384), (200, 1280), (64, 128), (128, 1024), (256, 256)] * 3),
    ("bf16", 64, 32, 8, 1, [(128, 1152), (40, 128), (129, 256), (64, 768), (17, 256), (255, 384), (100, 1408)] * 3),
    ("bf16", 128, 128, 5, 3, [(30, 640), (100, 256), (42, 384), (6, 128), (85, 512), (43, 896)] * 2),
    ("f16", 64, 16, 16, 1, [(64, 256 + 128 * (i * 7 % 5)) if i % 3 else (256, 256) for i in range(40)]),
]


@gpu
@pytest.mark.parametrize("shape", ALTERNATING, ids=lambda s: "-".join(map(str, s[:5])))
@pytest.mark.parametrize("causal", [False, True])
def test_tiles_of_one_and_of_two_halves_in_turn(shape, causal):
    """Tiles whose halves share the keys, followed by pieces of one block and by tiles of two halves."""
    dtype, dim, page, hk, group, seqs = shape
    ops.test_attention_over_long_contexts((dtype, dtype, dim, page, hk, group, [n for n, _ in seqs],
                                           [total - n for n, total in seqs], causal, 0))


def unseen(st, first):
    """Whether each place of the cache [pages][page] holds no key that some row sees (first: of each sequence)."""
    hidden = np.ones((st["pages"], st["page"]), bool)
    for s, n in enumerate(st["length"]):
        for p in range(max(first[s], 0), n):
            hidden[int(st["table"][s, p // st["page"]]), p % st["page"]] = False
    return torch.from_numpy(hidden).cuda()


@gpu
@pytest.mark.parametrize("byte", [0, 1, 254, 255])
@pytest.mark.parametrize("dtype,dim", [("f16", 64), ("f16", 128), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("new,past,window", [([1, 1, 2], [4, 100, 33], 0), ([3, 2], [30, 200], 20), ([150], [20], 0),
                                             ([90, 40], [200, 333], 64)])
def test_powers_of_two_that_no_row_sees(dtype, dim, byte, new, past, window):
    """Any exponent byte behind a context's end, in unused pages and in front of the window, beside NaN codes."""
    st = ops.make(dtype, "e4m3", dim, 16, 2, 2, new, past)
    hidden = unseen(st, [p - window + 1 if window else 0 for p in past])
    for m in "kv":
        st[m].masked_fill_(hidden[:, None, :, None], 0x7f)
        st[m + "_exp"].masked_fill_(hidden[:, None], byte)
    out = ops.attend(st, window=window)
    assert kernels.device_error() == 0
    ops.check_attention(st, out, window=window)


@gpu
@pytest.mark.parametrize("byte", [0, 255])
@pytest.mark.parametrize("new,past,window", [([4], [40], 0), ([150], [20], 0), ([90], [200], 64)])
def test_a_power_of_two_that_one_row_sees(byte, new, past, window):
    """The newest token's exponent bytes are no numbers: the rows before it do not know."""
    st = ops.make("f16", "e4m3", 64, 16, 2, 2, new, past)
    p = st["length"][0] - 1
    for m in "kv":
        st[m + "_exp"][int(st["table"][0, p // 16]), :, p % 16] = byte
    out = ops.attend(st, window=window)
    out[new[0] - 1] = 7.0  # the row that sees it
    ops.check_attention(dict(st, new=[new[0] - 1]), out, window=window)


UNITS = """
#include <cstdio>
#include <cstdlib>
#include "%s/cn_paged.cuh"
int main(int, char** v) {
  cn::PagedArgs a = {};
  cn::PagedSeq q = {};
  a.tile_tokens = atoi(v[1]), a.extra = 2, a.causal = atoi(v[4]), a.window = atoi(v[5]);
  q.n = atoi(v[2]), q.past = atoi(v[3]), q.len = q.n + q.past;
  q.tiles = (q.n + a.tile_tokens - 1) / a.tile_tokens;
  long long sum = 0;
  for (int lane = 0; lane < 32; ++lane) sum += cn::paged_lane_units<128>(a, q, lane);
  printf("%%lld %%d %%d", sum, (int)sizeof(cn::paged_lane_units<128>(a, q, 0)), (int)sizeof(cn::PagedScratch<32>::seq_units[0]));
}
"""


def test_units_of_long_prompts_are_counted_in_64_bits(tmp_path):
    """The line of work of one head is longer than 2^31 units for prompts that a call may bring."""
    import subprocess
    import build
    src, exe = tmp_path / "units.cu", tmp_path / "units"
    src.write_text(UNITS % build.CSRC)
    flags = [f for f in build.FLAGS if f not in ("-v", "-Xptxas", "-O3", "-lineinfo")]
    subprocess.run([build.NVCC, *flags, str(src), "-o", str(exe)], check=True, capture_output=True)
    for tile, n, past, causal, window in ((2, 1050001, 0, 1, 0), (32, 4200007, 0, 1, 0), (256, 12000000, 5, 1, 0), (2, 700000, 300000, 0, 0),
                                          (16, 1000, 77, 1, 300)):
        t0 = np.arange(0, n, tile, dtype=np.int64)
        last = past + np.minimum(t0 + tile, n)
        hi = last if causal else np.full_like(last, past + n)
        lo = np.maximum(past + t0 - window + 1, 0) // 128 * 128 if window else 0
        want = int((np.maximum(-(-(hi - lo) // 128), 1) + 2).sum())
        got = subprocess.run([exe, *map(str, (tile, n, past, causal, window))], check=True, capture_output=True, text=True).stdout
        assert got == f"{want} 8 8"
        assert n == 1000 or want >= 1 << 31


@pytest.mark.parametrize("tokens", [2 ** 28 + 1, 2 ** 62, 2 ** 63 - 1])
def test_more_rows_than_an_index_holds_are_refused(tokens):
    q = ops._heads(h=32)
    L = _lib.lib()
    assert L.cn_paged_attention(ops._cache(), ops._batch(), q, q, tokens, 0.125, 1, 0, 0x100, 1 << 40, None) == ops.CN_ERR_ARG
    assert b"2^30" in L.cn_last_error()


@gpu
@pytest.mark.parametrize("dtype,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3"), ("bf16", "e4m3")])
@pytest.mark.parametrize("dim,page,new,past", [(64, 16, [1, 2], [300, 90]), (128, 64, [150, 40], [600, 300]),
                                               (64, 128, [20, 300], [900, 100]), (128, 256, [64], [1000]),
                                               (64, 32, [33, 1, 200], [500, 400, 56])])
def test_keys_of_pages_outside_the_cache_are_zeros(dtype, cache, dim, page, new, past):
    """Their K and V read as zeros, in the middle of a context and where a row's keys end, for the rows of both kernels;
    what other sequences left on the chip does not show."""
    st = ops.make(dtype, cache, dim, page, 2, 2, new, past, tail_rows=0)
    for s, n in enumerate(st["length"]):
        for i, bad in ((n // page // 2, -1), ((n - 1) // page, 2 ** 31 - 1), (0, st["pages"])):
            if i == 0 and s:
                continue
            st["d_table"][s, i] = bad
            for m in "kv":
                st["ctx"][m][s][i * page:(i + 1) * page] = 0.0
    for causal in (True, False):
        out = ops.attend(st, causal=causal)
        torch.cuda.synchronize()
        assert kernels.device_error() == 6
        ops.check_attention(st, out, causal)
        assert torch.equal(out, ops.attend(st, causal=causal))
    torch.cuda.synchronize()
    assert kernels.device_error() == 6


@gpu
@pytest.mark.parametrize("dtype,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3")])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (128, 128), (64, 256)])
@pytest.mark.parametrize("new,past,window", [([1, 3], [700, 411], 60), ([1, 1], [640, 1023], 1), ([150], [900], 130),
                                             ([20, 300], [777, 555], 200)])
def test_pages_in_front_of_the_window_may_be_given_up(dtype, cache, dim, page, new, past, window):
    """Table entries of pages that lie wholly in front of every row's window name no page; nothing is reported."""
    st = ops.make(dtype, cache, dim, page, 2, 2, new, past)
    for s, p in enumerate(past):
        st["d_table"][s, : max(0, p - window + 1) // page] = -1
    out = ops.attend(st, window=window)
    torch.cuda.synchronize()
    assert kernels.device_error() == 0
    ops.check_attention(st, out, window=window)


def test_an_empty_step_needs_no_memory():
    """No tokens: tensors without elements have no address.  With tokens, or where the batch has sequences, what they
    need is still asked for."""
    L = _lib.lib()
    cache, batch, none = ops._cache(), ops._batch(), ops._heads(ptr=None)
    assert L.cn_rope(none, none, 0, None, 0x90000, 64, 0, 1.0, None) == 0
    assert L.cn_kv_write(cache, batch, none, none, 0, None) == 0
    assert L.cn_kv_read(cache, batch, none, none, 0, None) == 0
    assert L.cn_paged_attention(cache, batch, none, none, 0, 0.125, 1, 0, None, 0, None) == 0
    nobody = kernels.kv_batch(0, None, None, None, 0)
    assert L.cn_paged_attention(cache, nobody, none, none, 0, 0.125, 1, 0, None, 0, None) == 0
    assert kernels.paged_attention_workspace(cache, batch, none, 0) > 0
    assert kernels.paged_attention_workspace(cache, batch, none, 5) > 0  # only sizes are read
    for call in (lambda: L.cn_rope(none, none, 1, 0xa0000, 0x90000, 64, 0, 1.0, None),
                 lambda: L.cn_rope(ops._heads(), ops._heads(), 1, None, 0x90000, 64, 0, 1.0, None),
                 lambda: L.cn_kv_write(cache, batch, none, ops._heads(), 1, None),
                 lambda: L.cn_kv_read(cache, batch, ops._heads(), none, 1, None),
                 lambda: L.cn_paged_attention(cache, batch, none, ops._heads(), 1, 0.125, 1, 0, 0x100, 1 << 40, None)):
        assert call() == ops.CN_ERR_ARG


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_rows_codes_do_not_depend_on_its_neighbours(dtype, dim):
    """Negative zeros beside rows with infinities and NaN: their codes are the definition's."""
    n, hk = 6, 8
    x = torch.randn(n, hk, dim, generator=torch.Generator().manual_seed(1)).to(ops.TYPES[dtype])
    x[:, :, ::5] = -0.0
    x[1::2, 3, 1], x[::2, 4, 2], x[2, 6, 3] = math.inf, -math.inf, math.nan
    st = ops.make(dtype, "e4m3", dim, 16, hk, 1, [n], [0], fill=0.0)
    d = x.cuda()
    kernels.kv_write(*ops.descriptors(st), ops.handle(d, dtype), ops.handle(d, dtype), n, ops.stream())
    codes, exps = ops.quantise(x.double().numpy())
    at = int(st["table"][0, 0])
    for m in "kv":
        got, e = st[m][at, :, :n].cpu().numpy().swapaxes(0, 1), st[m + "_exp"][at, :, :n].cpu().numpy().T
        nan = (codes & 0x7f) == 0x7f
        assert np.array_equal(e, exps) and np.array_equal(np.where(nan, codes, got), codes)
        assert np.all((got[nan] & 0x7f) == 0x7f)


@gpu
def test_rope_of_one_token_in_place():
    """One token's or one head's stride says nothing: x and out are the same memory whatever it is."""
    freq, _ = kernels.rope_frequencies(64)
    d_freq, pos = torch.from_numpy(freq).cuda(), torch.tensor([5, 9]).cuda()
    for tokens, h, other in ((1, 4, dict(token_stride=4096)), (2, 1, dict(token_stride=64, head_stride=512))):
        x = torch.randn(tokens, h, 64, generator=torch.Generator().manual_seed(3)).half().cuda()
        want = torch.empty_like(x)
        kernels.rope(ops.handle(x, "f16"), ops.handle(want, "f16"), tokens, pos.data_ptr(), d_freq.data_ptr(), 64, stream=ops.stream())
        kernels.rope(ops.handle(x, "f16"), kernels.heads(x.data_ptr(), "f16", h, 64, **other), tokens, pos.data_ptr(),
                     d_freq.data_ptr(), 64, stream=ops.stream())
        assert torch.equal(x, want)


def check_columns(st, out, causal=True):
    """As check_attention, but a column answers for its own values alone: a weight is off by u(f16) of itself, or, where
    it is too small for that, by 2^-32 of the largest weight of its row."""
    got, row = out.cpu().double().numpy(), 0
    hq, scale = st["hk"] * st["group"], st["dim"] ** -0.5
    for s, (n, p) in enumerate(zip(st["new"], st["past"])):
        q = st["qkv"][row:row + n, :hq].double().numpy()
        for i in range(n):
            for h in range(hq):
                hi = p + i + 1 if causal else p + n
                k, v = (st["ctx"][m][s][:hi, h // st["group"]] for m in "kv")
                a = k @ q[i, h] * scale
                w = np.exp(a - a.max())
                w /= w.sum()
                ref = w @ v
                big = (np.abs(k) @ np.abs(q[i, h]) * scale).max()
                err = 2 * (st["dim"] + 4) * ops.U32 * big + 2.0 ** -21 + hi * ops.U32
                tol = ops.tiny(st["dtype"]) + ops.u(st["dtype"]) * np.abs(ref) + (ops.u("f16") + err) * (w @ np.abs(v)) \
                    + hi * 2.0 ** -32 * w.max() * np.abs(v).max(0)
                bad = ~(np.abs(got[row + i, h] - ref) <= tol * (1 + ops.u(st["dtype"])))
                assert not bad.any(), (s, i, h, np.argwhere(bad)[:4].tolist(), got[row + i, h][bad][:4], ref[bad][:4], tol[bad][:4])
        row += n


def put_v(st, s, p, x):
    """Row p of sequence s of the 8-bit cache's V becomes x [hk, dim]."""
    codes, exps = ops.quantise(x)
    at = int(st["table"][s, p // st["page"]]), p % st["page"]
    st["v"][at[0], :, at[1]] = torch.from_numpy(codes).cuda()
    st["v_exp"][at[0], :, at[1]] = torch.from_numpy(exps).cuda()
    st["ctx"]["v"][s][p] = ops.expand(codes, exps)


SIZES = [
    # dtype, size of the rows, (position, size, column or None: all) of others; size 0: a row of zeros
    ("f16", 2.0 ** -8, [(3, 2.0 ** 4, 0)]), ("f16", 2.0 ** -8, [(300, 2.0 ** 12, 7)]), ("f16", 1.0, [(2, 2.0 ** -12, 9)]),
    ("bf16", 1.0, [(3, 2.0 ** 26, 0)]), ("bf16", 2.0 ** -3, [(3, 2.0 ** 17, 5), (200, 2.0 ** 30, 3)]),
    ("bf16", 2.0 ** -20, [(70, 2.0 ** 20, 0), (71, 0.0, None)]), ("bf16", 2.0 ** -45, [(40, 2.0 ** 45, 1)]),
    ("bf16", 2.0 ** -26, [(0, 0.0, None)]), ("bf16", 2.0 ** -36, [(5, 0.0, None), (290, 0.0, None)]),
    ("bf16", 1.0, [(7, 2.0 ** -20, 2), (250, 2.0 ** -40, 4)]), ("bf16", 2.0 ** 20, [(7, 2.0 ** -20, None), (8, 2.0 ** 45, 3)]),
]


@gpu
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{s[0]}-{math.log2(s[1]):.0f}-" + "-".join(f"{p}:{math.log2(x) if x else 0:.0f}" for p, x, _ in s[2]))
@pytest.mark.parametrize("dim,group,new,past", [(64, 1, [1], [320]), (128, 2, [3, 1], [309, 400]), (64, 2, [40], [300]),
                                                (128, 1, [150], [310]), (128, 3, [100], [512])])
def test_rows_of_very_different_sizes(sizes, dim, group, new, past):
    """An 8-bit cache whose V rows are powers of two apart, the large ones in one column: the other columns keep their
    average.  A row with a column of its own keeps that; a row of zeros moves nothing."""
    dtype, size, others = sizes
    st = ops.make(dtype, "e4m3", dim, 32, 2, group, new, past)
    rs = np.random.default_rng(5)
    for s in range(len(new)):
        own = [c for _, x, c in others if c is not None and 0 < x < size]
        for p in range(st["length"][s]):
            x = rs.standard_normal((2, dim)) * size * 2.0 ** rs.integers(-2, 1)
            x[:, own] = 0
            put_v(st, s, p, x)
        for p, amount, column in others:
            x = np.zeros((2, dim))
            if column is not None:
                x[:, column] = amount
            else:
                x[:] = amount * rs.standard_normal((2, dim))
                x[:, own] = 0
            put_v(st, s, p, x)
    out = ops.attend(st)
    assert kernels.device_error() == 0
    check_columns(st, out)
    assert torch.equal(out, ops.attend(st))


@gpu
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("new", [1, 20])
def test_many_small_weights_keep_their_sum(cache, new):
    """One key that outweighs each of 2,000 others by e^16 = 2^23.1: what those add up to.  Off by the weights' rounding
    and the output's, u(f16) each, and 2^-14 for all that is in f32 (scores of 23, sums of 2,000 values).  Sequences
    enough that no context is cut."""
    seqs, hk = 24, 16
    st = ops.make("f16", cache, 64, 256, hk, 1, [new] * seqs, [2000 - new] * seqs, fill=0.0, tail_rows=0)
    st["qkv"].zero_()
    st["qkv"][:, :hk, 0] = 8.0
    st["d_qkv"].copy_(st["qkv"])
    codes, exps = ops.quantise(np.eye(1, 64) * 16.0)     # the heavy key: 8 * 16 / sqrt(64) = 16; the others: 0
    at = st["table"][:, 0].long().cuda()                 # the first page of each sequence
    st["k"].zero_()
    if cache == "e4m3":
        st["k_exp"].fill_(127), st["v_exp"].fill_(127)
        st["k"][at, :, 0], st["k_exp"][at, :, 0] = torch.from_numpy(codes[0]).cuda(), int(exps[0])
        st["v"].fill_(0x38)                              # 1.0
    else:
        st["k"][at, :, 0, 0] = 16.0
        st["v"].fill_(1.0)
    st["v"][at, :, 0] = 0
    out = ops.attend(st, causal=False).double()
    want = 1999 * math.exp(-16.0) / (1 + 1999 * math.exp(-16.0))
    assert torch.all((out - want).abs() <= (2 * ops.u("f16") + 2.0 ** -14) * want + ops.tiny("f16"))


@gpu
@pytest.mark.parametrize("new", [1, 40, 200])
def test_a_page_outside_the_cache_beside_large_rows(new):
    """Its zeros count as rows far smaller than the others, and nothing is read for them."""
    st = ops.make("bf16", "e4m3", 64, 32, 2, 2, [new], [400], tail_rows=0)
    rs = np.random.default_rng(1)
    for p in range(st["length"][0]):
        put_v(st, 0, p, rs.standard_normal((2, 64)) * 2.0 ** 38)
    st["d_table"][0, 4] = -1
    st["d_table"][0, 9] = st["pages"]
    for m in "kv":
        for page in (4, 9):
            st["ctx"][m][0][page * 32:page * 32 + 32] = 0.0
    out = ops.attend(st)
    torch.cuda.synchronize()
    assert kernels.device_error() == 6
    check_columns(st, out)


@gpu
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("group,new", [(1, [64] + [0] * 63), (8, [0] * 40 + [64] + [0] * 23), (4, [64, 64]), (2, [100] + [1] * 99),
                                       (1, [1] * 600), (4, [0, 1] * 90), (16, [1] * 30 + [9, 0])])
def test_batches_that_either_kernel_may_take(cache, group, new):
    """Slots of which one has a frame and the others nothing or a token, two frames, hundreds of single tokens."""
    st = ops.make("bf16", cache, 64, 16, 1, group, new, [(37 * i) % 150 for i in range(len(new))])
    out = ops.attend(st)
    ops.check_attention(st, out)
    assert torch.equal(out, ops.attend(st)) and kernels.device_error() == 0


@gpu
@pytest.mark.parametrize("dim,dtype", [(128, "f16"), (64, "bf16")])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_large_rows_that_come_in_turn(dim, dtype, seed):
    """An 8-bit cache where one row in fifty is 2^13 larger, so that the power of two of V's blocks changes along a context,
    over batches whose tiles of one half, pieces of one block and tiles of two halves follow each other on an SM: each
    call gives the same, and what 64 bits give (of the other columns, and of the large rows' own)."""
    rng, g = np.random.default_rng(seed), torch.Generator(device="cuda").manual_seed(seed)
    hk, page, n = 8, 32, 40
    new = [int(x) for x in rng.choice([0, 1, 36, 64, 64, 50, 17, 64, 200], n)]
    length = [a + int(b) for a, b in zip(new, rng.choice([0, 20, 50, 600, 650, 1300, 4000], n))]
    used = [-(-x // page) for x in length]
    pages, first = sum(used) + 2, np.concatenate([[0], np.cumsum(used)])
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((n, max(used)), -1, dtype=torch.int32, device="cuda")
    for s in range(n):
        table[s, : used[s]] = order[first[s]:first[s + 1]]
    st = dict(dtype=dtype, cache="e4m3", dim=dim, page=page, hk=hk, group=1, new=new, pages=pages, width=max(used), d_table=table,
              d_cu=torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32).cuda(), d_len=torch.tensor(length, dtype=torch.int32).cuda(),
              d_qkv=torch.randn(sum(new) + 1, hk, dim, generator=g, device="cuda").to(ops.TYPES[dtype]))
    wide = {}
    for m in "kv":
        x = torch.randn(pages, hk, page, dim, generator=g, device="cuda")
        if m == "v":
            big = torch.rand(pages, hk, page, 1, generator=g, device="cuda") < 0.02
            x *= torch.where(big, 2.0 ** 8, 2.0 ** -5)
            x[..., : dim // 2].masked_fill_(big, 0.0)
        part, e = torch.frexp(x.abs().amax(-1))
        e = e - 9 + (part > 0.875).int()
        codes = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
        st[m], st[m + "_exp"], wide[m] = codes.view(torch.uint8), (e + 127).to(torch.uint8), torch.ldexp(codes.double(), e[..., None])
    out = ops.attend(st)
    for _ in range(30):
        assert torch.equal(out, ops.attend(st))
    assert kernels.device_error() == 0
    row = 0
    for s in range(n):
        keys = torch.arange(length[s], device="cuda")
        k, v = (wide[m][table[s].long()[keys // page], :, keys % page].transpose(0, 1) for m in "kv")  # [hk, keys, dim]
        q = st["d_qkv"][row:row + new[s]].double().transpose(0, 1)
        a = (q @ k.mT) * dim ** -0.5
        a.masked_fill_(keys > length[s] - new[s] + torch.arange(new[s], device="cuda")[:, None], -math.inf)
        w = torch.softmax(a, -1)
        big = (q.abs() @ k.abs().mT * dim ** -0.5).amax(-1, keepdim=True) if new[s] else 0.0
        err = 2 * (dim + 4) * ops.U32 * big + 2.0 ** -21 + length[s] * ops.U32
        tol = ops.tiny(dtype) + ops.u(dtype) * (w @ v).abs() + (ops.u("f16") + err) * (w @ v.abs()) + (w > 0).double() @ v.abs() * 2.0 ** -32
        off = (out[row:row + new[s]].double().transpose(0, 1) - w @ v).abs() - tol * (1 + ops.u(dtype))
        assert new[s] == 0 or off.max() <= 0, (s, off.max().item())
        row += new[s]
