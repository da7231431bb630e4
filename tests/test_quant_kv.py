"""A key/value cache in 8 or 4 bits on the CPU: the references against the formulas in float64, what is not there, and what is refused.  The kernels' tests
(test_quant_kv_gpu.py) take their cases from here."""
import math

import pytest
import torch

from chronos import ops
from tests.oracles import quant_kv_plain as plain

KINDS = ("int8", "mxfp4")
BF = torch.bfloat16
HALF = torch.finfo(BF).eps / 2


def table_of(ctx, page, wide=None, spare=3, seed=0):
    """(pages in all, block table): every sequence's pages, their numbers in no order."""
    need = [-(-c // page) for c in ctx]
    names = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    wide = wide or max(1, max(need))
    return sum(need) + spare, torch.tensor([[names.pop() for _ in range(n)] + [0] * (wide - n) for n in need], dtype=torch.int32).reshape(len(ctx), wide)


def filled(pages, page, hkv, D, kind, device="cpu", seed=0, loud=4.0):
    """A cache of normal numbers, a few large channels among the keys."""
    g = torch.Generator().manual_seed(seed)
    cache = ops.quant_kv_cache(pages, page, hkv, D, kind)
    k = torch.randn(pages, hkv, page, D, generator=g) * (1 + (loud - 1) * (torch.rand(D, generator=g) < 0.05))
    v = torch.randn(pages, hkv, page, D, generator=g)
    for codes, scales, x in ((cache.k, cache.ks, k), (cache.v, cache.vs, v)):
        c, s = ops.quant_kv.ref.encode(x.to(BF).double(), kind)
        codes.copy_(c)
        scales.copy_(s)
    return ops.QuantKV(*(t.to(device) for t in (cache.k, cache.v, cache.ks, cache.vs)))


def rows_of(T, heads, D, seed=0):
    return torch.randn(T, heads, D, generator=torch.Generator().manual_seed(100 + seed)).to(BF)


def rope(positions, R, base=10000.0):
    a = torch.outer(torch.arange(positions, dtype=torch.float64), base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R))
    return torch.cat([a.cos(), a.sin()], 1).float()


def starts(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def check_attention(out, q, cache, table, ctx, q_start, scale=None):
    """Half a step of the output's type, half a step for every probability (relative to what they multiply), and 2^-10 for sums in float32: products of 128 dimensions,
    scores of up to 30, are off by 128 * 2^-24 * 30 < 2^-11."""
    want, size = plain.attention(q, cache, table, ctx, q_start, scale)
    off = (out.double().cpu() - want).abs()
    most = HALF * want.abs() + (HALF + 2 ** -10) * size + 1e-30
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want))
    worst = torch.nan_to_num(off / most, nan=0.0).max() if off.numel() else 0.0
    assert worst <= 1, f"{float(worst)} of what roundings allow"


# (kind, D, hq, hkv, page, contexts, tokens of each sequence or None)
ATTENTION = [
    ("int8", 128, 8, 2, 16, [1], None),
    ("mxfp4", 128, 8, 2, 16, [1], None),
    ("int8", 128, 32, 8, 16, [140, 17, 16, 0, 33], None),
    ("mxfp4", 128, 32, 8, 32, [140, 31, 32, 0, 257], None),
    ("int8", 64, 4, 2, 16, [77, 300], None),
    ("mxfp4", 64, 12, 4, 48, [77, 300, 1], None),
    ("int8", 128, 5, 5, 16, [63, 64, 65], None),
    ("mxfp4", 128, 7, 1, 64, [129, 511], None),
    ("int8", 128, 40, 2, 16, [95, 200], None),                  # more query heads per key head than a tile has rows
    ("mxfp4", 64, 34, 1, 16, [95, 200], None),
    ("int8", 128, 8, 2, 16, [50, 7, 3], [5, 7, 0]),             # a whole prompt, a chunk, no token
    ("mxfp4", 128, 8, 2, 16, [50, 7, 3], [5, 7, 3]),
    ("int8", 64, 6, 2, 32, [90, 40], [33, 40]),
    ("mxfp4", 64, 8, 4, 16, [150, 2, 64], [70, 1, 64]),
    ("int8", 128, 16, 4, 16, [4, 30], [9, 2]),                  # more tokens than context: rows in front see nothing
    ("mxfp4", 128, 16, 4, 16, [0, 30], [3, 2]),
]


def attention_case(kind, D, hq, hkv, page, ctx, lens, device="cpu", tail=0, seed=0):
    pages, table = table_of(ctx, page, seed=seed)
    q_start = None if lens is None else starts(lens)
    T = (len(ctx) if lens is None else sum(lens)) + tail
    return rows_of(T, hq, D, seed).mul(2).to(device), filled(pages, page, hkv, D, kind, device, seed), table.to(device), ints(ctx).to(device), \
        None if q_start is None else q_start.to(device)


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(map(str, c[:5])) + f"-{len(c[5])}")
def test_attention_reference(case):
    q, cache, table, ctx, q_start = attention_case(*case, tail=2)
    out = ops.quant_attention(q, cache, table, ctx, q_start)
    check_attention(out, q, cache, table, ctx, q_start)
    assert not out[-2:].any()
    same = ops.prefix_attention(q, cache, table, ctx, ints([0, len(case[5])]), ints([0]), q_start)
    assert torch.equal(same, out)


def edge_rows(D):
    """Rows at borders between codes, of zeros, of very large and small numbers, and with numbers that are none."""
    g = torch.Generator().manual_seed(3)
    r = torch.randn(12, D, generator=g)
    r[0] = 0
    r[1] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 7.0, 1.0, 0.0, -2.5, -3.5, -7.0] * (D // 16))
    r[2] = torch.arange(D) - D / 2 + 0.5
    r[3] *= 1e30
    r[4] *= 1e-30
    r[5, 0] = float("inf")
    r[6, D - 1] = float("nan")
    r[7] = torch.finfo(BF).max
    r[8] = 7.03125          # just over seven scales of one
    r[9, :32] = 0
    r[10] = 1e-39
    r[11] = 127
    r[11, 1::2] = 0.5
    return r.to(BF)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", (64, 128))
def test_codes_of_the_reference(kind, D):
    x = edge_rows(D)
    codes, scales = ops.quant_kv.ref.encode(x.double(), kind)
    want, ws = plain.quantise(x, kind)
    got = codes.long() if kind == "int8" else torch.stack([codes.long() & 15, codes.long() >> 4], -1).flatten(-2)
    assert torch.equal(got, want)
    assert torch.equal(scales.nan_to_num(nan=-1.0) if kind == "int8" else scales.long(), ws.nan_to_num(nan=-1.0) if kind == "int8" else ws)


def write_case(kind, D, hq, hkv, page, R, norm, lens, ctx, seed=0, device="cpu"):
    pages, table = table_of(ctx, page, seed=seed)
    g = torch.Generator().manual_seed(seed)
    pos = torch.cat([torch.arange(c - n, c) for c, n in zip(ctx, lens)]).int()
    seq = torch.repeat_interleave(torch.arange(len(ctx)), torch.tensor(lens)).int()
    qkv = torch.randn(len(pos), (hq + 2 * hkv) * D, generator=g).to(BF)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(BF) if norm else None for _ in "qk")
    return tuple(t.to(device) if t is not None else None for t in (qkv, pos, seq, table, rope(max(ctx) + 1, R), wq, wk)), \
        filled(pages, page, hkv, D, kind, device, seed)


WRITE = [
    ("int8", 128, 8, 2, 16, 128, True, [1], [1]),
    ("mxfp4", 128, 8, 2, 16, 128, True, [1], [140]),
    ("int8", 128, 32, 8, 16, 128, False, [1, 1, 1], [5, 16, 33]),
    ("mxfp4", 128, 4, 4, 32, 64, True, [5, 0, 37], [5, 9, 70]),
    ("int8", 64, 3, 1, 48, 32, True, [50, 2], [50, 49]),
    ("mxfp4", 64, 6, 2, 16, 64, False, [17, 1], [40, 1]),
    ("int8", 128, 0, 2, 16, 16, True, [9], [20]),
]


def check_write(case, device):
    (qkv, pos, seq, table, cs, wq, wk), cache = write_case(*case, device=device)
    kind, D, hq, hkv, page = case[:5]
    before = [t.clone() for t in (cache.k, cache.v, cache.ks, cache.vs)]
    x = qkv.cpu().view(-1, hq + 2 * hkv, D)
    q = ops.norm_rope_kv_quant(qkv, pos, seq, table, cs, cache, hq, wq, wk, eps=1e-5)
    cpu = [None if t is None else t.cpu() for t in (wq, wk)]
    wantq = plain.norm_rotation(x[:, :hq], cpu[0], 1e-5, cs.cpu(), pos.cpu())
    # half a step, and float32 products: two of them and a sum, relative to the larger of the pair
    top = x[:, :hq].double().abs().amax(-1, keepdim=True) if wq is None else \
        wantq.abs().amax(-1, keepdim=True)
    assert ((q.double().cpu() - wantq).abs() <= HALF * wantq.abs() + 2 ** -20 * top).all()
    p = table.cpu()[seq.long().cpu(), pos.long().cpu() // page].long()
    o = pos.long().cpu() % page
    codes = plain.whole_codes(cache)
    for got, scales, y in ((codes[0], cache.ks, plain.norm_rotation(x[:, hq:hq + hkv], cpu[1], 1e-5, cs.cpu(), pos.cpu())), (codes[1], cache.vs, x[:, hq + hkv:])):
        c, s = plain.quantise(y, kind)
        assert torch.equal(scales.cpu()[p, :, o].double(), s.double())
        assert torch.equal(got[p, :, o], c)
    for t, b in zip((cache.k, cache.v, cache.ks, cache.vs), before):       # nothing else is touched
        t, b = t.clone().cpu(), b.cpu()
        t[p, :, o] = b[p, :, o]
        assert torch.equal(t, b)
    k, v = ops.quant_kv_read(cache, table, pos, seq)
    for got, want in zip((k, v), plain.values(cache)):
        assert ((got.double().cpu() - want[p, :, o]).abs() <= HALF * want[p, :, o].abs()).all()


@pytest.mark.parametrize("case", WRITE, ids=lambda c: "-".join(map(str, c[:7])))
def test_write_and_read_reference(case):
    check_write(case, "cpu")


def check_left_out(kind, device):
    """Tokens without a place: padding, pages that the cache or the table does not have, positions behind the rope table."""
    (qkv, pos, seq, table, cs, wq, wk), cache = write_case(kind, 128, 2, 1, 16, 128, True, [8], [40], device=device)
    pos = ints([-1, 35, 36, 37, 200, 38, 39, 5]).to(device)       # 200: outside the table; 39: behind the rope table
    seq = ints([0, -1, 3, 0, 0, 0, 0, 0]).to(device)
    table[0, 0] = cache.k.shape[0]                                # token 5's page: one behind the last
    cs = cs[:39].contiguous()
    before = [t.clone() for t in (cache.k, cache.v, cache.ks, cache.vs)]
    q = ops.norm_rope_kv_quant(qkv, pos, seq, table, cs, cache, 2, wq, wk)
    live = [3, 5]
    assert [i for i in range(8) if q[i].any()] == live
    k, v = ops.quant_kv_read(cache, table, pos, seq)
    assert [i for i in range(8) if k[i].any() and v[i].any()] == [3, 5, 6] and not k[[0, 1, 2, 4, 7]].any()
    blk = int(table[0, 2])
    for t, b in zip((cache.k, cache.v, cache.ks, cache.vs), before):
        t[blk, :, 5:7] = b[blk, :, 5:7]
        assert torch.equal(t, b)


@pytest.mark.parametrize("kind", KINDS)
def test_tokens_without_a_place(kind):
    check_left_out(kind, "cpu")


def check_not_numbers(kind, device):
    """Infinities and NaN: a row of the cache is NaN as a whole, on reading and for rows that see it, and for no others."""
    ctx, page, D, hkv = [37, 40], 16, 128, 2
    pages, table = table_of(ctx, page)
    cache, table = filled(pages, page, hkv, D, kind, device), table.to(device)
    x = torch.randn(3, 6, D).to(BF)
    x[0, 2, 7], x[1, 5, 100] = float("nan"), float("-inf")        # key head 0 of the first token, value head 1 of the second; no query among them
    pos, seq = ints([20, 30, 36]).to(device), ints([0, 0, 0]).to(device)
    ops.norm_rope_kv_quant(x.flatten(1).to(device), pos, seq, table, rope(64, D).to(device), cache, 2)
    k, v = ops.quant_kv_read(cache, table, pos, seq)
    assert torch.isnan(k[0, 0]).all() and torch.isnan(v[1, 1]).all()
    assert torch.isfinite(k[1:]).all() and torch.isfinite(k[0, 1]).all() and torch.isfinite(v[[0, 2]]).all() and torch.isfinite(v[1, 0]).all()
    q, q_start = rows_of(37 + 2, 4, D).to(device), ints([0, 37, 39]).to(device)
    out = ops.quant_attention(q, cache, table, ints(ctx).to(device), q_start)
    check_attention(out, q, cache, table, ints(ctx), q_start)
    bad = torch.isnan(out).any(-1).cpu()
    assert bad[20:37, :2].all() and not bad[:20].any() and bad[30:37, 2:].all() and not bad[20:30, 2:].any() and not bad[37:].any()
    # behind the context's end, in its last page, and in pages of nobody
    out = ops.quant_attention(q[:2], cache, table, ints([20, 40]).to(device))
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("kind", KINDS)
def test_not_numbers(kind):
    check_not_numbers(kind, "cpu")


def check_missing_pages(kind, device):
    ctx, page = [100, 64, 40], 16
    q, cache, table, ctx, _ = attention_case(kind, 128, 8, 2, page, ctx, None, device)
    table[0, 2], table[0, 6] = -1, cache.k.shape[0]               # a hole, and the page of the last keys
    table[2] = -(1 << 31)                                         # nothing left
    out = ops.quant_attention(q, cache, table, ctx)
    check_attention(out, q, cache, table, ctx.cpu(), None)
    assert not out[2].any() and out[0].any()
    out = ops.quant_attention(q, cache, table, ints([1 << 30, -5, 7]).to(device))      # as far as the table goes; none; nothing left
    check_attention(out, q, cache, table, ints([table.shape[1] * page, 0, 0]), None)


@pytest.mark.parametrize("kind", KINDS)
def test_pages_that_are_not_there(kind):
    check_missing_pages(kind, "cpu")


def check_refusals(device):
    (qkv, pos, seq, table, cs, wq, wk), cache = write_case("int8", 128, 4, 2, 16, 128, True, [3, 2], [20, 30], device=device)
    four = ops.quant_kv_cache(2, 16, 2, 128, "mxfp4", device)
    q, ctx = torch.zeros(2, 4, 128, dtype=BF, device=device), ints([20, 30]).to(device)
    gs, pl = ints([0, 2]).to(device), ints([16]).to(device)
    C = ops.QuantKV

    def no(match, fn, *a, **k):
        with pytest.raises(RuntimeError, match=match):
            fn(*a, **k)

    write, read, attend, prefix = ops.norm_rope_kv_quant, ops.quant_kv_read, ops.quant_attention, ops.prefix_attention
    no("kind must be", ops.quant_kv_cache, 1, 16, 1, 128, "int4", device)
    no("64 or 128", ops.quant_kv_cache, 1, 16, 1, 96, "int8", device)
    no("multiple of 16 tokens", ops.quant_kv_cache, 1, 8, 1, 128, "int8", device)
    no("int8 codes or uint8", attend, q, C(cache.k.float(), cache.v, cache.ks, cache.vs), table, ctx)
    no("of one type", attend, q, C(cache.k, four.v, cache.ks, cache.vs), table, ctx)
    no("scales must be float32", attend, q, C(cache.k, cache.v, four.ks, four.vs), table, ctx)
    no("scales must be", attend, q, C(cache.k, cache.v, cache.ks[:, :1].contiguous(), cache.vs), table, ctx)
    no("contiguous", attend, q, C(cache.k.transpose(0, 1).contiguous().transpose(0, 1), cache.v, cache.ks, cache.vs), table, ctx)
    no("q must be", attend, q.float(), cache, table, ctx)
    no("q must be", attend, q[..., :64], cache, table, ctx)
    no("multiple of the cache's", attend, q[:, :3], cache, table, ctx)
    no("block_table must be", attend, q, cache, table.long(), ctx)
    no("row per sequence", attend, q, cache, table[:1], ctx)
    no("ctx_len must be", attend, q, cache, table, ctx.long())
    no("q_start needs 3", attend, q, cache, table, ctx, ctx)
    no("every sequence has a token", attend, q[:1], cache, table, ctx)
    no("group_start needs 2", prefix, q, cache, table, ctx, gs[:1], pl)
    no("prefix_len must be", prefix, q, cache, table, ctx, gs, pl.long())
    no("has rows of", write, qkv, pos, seq, table, cs, cache, 5)
    no("qkv must be bfloat16", write, qkv.float(), pos, seq, table, cs, cache, 4)
    no("entry per token", write, qkv, pos[:-1], seq, table, cs, cache, 4)
    no("pos must be", write, qkv, pos.long(), seq, table, cs, cache, 4)
    no("cos_sin must be", write, qkv, pos, seq, table, cs[:, :24].contiguous(), cache, 4)
    no("cos_sin must be", write, qkv, pos, seq, table, cs.double(), cache, 4)
    no("cos_sin has no positions", write, qkv, pos, seq, table, cs[:0], cache, 4)
    no("k_norm must be", write, qkv, pos, seq, table, cs, cache, 4, wq, wk[:64])
    no("eps must not", write, qkv, pos, seq, table, cs, cache, 4, wq, wk, eps=-1.0)
    no("entry per token", read, cache, table, pos, seq[:-1])
    no("block_table must be", read, cache, table[0], pos, seq)
    if device != "cpu":
        no("must be on", attend, q, cache, table.cpu(), ctx)
        no("must be on", write, qkv, pos.cpu(), seq, table, cs, cache, 4)
        no("must be on", read, cache, table, pos, seq.cpu())


def test_refusals():
    check_refusals("cpu")


def test_nothing_to_do():
    check_nothing("cpu")


def check_nothing(device):
    cache = ops.quant_kv_cache(1, 16, 1, 64, "mxfp4", device)
    none, table = ints([]).to(device), torch.zeros(0, 1, dtype=torch.int32, device=device)
    cs = rope(4, 64).to(device)
    assert ops.norm_rope_kv_quant(torch.zeros(0, 192, dtype=BF, device=device), none, none, table, cs, cache, 1).shape == (0, 1, 64)
    assert ops.quant_kv_read(cache, table, none, none)[0].shape == (0, 1, 64)
    assert ops.quant_attention(torch.zeros(0, 2, 64, dtype=BF, device=device), cache, table, none).shape == (0, 2, 64)
    out = ops.quant_attention(torch.ones(3, 2, 64, dtype=BF, device=device), cache, table, none, ints([0]).to(device))
    assert out.shape == (3, 2, 64) and not out.any()
    out = ops.quant_attention(torch.ones(3, 2, 64, dtype=BF, device=device), cache, torch.zeros(3, 0, dtype=torch.int32, device=device), ints([4, 4, 4]).to(device))
    assert not out.any()
    assert cache.nbytes() == 16 * 2 * (32 + 2) and cache.kind == "mxfp4" and math.prod(cache.k.shape) == 16 * 32
