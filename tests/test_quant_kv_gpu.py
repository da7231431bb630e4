"""The kernels of a key/value cache in 8 or 4 bits (csrc/kernels/quant_kv.hip, quant_attention.hip) against float64: the cases of test_quant_kv.py, and what only a
GPU has: streams, graphs, strides, offsets past 32 bits, every form that the rules choose."""
import pytest
import torch

from chronos import ops
from tests import test_quant_kv as t
from tests.oracles import quant_kv_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def cpu(cache):
    return ops.QuantKV(cache.k.cpu(), cache.v.cpu(), cache.ks.cpu(), cache.vs.cpu())


@pytest.mark.parametrize("case", t.WRITE, ids=lambda c: "-".join(map(str, c[:7])))
def test_write_and_read(case):
    t.check_write(case, DEV)


@pytest.mark.parametrize("kind", t.KINDS)
@pytest.mark.parametrize("D", (64, 128))
def test_codes_at_borders(kind, D):
    """Values go to their codes as they are; keys at position 0 too."""
    x = t.edge_rows(D)
    x = torch.cat([x, x], 1)                                   # one key head, one value head
    cache = ops.quant_kv_cache(1, 16, 1, D, kind, DEV)
    n = len(x)
    zero = torch.zeros(n, dtype=torch.int32, device=DEV)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    cs = torch.cat([torch.ones(16, D // 2), torch.zeros(16, D // 2)], 1).to(DEV)
    ops.norm_rope_kv_quant(x.to(DEV), torch.arange(n, dtype=torch.int32, device=DEV), zero, table, cs, cache, 0)
    rows = torch.arange(n) != 6 if kind == "int8" else torch.arange(n) >= 0
    codes, (c, s) = plain.whole_codes(cache), plain.quantise(x[:, D:], kind)
    turned = plain.quantise(torch.where(torch.isfinite(x[:, :D]).all(1, keepdim=True), x[:, :D].double(), float("nan")), kind)
    for got, scales, (want, ws) in ((codes[1], cache.vs, (c, s)), (codes[0], cache.ks, turned)):
        assert torch.equal(got[0, 0, :n][rows], want[rows])
        assert torch.equal(scales[0, 0, :n].cpu().double().nan_to_num(nan=-1), ws.double().nan_to_num(nan=-1))


@pytest.mark.parametrize("kind", t.KINDS)
def test_tokens_without_a_place(kind):
    t.check_left_out(kind, DEV)


@pytest.mark.parametrize("kind", t.KINDS)
def test_not_numbers(kind):
    t.check_not_numbers(kind, DEV)


@pytest.mark.parametrize("kind", t.KINDS)
def test_pages_that_are_not_there(kind):
    t.check_missing_pages(kind, DEV)


def test_refusals():
    t.check_refusals(DEV)


def test_nothing_to_do():
    t.check_nothing(DEV)


MORE = [
    ("int8", 128, 32, 8, 16, [3000, 700, 5], None),             # pieces of the keys
    ("mxfp4", 128, 64, 8, 16, [2500], None),
    ("mxfp4", 64, 8, 2, 64, [1999, 2000], [3, 1]),
    ("int8", 64, 16, 1, 32, [1200], [9]),                       # 144 rows of one key head
    ("int8", 128, 8, 2, 16, [400, 700], [300, 129]),            # prompts
    ("mxfp4", 128, 8, 1, 16, [333, 257, 90], [333, 128, 1]),
    ("int8", 64, 8, 8, 48, [300], [299]),
    ("mxfp4", 64, 32, 4, 16, [260, 40], [250, 40]),
    ("int8", 128, 8, 1, 16, [2100], [40]),                      # tiles of 256 rows
    ("mxfp4", 64, 16, 2, 32, [2050, 2100], [35, 33]),
    ("int8", 64, 16, 1, 16, [2049], [20]),
    ("int8", 128, 8, 2, 16, [1 + 97 * i % 1500 for i in range(20)] + [0, 1500], None),      # lengths far apart
    ("mxfp4", 64, 8, 4, 16, [(31 * i * i) % 700 for i in range(150)], None),
    ("mxfp4", 128, 16, 2, 64, [20] * 30 + [3000], None),
]


@pytest.mark.parametrize("case", t.ATTENTION + MORE, ids=lambda c: "-".join(map(str, c[:5])) + f"-{max(c[5])}-{len(c[5])}-{max(c[6] or [0])}")
def test_attention(case):
    q, cache, table, ctx, q_start = t.attention_case(*case, DEV, tail=3)
    out = ops.quant_attention(q, cache, table, ctx, q_start)
    t.check_attention(out, q, cpu(cache), table, ctx.cpu(), None if q_start is None else q_start.cpu())
    assert not out[-3:].any()
    assert torch.equal(out, ops.quant_attention(q, cache, table, ctx, q_start))


# the other forms that the rules choose, by heads rather than rows
FORMS = [
    ("mxfp4", 64, 64, 64, 16, [800, 31], [300, 30]),            # tiles of 256 rows, the keys in two pieces
    ("int8", 128, 32, 32, 16, [900], [900]),
    ("int8", 64, 64, 64, 32, [700], [600]),                     # in one
    ("int8", 128, 16, 8, 16, [5000] + [37 * i % 300 for i in range(20)], None),             # lengths far apart
    ("mxfp4", 64, 8, 4, 16, [4100] + [1 + 91 * i % 1300 for i in range(39)], None),
    ("int8", 128, 8, 1, 64, [300] * 140 + [17000, 0, 9000], None),
    ("int8", 64, 16, 8, 64, [4100] + [100 + i for i in range(29)], [1 + i % 2 for i in range(30)]),      # two pieces
    ("mxfp4", 128, 16, 8, 32, [500] * 28, [9 + i % 3 for i in range(28)]),                  # 32 rows
]


@pytest.mark.parametrize("case", FORMS, ids=lambda c: "-".join(map(str, c[:5])) + f"-{max(c[5])}-{len(c[5])}")
def test_forms(case):
    q, cache, table, ctx, q_start = t.attention_case(*case, DEV, tail=3)
    out = ops.quant_attention(q, cache, table, ctx, q_start)
    t.check_attention(out, q, cpu(cache), table, ctx.cpu(), None if q_start is None else q_start.cpu())
    assert not out[-3:].any()


# more tiles than the card holds at a time, which go by their lengths: (kind, D, hq, hkv, page, contexts, tokens, keys that the table has room for)
LONGEST = [
    ("int8", 64, 64, 64, 16, [300, 0, 517, 129, 64, 700], [300, 0, 260, 129, 5, 600], 0),
    ("mxfp4", 64, 128, 32, 32, [400, 90, 33], [333, 90, 133], 2080),       # tiles of 256 rows
    ("mxfp4", 128, 64, 64, 16, [7, 250] + [(37 * i) % 200 for i in range(70)], [9, 40] + [(37 * i) % 200 // 3 + 5 for i in range(70)], 0),   # more tokens than context, too
    ("int8", 128, 96, 32, 16, [(53 * i) % 97 for i in range(254)] + [300], [11] * 255, 0),      # as many sequences as there may be
]


@pytest.mark.parametrize("case", LONGEST, ids=lambda c: "-".join(map(str, c[:5])) + f"-{len(c[5])}")
def test_longest_first(case):
    q, cache, table, ctx, q_start = t.attention_case(*case[:7], DEV, tail=3)
    wide = torch.zeros(table.shape[0], max(table.shape[1], case[7] // case[4]), dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    out = ops.quant_attention(q, cache, wide, ctx, q_start)
    t.check_attention(out, q, cpu(cache), table, ctx.cpu(), q_start.cpu())
    assert not out[-3:].any()


@pytest.mark.parametrize("lens", (None, [1, 90]), ids=("rows", "tiles"))
@pytest.mark.parametrize("D", (64, 128))
def test_scales_far_apart(D, lens):
    """int8: value scales that grow and shrink by orders of magnitude along the keys, and scores that grow all the way, so that every step moves the maximum."""
    q, cache, table, ctx, q_start = t.attention_case("int8", D, 8, 2, 16, [420, 400], lens, DEV)
    at = torch.arange(cache.vs.numel(), device=DEV).view(cache.vs.shape)
    cache.vs.mul_(torch.exp2(((at * 37) % 61 - 30).float()))
    cache.vs[table[1, 3].long()] = 0                            # values of nothing
    for b in range(2):
        for i, p in enumerate(table[b, :-(-int(ctx[b]) // 16)].tolist()):
            cache.ks[p] *= 1 + i
    out = ops.quant_attention(q, cache, table, ctx, q_start)
    want, size = plain.attention(q.cpu(), cpu(cache), table.cpu(), ctx.cpu(), None if q_start is None else q_start.cpu())
    # Scores of up to 30 * 27: off by 2^-11 * 27 relative to the probabilities, and the roundings as ever.  Probabilities times scales are float16, a row's largest, W, at
    # 2^7 or more: each is off by up to half of float16's least step, 2^-25 = 2^-32 W, times a code of up to 127; the largest's row has a code of 127, so 127 W is
    # no more than the largest of the row's sizes.
    least = 420 * 2 ** -32 * size.amax(-1, keepdim=True)
    assert ((out.double().cpu() - want).abs() <= t.HALF * want.abs() + (t.HALF + 2 ** -6) * size + least + 1e-30).all()
    cache.vs.fill_(0)
    assert not ops.quant_attention(q, cache, table, ctx, q_start).any()


@pytest.mark.parametrize("kind", t.KINDS)
def test_tables_wider_than_contexts(kind):
    """Work is cut up by the table, or by max_ctx; how codes are read (marked, from 192 MiB on) changes nothing."""
    q, cache, table, ctx, _ = t.attention_case(kind, 128, 8, 2, 16, [500, 33], None, DEV)
    want = ops.quant_attention(q, cache, table, ctx)
    wide = torch.zeros(2, 40000, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    assert torch.equal(want, ops.quant_attention(q, cache, wide, ctx, max_ctx=table.shape[1] * 16))
    t.check_attention(ops.quant_attention(q, cache, wide, ctx), q, cpu(cache), table, ctx.cpu(), None)


# (kind, D, hq, hkv, page, whole shared pages of each group, sequences of each group, own tokens, tokens of each or None, sequences before and behind the groups)
PREFIX = [
    ("int8", 128, 8, 2, 16, [3], [4], [1, 20, 16, 33], None, 0),
    ("mxfp4", 128, 32, 8, 32, [4], [9], [5, 40, 1, 2, 3, 64, 7, 8, 9], [3, 1, 2, 3, 3, 3, 1, 1, 2], 0),
    ("int8", 128, 4, 4, 16, [20, 0, 7], [5, 3, 0], [9, 1, 30, 2, 17, 4, 5, 6], None, 2),
    ("mxfp4", 64, 12, 4, 48, [5, 2], [2, 6], [9, 100, 30, 2, 17, 4, 5, 6], None, 1),
    ("int8", 64, 34, 1, 16, [40], [7], [1, 2, 3, 4, 5, 6, 7], [1, 2, 3, 1, 1, 1, 0], 0),
    ("mxfp4", 128, 8, 1, 16, [150], [40], [1 + i % 29 for i in range(40)], None, 0),
    ("int8", 128, 8, 1, 16, [64], [30], [8 + i % 29 for i in range(30)], [1 + i % 8 for i in range(30)], 3),
    ("mxfp4", 64, 16, 2, 16, [10], [20], [4] * 20, [40] * 20, 0),   # prompts longer than their own keys: rows whose last key is a shared one
    ("int8", 64, 16, 2, 16, [1] * 70, [1, 2] * 35, [1 + i % 40 for i in range(105)], None, 2),   # more groups than a wave has lanes
]


def prefix_case(kind, D, hq, hkv, page, whole, seqs, own, lens, more, seed=0):
    shared = [g for g, n in enumerate(seqs) for _ in range(n)]
    ctx = [whole[g] * page + o for g, o in zip(shared, own)]
    extra = [50 + 7 * i for i in range(2 * more)]
    ctx = extra[:more] + ctx + extra[more:]
    pages, table = t.table_of(ctx, page, seed=seed)
    at = more
    group_start = [more]
    for g, n in enumerate(seqs):
        table[at:at + n, :whole[g]] = table[at:at + 1, :whole[g]]
        at += n
        group_start.append(at)
    if lens is not None:
        lens = [1] * more + lens + [2] * more
    q = t.rows_of(len(ctx) if lens is None else sum(lens), hq, D, seed).mul(2)
    return (x.to(DEV) if x is not None else None for x in (q, table, t.ints(ctx), t.ints(group_start), t.ints([w * page for w in whole]),
                                                           None if lens is None else t.starts(lens))), t.filled(pages, page, hkv, D, kind, DEV, seed)


@pytest.mark.parametrize("case", PREFIX, ids=lambda c: "-".join(map(str, c[:5])) + f"-{max(c[5])}-{len(c[7])}")
def test_prefix(case):
    (q, table, ctx, groups, prefix, q_start), cache = prefix_case(*case)
    out = ops.prefix_attention(q, cache, table, ctx, groups, prefix, q_start)
    t.check_attention(out, q, cpu(cache), table, ctx.cpu(), None if q_start is None else q_start.cpu())
    assert torch.equal(out, ops.prefix_attention(q, cache, table, ctx, groups, prefix + case[4] - 1, q_start))    # whole pages only
    alone = ops.prefix_attention(q, cache, table, ctx, groups[:1], prefix[:0], q_start)                           # no groups
    assert torch.equal(alone, ops.quant_attention(q, cache, table, ctx, q_start))


PREFIX_FORMS = [
    ("int8", 128, 32, 16, 16, [40], [100], [1 + i % 29 for i in range(100)], None, 1),      # tiles of 128 rows
    ("mxfp4", 64, 64, 32, 16, [40], [60], [1 + i % 29 for i in range(60)], None, 2),        # of 256
    ("int8", 64, 64, 32, 32, [9, 20], [40, 30], [3 + i % 29 for i in range(70)], [1 + i % 3 for i in range(70)], 0),
    ("mxfp4", 128, 32, 8, 16, [50], [40], [1 + i % 29 for i in range(40)], None, 0),        # of 32
    ("int8", 64, 64, 64, 16, [3], [3], [200, 160, 170], [150, 150, 160], 1),                # the own keys' of 256
]


@pytest.mark.parametrize("case", PREFIX_FORMS, ids=lambda c: "-".join(map(str, c[:5])) + f"-{max(c[5])}-{len(c[7])}")
def test_prefix_forms(case):
    (q, table, ctx, groups, prefix, q_start), cache = prefix_case(*case)
    out = ops.prefix_attention(q, cache, table, ctx, groups, prefix, q_start)
    t.check_attention(out, q, cpu(cache), table, ctx.cpu(), None if q_start is None else q_start.cpu())


@pytest.mark.parametrize("kind", t.KINDS)
def test_prefix_longer_than_contexts(kind):
    """Contexts that end inside the shared pages, or have none; an empty sequence; pages that are not there."""
    (q, table, ctx, groups, prefix, _), cache = prefix_case(kind, 128, 8, 2, 16, [6], [6], [1, 2, 3, 40, 5, 6], None, 1)
    ctx[1], ctx[2], ctx[3] = 17, 0, 96
    table[1:7, 4] = -1
    out = ops.prefix_attention(q, cache, table, ctx, groups, prefix)
    t.check_attention(out, q, cpu(cache), table, ctx.cpu(), None)
    assert not out[2].any()


@pytest.mark.parametrize("kind", t.KINDS)
def test_not_numbers_in_a_prefix(kind):
    (q, table, ctx, groups, prefix, _), cache = prefix_case(kind, 128, 8, 2, 16, [6], [6], [1, 2, 3, 40, 5, 6], None, 1)
    ctx[1] = 50
    cache.vs[int(table[1, 3]), 1, 7] = float("nan") if kind == "int8" else 255      # token 55, value head 1
    out = ops.prefix_attention(q, cache, table, ctx, groups, prefix)
    bad = torch.isnan(out).all(-1)
    assert bad[2:7, 4:].all() and not torch.isnan(out[:, :4]).any() and not torch.isnan(out[:2]).any() and not torch.isnan(out[7:]).any()


def test_strides():
    """Rows of a wider projection, queries that are a slice or lie across, tables that are a slice, weights that start off the 16 bytes."""
    q, cache, table, ctx, q_start = t.attention_case("int8", 128, 8, 2, 16, [90, 33], [4, 2], DEV)
    want = ops.quant_attention(q, cache, table, ctx, q_start)
    wide = torch.zeros(6, 12, 128, dtype=q.dtype, device=DEV)
    wide[:, :8] = q
    off = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)
    off[1:] = q.flatten()
    long_table = torch.full((5, 40), -7, dtype=torch.int32, device=DEV)
    long_table[1:3, 3:3 + table.shape[1]] = table
    for other in (wide[:, :8], off[1:].view(q.shape), q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert not other.is_contiguous() or other.data_ptr() % 16
        assert torch.equal(want, ops.quant_attention(other, cache, long_table[1:3, 3:3 + table.shape[1]], ctx, q_start))
    assert torch.equal(want, ops.quant_attention(q, cache, table, ctx, q_start, max_ctx=90))
    (qkv, pos, seq, table, cs, wq, wk), cache = t.write_case("mxfp4", 64, 4, 2, 16, 64, True, [7, 2], [20, 30], device=DEV)
    want = ops.norm_rope_kv_quant(qkv, pos, seq, table, cs, cache, 4, wq, wk)
    kept = [x.clone() for x in (cache.k, cache.v, cache.ks, cache.vs)]
    weights = torch.zeros(130, dtype=wq.dtype, device=DEV)
    weights[1:65], weights[65:129] = wq, wk
    for pad, lead in ((8, 0), (3, 0), (5, 1)):
        wide = torch.randn(9, qkv.shape[1] + pad, device=DEV).to(qkv.dtype)
        wide[:, lead:lead + qkv.shape[1]] = qkv
        got = ops.norm_rope_kv_quant(wide[:, lead:lead + qkv.shape[1]], pos, seq, table, cs, cache, 4, weights[1:65], weights[65:129])
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(kept, (cache.k, cache.v, cache.ks, cache.vs)))


def chain(qkv, pos, seq, table, cs, cache, hq, norms, ctx, q_start, groups, prefix):
    q = ops.norm_rope_kv_quant(qkv, pos, seq, table, cs, cache, hq, *norms)
    return q, ops.quant_attention(q, cache, table, ctx, q_start), ops.prefix_attention(q, cache, table, ctx, groups, prefix, q_start), \
        *ops.quant_kv_read(cache, table, pos, seq)


def chain_case(kind, seed=0, seqs=5, D=128, hq=8, hkv=2, page=16):
    (q, table, ctx, groups, prefix, _), cache = prefix_case(kind, D, hq, hkv, page, [9], [seqs], [3 + 5 * i for i in range(seqs)], None, 0, seed)
    lens = [1 + i % 3 for i in range(seqs)]
    q_start = t.starts(lens).to(DEV)
    seq = torch.repeat_interleave(torch.arange(seqs), torch.tensor(lens)).int().to(DEV)
    pos = torch.cat([torch.arange(c - n, c) for c, n in zip(ctx.tolist(), lens)]).int().to(DEV)
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(len(pos), (hq + 2 * hkv) * D, generator=g).to(torch.bfloat16).to(DEV)
    norms = [(1 + 0.3 * torch.randn(D, generator=g)).to(torch.bfloat16).to(DEV) for _ in "qk"]
    return qkv, pos, seq, table, t.rope(400, D).to(DEV), cache, hq, norms, ctx, q_start, groups, prefix


@pytest.mark.parametrize("kind", t.KINDS)
def test_run_together(kind):
    """A step as it is used: written, attended to both ways, read back."""
    case = chain_case(kind)
    q, out, shared, k, v = chain(*case)
    qkv, pos, seq, table, cs, cache, hq, norms, ctx, q_start, groups, prefix = case
    for o in (out, shared):
        t.check_attention(o, q, cpu(cache), table, ctx.cpu(), q_start.cpu())
    x = qkv.cpu().view(len(pos), -1, 128)
    turned = plain.norm_rotation(x[:, hq:hq + 2], norms[1].cpu(), 1e-6, cs.cpu(), pos.cpu())
    for got, want in ((k, turned), (v, x[:, hq + 2:].double())):
        codes, s = plain.quantise(want, kind)
        held = codes.double() * s.double()[..., None] if kind == "int8" else \
            torch.tensor(plain.GRID + tuple(-g for g in plain.GRID), dtype=torch.float64)[codes] * (2.0 ** (s.double() - 127)).repeat_interleave(32, -1)
        assert ((got.double().cpu() - held).abs() <= t.HALF * held.abs()).all()


def test_other_stream_and_graphs():
    """The chain on a stream of its own, and captured twice; replays among eager work, every one against the eager result."""
    cases = [chain_case("int8", 1), chain_case("mxfp4", 2, seqs=9)]
    want = [[x.clone() for x in chain(*c)] for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [chain(*c) for c in cases]
    side.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(*c))
        graphs.append(g)
    for turn in range(3):
        for c in cases:                                        # other inputs in the same tensors
            c[0].copy_(torch.randn(c[0].shape, generator=torch.Generator().manual_seed(turn)).to(c[0].dtype))
        for i in (0, 1):
            graphs[i].replay()
        torch.cuda.synchronize()
        got = [[x.clone() for x in o] for o in outs]
        for x, c in zip(got, cases):
            assert all(torch.equal(a, b) for a, b in zip(x, chain(*c)))


@pytest.mark.parametrize("kind,D", (("int8", 128), ("mxfp4", 64)))
def test_offsets_past_32_bits(kind, D):
    """A cache whose codes are more than 2^32 bytes: the last pages."""
    row = D if kind == "int8" else D // 2
    pages = (1 << 32) // (8 * 16 * row) + 40
    cache = ops.QuantKV(*(torch.empty(pages, 8, 16, row, dtype=torch.int8 if kind == "int8" else torch.uint8, device=DEV) for _ in "kv"),
                        *(torch.empty((pages, 8, 16) + (() if kind == "int8" else (D // 32,)), dtype=torch.float32 if kind == "int8" else torch.uint8, device=DEV) for _ in "kv"))
    small = t.filled(40, 16, 8, D, kind, DEV)
    for a, b in zip((cache.k, cache.v, cache.ks, cache.vs), (small.k, small.v, small.ks, small.vs)):
        a[-40:] = b
    table, ctx = torch.randperm(40).int().view(2, 20).to(DEV), t.ints([300, 311]).to(DEV)
    far = table + (pages - 40)
    q = t.rows_of(2, 32, D).to(DEV)
    assert torch.equal(ops.quant_attention(q, cache, far, ctx), ops.quant_attention(q, small, table, ctx))
    pos, seq = t.ints([299, 310]).to(DEV), t.ints([0, 1]).to(DEV)
    x, cs = t.rows_of(2, 32 + 16, D, 5).flatten(1).to(DEV), t.rope(400, D).to(DEV)
    got, want = (ops.norm_rope_kv_quant(x, pos, seq, tb, cs, c, 32) for tb, c in ((far, cache), (table, small)))
    assert torch.equal(got, want)
    for a, b in zip(ops.quant_kv_read(cache, far, pos, seq), ops.quant_kv_read(small, table, pos, seq)):
        assert torch.equal(a, b)
    for a, b in zip((cache.k, cache.v, cache.ks, cache.vs), (small.k, small.v, small.ks, small.vs)):
        assert torch.equal(a[-40:], b)


def test_more_tokens_than_a_launch_has():
    """2^24 tokens and some, most of them padding; and for the attention, which takes fewer, a refusal before anything is made."""
    n, D = (1 << 24) + 3, 64
    cache = ops.quant_kv_cache(2, 16, 1, D, "int8", DEV)
    qkv = torch.zeros(n, 2 * D, dtype=torch.bfloat16, device=DEV)
    pos, seq = torch.full((n,), -1, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    table, cs = t.ints([[1, 0]]).to(DEV), t.rope(32, D).to(DEV)
    live = [0, 1 << 23, (1 << 23) + 1, n - 1]
    x = t.rows_of(4, 2, D).flatten(1).to(DEV)
    pos[live], qkv[live] = t.ints([3, 17, 4, 30]).to(DEV), x
    assert ops.norm_rope_kv_quant(qkv, pos, seq, table, cs, cache, 0).shape == (n, 0, D)
    small = ops.quant_kv_cache(2, 16, 1, D, "int8", DEV)
    ops.norm_rope_kv_quant(x, pos[live], seq[:4], table, cs, small, 0)
    assert all(torch.equal(a, b) for a, b in zip((cache.k, cache.v, cache.ks, cache.vs), (small.k, small.v, small.ks, small.vs))) and cache.k.any()
    q = torch.zeros(1, 1, D, dtype=torch.bfloat16, device=DEV).expand(n, 1, D)
    with pytest.raises(RuntimeError, match="too many tokens or sequences"):
        ops.quant_attention(q, cache, table.expand(n, 2), seq)
    with pytest.raises(RuntimeError, match="too many tokens or sequences"):
        ops.quant_attention(q.expand(n, 16, D), cache, table, seq[:1], t.ints([0, n]).to(DEV))


def test_contexts_of_less_than_nothing():
    """The least number that a length can be, in a group and outside: rows that see nothing."""
    (q, table, ctx, groups, prefix, q_start), cache = prefix_case("int8", 128, 8, 2, 16, [6], [4], [9, 2, 3, 40], [3, 2, 1, 3], 1)
    want = ops.prefix_attention(q, cache, table, ctx, groups, prefix, q_start)
    ctx[0] = ctx[2] = -(1 << 31)
    got = ops.prefix_attention(q, cache, table, ctx, groups, prefix, q_start)
    rows = q_start.tolist()
    for b in range(6):
        a, e = rows[b], rows[b + 1]
        assert not got[a:e].any() if b in (0, 2) else torch.equal(got[a:e], want[a:e])
