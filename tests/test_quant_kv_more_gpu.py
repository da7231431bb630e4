"""The kernels of a key/value cache in 8 or 4 bits at the ends of their ranges, in every form that the rules choose (csrc/kernels/quant_kv.hip, quant_attention.hip)."""
import pytest
import torch

from chronos import ops
from tests import test_quant_kv as t
from tests import test_quant_kv_gpu as g
from tests import test_quant_kv_more as m

pytestmark = pytest.mark.gpu
DEV = "cuda"
cpu = g.cpu

OWN, SHARED = m.OWN, m.SHARED


def widened(table, keys, page):
    wide = torch.zeros(table.shape[0], max(table.shape[1], -(-keys // page)), dtype=torch.int32, device=table.device)
    wide[:, :table.shape[1]] = table
    return wide


def own_case(form, kind, D):
    """q, cache, table, ctx, q_start, the table as wide as the form asks; three rows behind the last sequence."""
    hq, hkv, page, ctx, lens, keys, _ = OWN[form]
    q, cache, table, ctx, q_start = t.attention_case(kind, D, hq, hkv, page, ctx, lens, DEV, tail=3)
    poison()
    return q, cache, table, ctx, q_start, widened(table, keys, page)


def shared_case(form, kind, D):
    """q, cache, table, ctx, groups, prefix, q_start, the wide table."""
    *case, keys, _ = SHARED[form]
    (q, table, ctx, groups, prefix, q_start), cache = g.prefix_case(kind, D, *case)
    q = torch.cat([q, t.rows_of(3, q.shape[1], D, 7).to(DEV)])
    poison()
    return q, cache, table, ctx, groups, prefix, q_start, widened(table, keys, case[2])


def poison():
    """What the allocator hands out next holds NaN: partial sums that nobody wrote show."""
    for n in (1 << 16, 1 << 20, 1 << 22, 1 << 24, 1 << 26):
        torch.full((n,), float("nan"), device=DEV)


@pytest.mark.parametrize("form", OWN)
def test_plans(form):
    hq, hkv, page, ctx, lens, keys, want = OWN[form]
    T = (len(ctx) if lens is None else sum(lens)) + 3
    assert m.plan(T, len(ctx), lens is None, 0, hq, hkv, -(-max(max(ctx), keys) // page) * page) == want


@pytest.mark.parametrize("form", SHARED)
def test_shared_plans(form):
    hq, hkv, page, pages, seqs, own, lens, more, keys, want = SHARED[form]
    ctx = [50 + 7 * i for i in range(2 * more)] + [pages[g] * page + o for g, o in zip([g for g, n in enumerate(seqs) for _ in range(n)], own)]
    T = (len(ctx) if lens is None else 3 * more + sum(lens)) + 3
    assert m.plan(T, len(ctx), lens is None, len(seqs), hq, hkv, -(-max(max(ctx), keys) // page) * page) == want


def test_plans_that_cannot_be():
    ops.load()
    for bad in ((0, 1, True, 0, 8, 2, 100), (1, 0, True, 0, 8, 2, 100), (1, 1, True, -1, 8, 2, 100), (1, 1, True, 0, 8, 3, 100), (1, 1, True, 0, 8, 0, 100), (1, 1, True, 0, 8, 2, 0)):
        with pytest.raises(RuntimeError, match="chronos"):
            torch.ops.chronos.quant_attention_plan(*bad)


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", OWN)
def test_values_at_the_end_of_the_range(form, D):
    q, cache, table, ctx, q_start, wide = own_case(form, "mxfp4", D)
    m.check_loud(q, cache, table, ctx, q_start, lambda x: ops.quant_attention(x, cache, wide, ctx, q_start))


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", SHARED)
def test_values_at_the_end_of_the_range_in_a_prefix(form, D):
    q, cache, table, ctx, groups, prefix, q_start, wide = shared_case(form, "mxfp4", D)
    m.check_loud(q, cache, table, ctx, q_start, lambda x: ops.prefix_attention(x, cache, wide, ctx, groups, prefix, q_start))


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", OWN)
def test_bytes_of_no_number(form, D):
    q, cache, table, ctx, q_start, wide = own_case(form, "mxfp4", D)
    start = list(range(len(ctx) + 1)) if q_start is None else q_start.tolist()
    seq = next(b for b, c in enumerate(ctx.tolist()) if start[b + 1] > start[b] and c - start[b + 1] + start[b] > 9)       # tokens 2 and 9 are before all of its rows
    seen = torch.zeros(q.shape[0], dtype=torch.bool)
    seen[start[seq]:start[seq + 1]] = True
    m.check_bytes_of_no_number(q, cache, table, ctx, q_start, lambda x: ops.quant_attention(x, cache, wide, ctx, q_start), seq, seen)


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", SHARED)
def test_bytes_of_no_number_in_a_prefix(form, D):
    q, cache, table, ctx, groups, prefix, q_start, wide = shared_case(form, "mxfp4", D)
    seen = torch.zeros(q.shape[0], dtype=torch.bool)
    start = list(range(len(ctx) + 1)) if q_start is None else q_start.tolist()
    seen[start[int(groups[0])]:start[int(groups[1])]] = True      # the first group's rows: its shared pages hold tokens 2 and 9
    m.check_bytes_of_no_number(q, cache, table, ctx, q_start, lambda x: ops.prefix_attention(x, cache, wide, ctx, groups, prefix, q_start), int(groups[0]), seen)


@pytest.mark.parametrize("eps", (0.0, 1e-6))
@pytest.mark.parametrize("tokens", (9, 1030), ids=("a row a lane", "four"))
@pytest.mark.parametrize("D", (64, 128))
def test_norms_of_large_and_small_rows(D, tokens, eps):
    m.check_norms(DEV, D, tokens, eps)


@pytest.mark.parametrize("kind", t.KINDS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", OWN)
def test_equal_values(form, D, kind):
    q, cache, table, ctx, q_start, wide = own_case(form, kind, D)
    m.check_equal_values(q, cache, table, ctx, q_start, lambda x: ops.quant_attention(x, cache, wide, ctx, q_start))


@pytest.mark.parametrize("kind", t.KINDS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", SHARED)
def test_equal_values_in_a_prefix(form, D, kind):
    q, cache, table, ctx, groups, prefix, q_start, wide = shared_case(form, kind, D)
    m.check_equal_values(q, cache, table, ctx, q_start, lambda x: ops.prefix_attention(x, cache, wide, ctx, groups, prefix, q_start))


@pytest.mark.parametrize("kind", t.KINDS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", OWN)
def test_forms(form, D, kind):
    q, cache, table, ctx, q_start, wide = own_case(form, kind, D)
    out = ops.quant_attention(q, cache, wide, ctx, q_start)
    m.check(out, q, cache, table, ctx, q_start)
    assert not out[-3:].any()
    assert torch.equal(out, ops.quant_attention(q, cache, wide, ctx, q_start))


@pytest.mark.parametrize("kind", t.KINDS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", SHARED)
def test_shared_forms(form, D, kind):
    q, cache, table, ctx, groups, prefix, q_start, wide = shared_case(form, kind, D)
    out = ops.prefix_attention(q, cache, wide, ctx, groups, prefix, q_start)
    m.check(out, q, cache, table, ctx, q_start)
    assert not out[-3:].any()
    assert torch.equal(out, ops.prefix_attention(q, cache, wide, ctx, groups, prefix, q_start))


def holes(cache, table, ctx, rows):
    """Of the sequences `rows`, whose first pages may be the same: a hole, a page behind the cache's last, no pages at all behind some; a key and a value of NaN, an infinite key."""
    nan, inf = (float("nan"), float("inf")) if cache.kind == "int8" else (255, 255)
    first, page = rows[0], cache.k.shape[2]
    at = [i for i in range(-(-int(ctx[first]) // page)) if i * page < int(ctx[rows].min())]      # pages that all of them have
    head, pages = cache.heads - 1, table[first].tolist()
    cache.vs[pages[at[0]], head, 5] = nan
    cache.ks[pages[at[-1]], 0, min(3, int(ctx[rows].min()) - 1 - at[-1] * page)] = nan
    if len(at) > 4:
        cache.ks[pages[at[4]], head, page - 1] = inf
    if len(at) > 3:
        table[rows, at[1]], table[rows, at[3]] = -1, cache.k.shape[0]


@pytest.mark.parametrize("kind", t.KINDS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", OWN)
def test_holes_and_not_numbers(form, D, kind):
    q, cache, table, ctx, q_start, _ = own_case(form, kind, D)
    alive = [b for b in range(len(ctx)) if int(ctx[b]) > 40]
    holes(cache, table, ctx, alive[:1])
    table[alive[1], 1:] = -(1 << 31)
    if len(alive) > 3:
        holes(cache, table, ctx, alive[-1:])
    wide = widened(table, OWN[form][5], OWN[form][2])
    out = ops.quant_attention(q, cache, wide, ctx, q_start)
    m.check(out, q, cache, table, ctx, q_start)
    assert torch.isnan(out).any() and not torch.isnan(out).all()


@pytest.mark.parametrize("kind", t.KINDS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", SHARED)
def test_holes_and_not_numbers_in_a_prefix(form, D, kind):
    """And contexts that end inside the shared pages, at their end, or are less than nothing."""
    q, cache, table, ctx, groups, prefix, q_start, _ = shared_case(form, kind, D)
    page, a, e = SHARED[form][2], int(groups[0]), int(groups[1])
    holes(cache, table, ctx, list(range(a, e)))
    ctx[a] = int(prefix[0]) - 7
    ctx[a + 1] = int(prefix[0])
    ctx[e - 1] = -(1 << 31)
    ctx[0] = 3
    wide = widened(table, SHARED[form][8], page)
    out = ops.prefix_attention(q, cache, wide, ctx, groups, prefix, q_start)
    m.check(out, q, cache, table, ctx, q_start)
    assert torch.isnan(out).any() and not torch.isnan(out).all()


def scattered(cache, table):
    """int8: value scales over 2^61, some of nothing, and keys that grow with their page's place, so that scores do all the way."""
    at = torch.arange(cache.vs.numel(), device=DEV).view(cache.vs.shape)
    cache.vs.mul_(torch.exp2(((at * 37) % 61 - 30).float()))
    for p, i in {p: i for row in table.tolist() for i, p in enumerate(row) if i}.items():
        cache.ks[p] *= min(1 + i, 27)
        if i % 7 == 3:
            cache.vs[p] = 0


def check_scattered(out, q, cache, table, ctx, q_start):
    """Scores of up to 30 * 27: off by 2^-11 * 27 < 2^-6 relative to the probabilities, and the roundings as ever.  Probabilities times scales are float16, the largest, W, of a row's piece at 2^7 or
    more: each is off by up to half of float16's least step, 2^-25 = 2^-32 W, times a code of up to 127; the largest's row has a code of 127, so 127 W is no more than the largest of the row's
    sizes.  1600 keys at most.  Where the largest probabilities are of keys whose values are nothing, what is left are probabilities that float32 may not hold: less than 2^-126 each, times
    1600 < 2^11 values of less than 2^33, is less than 2^-82."""
    want, size = m.whole.attention(q, cache, table, ctx, q_start)
    least = 1600 * 2 ** -32 * size.amax(-1, keepdim=True)
    assert ((out.double() - want).abs() <= t.HALF * want.abs() + (t.HALF + 2 ** -6) * size + least + 2 ** -82).all()


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", OWN)
def test_scales_far_apart(form, D):
    q, cache, table, ctx, q_start, wide = own_case(form, "int8", D)
    scattered(cache, table)
    check_scattered(ops.quant_attention(q, cache, wide, ctx, q_start), q, cache, table, ctx, q_start)
    cache.vs.fill_(0)
    assert not ops.quant_attention(q, cache, wide, ctx, q_start).any()


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", SHARED)
def test_scales_far_apart_in_a_prefix(form, D):
    q, cache, table, ctx, groups, prefix, q_start, wide = shared_case(form, "int8", D)
    scattered(cache, table)
    check_scattered(ops.prefix_attention(q, cache, wide, ctx, groups, prefix, q_start), q, cache, table, ctx, q_start)
    cache.vs.fill_(0)
    assert not ops.prefix_attention(q, cache, wide, ctx, groups, prefix, q_start).any()


@pytest.mark.parametrize("kind,D", (("int8", 128), ("mxfp4", 64)))
def test_many_pieces_of_many_rows(kind, D):
    """64 pieces of 32768 rows, which the joining launch takes in more than one turn: a table of 2^21 keys, the same for all sequences but for its first page."""
    B, page = 2048, 1024
    assert m.plan(B, B, True, 0, 16, 1, 1 << 21) == (16, 64, 0, 0, False, False)
    cache = t.filled(17, page, 1, D, kind, DEV)
    table = torch.arange(1 << 11, dtype=torch.int32, device=DEV).expand(B, -1) % 17
    ctx = torch.tensor([(37 * i) % 300 if i % 100 else 9000 + 50 * i for i in range(B)], dtype=torch.int32, device=DEV).clamp(max=17 * page)
    q = t.rows_of(B, 16, D).mul(2).to(DEV)
    poison()
    out = ops.quant_attention(q, cache, table, ctx)
    m.check(out, q, cache, table, ctx)


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("power", (-77, 105))
@pytest.mark.parametrize("form", ("16 rows", "32 rows, pieces", "256 rows, pieces"))
def test_ends_of_the_value_scales(form, power, D):
    """int8 values of about 1 times 2^-77 and 2^105, scales of 2^-83 and 2^101: no less is lost than elsewhere, 2^-32 of a row's largest of each of 1600 keys at most."""
    q, cache, table, ctx, q_start, wide = own_case(form, "int8", D)
    cache.vs.mul_(2.0 ** power)
    out = ops.quant_attention(q, cache, wide, ctx, q_start)
    want, size = m.whole.attention(q, cache, table, ctx, q_start)
    least = 1600 * 2 ** -32 * size.amax(-1, keepdim=True)
    assert ((out.double() - want).abs() <= t.HALF * want.abs() + (t.HALF + 2 ** -10) * size + least).all() and out[:-3].any()


def test_checked_inputs():
    ops.set_input_checks(True)
    try:
        m.check_checked(DEV)
    finally:
        ops.set_input_checks(False)


@pytest.mark.parametrize("four", (False, True), ids=("a row a lane", "four"))
def test_one_norm(four):
    m.check_one_norm(DEV, four)


def test_forms_in_graphs():
    """Every form captured, two graphs of it at a time; replays among eager work and other replays, on new inputs, every one against the eager result."""
    for kind, D in (("int8", 128), ("mxfp4", 64)):
        calls = []
        for form in OWN:
            q, cache, _, ctx, q_start, wide = own_case(form, kind, D)
            calls.append((q, lambda q=q, c=cache, x=ctx, s=q_start, w=wide: ops.quant_attention(q, c, w, x, s)))
        for form in SHARED:
            q, cache, _, ctx, groups, prefix, q_start, wide = shared_case(form, kind, D)
            calls.append((q, lambda q=q, c=cache, x=ctx, a=groups, p=prefix, s=q_start, w=wide: ops.prefix_attention(q, c, w, x, a, p, s)))
        graphs = []
        for q, call in calls + calls:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = call()
            graphs.append((graph, out))
        for turn in range(3):
            poison()
            for i, (q, _) in enumerate(calls):
                q.copy_(t.rows_of(q.shape[0], q.shape[1], D, 100 * turn + i))
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for i, (_, call) in enumerate(calls):
                want = call()
                assert torch.equal(graphs[i][1], want) and torch.equal(graphs[i + len(calls)][1], want), (turn, i)


def test_forms_on_two_streams():
    """Two calls of every form at once."""
    streams = [torch.cuda.Stream() for _ in "ab"]
    for form in SHARED:
        cases = [shared_case(form, kind, 64) for kind in t.KINDS]
        calls = [lambda c=c: ops.prefix_attention(c[0], c[1], c[7], c[3], c[4], c[5], c[6]) for c in cases]
        want, got = [c() for c in calls], [[], []]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(calls[i]())
        torch.cuda.synchronize()
        assert all(torch.equal(x, w) for g_, w in zip(got, want) for x in g_), form
