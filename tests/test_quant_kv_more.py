"""A key/value cache in 8 or 4 bits: the ends of its ranges and what its documentation allows, on the CPU.  The kernels' tests (test_quant_kv_more_gpu.py) take their cases from here."""
import pytest
import torch

from chronos import ops
from tests import test_quant_kv as t
from tests.oracles import quant_kv_plain as plain
from tests.oracles import quant_kv_whole as whole

BF = torch.bfloat16


# The forms that attention's rules choose, and the plan that each has to have: rows of a tile of the sequences' own keys, pieces of those, the same of what groups share, whether the own keys'
# launch joins the groups' pieces, whether it takes its longest tiles first.
# Of own keys: (hq, hkv, page, contexts, tokens, keys that the table has room for at least, plan)
OWN = {
    "16 rows": (8, 2, 16, [500, 33, 200], None, 0, (16, 1, 0, 0, False, False)),
    "16 rows, pieces": (8, 2, 16, [1500, 700], None, 0, (16, 6, 0, 0, False, False)),
    "32 rows": (64, 32, 16, [90, 40, 130], [60, 20, 60], 0, (32, 1, 0, 0, False, False)),
    "32 rows, pieces": (64, 32, 16, [390, 40, 530], [60, 20, 60], 5000, (32, 3, 0, 0, False, False)),
    "256 rows": (64, 64, 16, [300, 200], [150, 112], 0, (256, 1, 0, 0, False, False)),
    "256 rows, pieces": (64, 64, 16, [300, 200], [150, 112], 2048, (256, 2, 0, 0, False, False)),
    "256 rows, longest first": (64, 64, 16, [300, 140, 200], [150, 140, 100], 0, (256, 1, 0, 0, False, True)),
    # more sequences than a wave has lanes, lengths far apart, some without a token, some with more tokens than context; as many as there may be
    "70 sequences, longest first": (64, 4, 16, [5, 60] + [(37 * i) % 170 + 1 for i in range(68)], [9, 60] + [(13 * i) % 17 for i in range(68)], 0, (256, 1, 0, 0, False, True)),
    "255 sequences, longest first": (16, 1, 32, [(53 * i) % 190 for i in range(255)], [(29 * i) % 16 for i in range(255)], 0, (256, 1, 0, 0, False, True)),
}
# Of what groups share: (hq, hkv, page, shared pages of each group, sequences of each, own tokens, tokens of each, sequences before and behind, keys that the table has room for, plan)
SHARED = {
    "16 rows": (8, 2, 16, [30], [6], [1, 20, 16, 33, 2, 40], None, 1, 0, (16, 1, 16, 9, True, False)),
    "32 rows": (8, 1, 16, [30], [40], [1 + i % 29 for i in range(40)], None, 1, 0, (16, 1, 32, 4, True, False)),
    "128 rows": (32, 16, 16, [20], [100], [1 + i % 29 for i in range(100)], None, 1, 0, (16, 1, 128, 2, True, False)),
    "256 rows": (64, 32, 16, [20], [60], [1 + i % 29 for i in range(60)], None, 1, 0, (16, 1, 256, 2, True, False)),
    # joined by a launch of its own: tables of more than 32768 keys, or own tiles of 256 rows; a group without pages, one of a single sequence
    "16 rows, joined": (8, 2, 16, [30, 0, 5], [6, 3, 1], [1, 20, 16, 33, 2, 40, 9, 50, 17, 60], None, 2, 70000, (16, 3, 16, 51, False, False)),
    "16 rows of some tokens, joined": (12, 2, 32, [9, 2], [4, 3], [40, 3, 160, 7, 1, 20, 90], [2, 1, 3, 3, 1, 0, 2], 1, 40000, (16, 2, 16, 36, False, False)),
    "32 rows, joined": (8, 1, 16, [30], [40], [1 + i % 29 for i in range(40)], None, 1, 70000, (16, 3, 32, 42, False, False)),
    "own 256 rows, joined": (32, 32, 16, [5, 2], [3, 1], [230, 200, 190, 205], [200, 190, 180, 150], 1, 0, (256, 1, 256, 2, False, False)),
}


def plan(T, B, single, groups, hq, hkv, keys):
    ops.load()
    p = torch.ops.chronos.quant_attention_plan(T, B, single, groups, hq, hkv, keys)
    return (*p[:4], bool(p[4]), bool(p[5]))


def check(out, q, cache, table, ctx, q_start=None, more=0.0):
    """:func:`test_quant_kv.check_attention`'s bound, against the oracle for many rows; ``more``: what else is off relative to sum_j p_j |v_j|."""
    want, size = whole.attention(q, cache, table, ctx, q_start)
    want, size = want.cpu(), size.cpu()
    off, most = (out.double().cpu() - want).abs(), t.HALF * want.abs() + (t.HALF + 2 ** -10 + more) * size + 1e-30
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want))
    worst = torch.nan_to_num(off / most, nan=0.0).max() if off.numel() else 0.0
    assert worst <= 1, f"{float(worst)} of what roundings allow"


@pytest.mark.parametrize("case", t.ATTENTION, ids=lambda c: "-".join(map(str, c[:5])) + f"-{len(c[5])}")
def test_the_oracles_agree(case):
    q, cache, table, ctx, q_start = t.attention_case(*case, tail=2)
    cache.vs[int(table[0, 0]), 0, 0] = float("nan") if case[0] == "int8" else 255
    table[-1, 0] = -1
    for a, b in zip(plain.attention(q, cache, table, ctx, q_start), whole.attention(q, cache, table, ctx, q_start)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-14, equal_nan=True)


def loud_values(cache, table, rising):
    """mxfp4 values up to the format's end, 6 2^125.  rising: exponents from 2^73 up to there, key by key, and keys that grow with their pages' places."""
    if not rising:
        cache.vs.fill_(252)
        return
    at = torch.arange(cache.vs[..., 0].numel(), device=cache.vs.device).view(cache.vs.shape[:-1])
    cache.vs.copy_((200 + (at * 37) % 53)[..., None].expand(cache.vs.shape))
    for p, i in {p: i for row in table.tolist() for i, p in enumerate(row) if i}.items():      # a shared page once
        cache.ks[p] += min(4, i // 6)


def check_loud(q, cache, table, ctx, q_start, attend):
    """Averages of values near the end of float32's range are finite, as sums of them are not."""
    loud_values(cache, table, False)
    check(attend(q * 0), q * 0, cache, table, ctx, q_start)
    check(attend(q), q, cache, table, ctx, q_start)
    loud_values(cache, table, True)
    q = q / 16                                                   # keys are up to 16 times as large
    check(attend(q), q, cache, table, ctx, q_start)


@pytest.mark.parametrize("lens", (None, [40, 130]), ids=("rows", "prompts"))
def test_values_at_the_end_of_the_range(lens):
    q, cache, table, ctx, q_start = t.attention_case("mxfp4", 64, 4, 2, 16, [120, 333], lens)
    check_loud(q, cache, table, ctx, q_start, lambda x: ops.quant_attention(x, cache, table, ctx, q_start))


def check_bytes_of_no_number(q, cache, table, ctx, q_start, attend, seq, seen_by):
    """Exponent bytes of 253 to 255, of a block of a key and of a value of sequence ``seq``'s tokens 2 and 9: NaN to whoever reads the block, and to the rows (a mask [T]) that see the token."""
    page, G, head = cache.k.shape[2], q.shape[1] // cache.heads, cache.heads - 1
    want = attend(q)
    assert not torch.isnan(want).any()
    pos = t.ints([2, 9, 1]).to(q.device)
    of = torch.full_like(pos, seq)
    for byte in (253, 254, 255):
        for which, token, other in (("ks", 2, "vs"), ("vs", 9, "ks")):
            place, scales = (int(table[seq, token // page]), head, token % page, 1), getattr(cache, which)
            kept = int(scales[place])
            scales[place] = byte
            read = dict(zip(("ks", "vs"), ops.quant_kv_read(cache, table, pos, of)))
            at = pos.tolist().index(token)
            bad = torch.isnan(read[which])
            assert bad[at, head, 32:64].all() and bad.sum() == 32 and not torch.isnan(read[other]).any()
            out = attend(q)
            bad = torch.isnan(out).cpu()
            assert bad[:, G * head:][seen_by].all() and bad.sum() == G * q.shape[2] * int(seen_by.sum()), (byte, which)
            scales[place] = kept
    assert torch.equal(attend(q), want)


def test_bytes_of_no_number():
    q, cache, table, ctx, q_start = t.attention_case("mxfp4", 64, 4, 2, 16, [70, 33], [20, 33])
    seen = torch.zeros(53, dtype=torch.bool)
    seen[:20] = True
    check_bytes_of_no_number(q, cache, table, ctx, q_start, lambda x: ops.quant_attention(x, cache, table, ctx, q_start), 0, seen)


SIZES = (1.0, 1e30, 3e38, 1e-18, 1e-30, 1e-38)


def check_norms(device, D, tokens, eps):
    """Rows whose squares are no numbers of float32, and ordinary ones beside them: normed as others are."""
    hq, hkv, page = 8, 2, 16
    (qkv, pos, seq, table, cs, wq, wk), cache = t.write_case("int8", D, hq, hkv, page, D, True, [tokens], [tokens], device=device)
    x = torch.randn(tokens, hq + 2 * hkv, D, generator=torch.Generator().manual_seed(9)).clamp(-1, 1)
    x = (x * torch.tensor(SIZES)[torch.arange(tokens * (hq + 2 * hkv)).view(tokens, -1, 1) % len(SIZES)]).to(BF)
    q = ops.norm_rope_kv_quant(x.flatten(1).to(device), pos, seq, table, cs, cache, hq, wq, wk, eps=eps)
    want = plain.norm_rotation(x[:, :hq], wq.cpu(), eps, cs.cpu(), pos.cpu())
    # Half a step of the output's type, and float32 products: relative to a row's largest.  bfloat16's numbers below 2^-126 are 2^-133 apart: rows of 1e-38 over 1e-3 have such
    # numbers, whose half step is 2^-134 whatever their size.
    assert ((q.double().cpu() - want).abs() <= t.HALF * want.abs() + 2 ** -20 * want.abs().amax(-1, keepdim=True) + 2 ** -134).all()
    if eps == 0:
        assert (want.abs().amax(-1) > 0.5).all()
    codes, scales = plain.quantise(plain.norm_rotation(x[:, hq:hq + hkv], wk.cpu(), eps, cs.cpu(), pos.cpu()), "int8")
    p, o = table.cpu()[0, torch.arange(tokens) // page].long(), torch.arange(tokens) % page
    assert torch.equal(cache.k.cpu()[p, :, o].long(), codes) and torch.equal(cache.ks.cpu()[p, :, o], scales)


@pytest.mark.parametrize("eps", (0.0, 1e-6))
@pytest.mark.parametrize("D", (64, 128))
def test_norms_of_large_and_small_rows(D, eps):
    check_norms("cpu", D, 9, eps)


def check_equal_values(q, cache, table, ctx, q_start, attend):
    """All of a head's values alike: rows that see any key have that value, whatever the scores.  Codes of seven bits at most and scales of powers of two: bfloat16 holds the value, and half a
    step of it, 2^-9 of its size at least, is more than float16's rounding of the probabilities (2^-11 at most) and float32 sums of some 500 (2^-14) come to."""
    cache.v.copy_(cache.v[0, :, :1].clone())
    cache.vs.fill_(2.0 ** -3) if cache.kind == "int8" else cache.vs.fill_(124)
    v = plain.values(cache)[1][0, :, 0].to(q.device)
    start = list(range(len(ctx) + 1)) if q_start is None else q_start.tolist()
    want = v.repeat_interleave(q.shape[1] // cache.heads, 0).expand(q.shape).clone()
    for b, c in enumerate(ctx.tolist()):
        want[start[b]:min(start[b + 1], max(start[b], start[b + 1] - c))] = 0      # more tokens than context
    want[start[-1]:] = 0
    assert torch.equal(attend(q).double(), want)


@pytest.mark.parametrize("kind", t.KINDS)
@pytest.mark.parametrize("lens", (None, [40, 130]), ids=("rows", "prompts"))
def test_equal_values(kind, lens):
    q, cache, table, ctx, q_start = t.attention_case(kind, 64, 4, 2, 16, [120, 333], lens)
    check_equal_values(q, cache, table, ctx, q_start, lambda x: ops.quant_attention(x, cache, table, ctx, q_start))


def check_checked(device):
    """With inputs checked: what the documentation leaves out is left out as ever, what it rules out is named."""
    for kind in t.KINDS:
        t.check_left_out(kind, device)
    (qkv, pos, seq, table, cs, wq, wk), cache = t.write_case("int8", 64, 2, 1, 16, 64, True, [4], [20], device=device)
    padded, ones = t.ints([17, -1, -1, 18]).to(device), torch.zeros_like(seq)
    ops.norm_rope_kv_quant(qkv, padded, ones, table, cs, cache, 2, wq, wk)
    ops.norm_rope_kv_quant(qkv, t.ints([17, 19, 19, 18]).to(device), ones, table, cs[:19].contiguous(), cache, 2, wq, wk)      # both 19s are behind the rope table
    with pytest.raises(IndexError, match="two tokens in one place"):
        ops.norm_rope_kv_quant(qkv, t.ints([17, 18, 3, 18]).to(device), ones, table, cs, cache, 2, wq, wk)
    q, cache, table, ctx, _ = t.attention_case("int8", 64, 2, 1, 16, [40, 70], None, device)
    want, groups = ops.quant_attention(q, cache, table, ctx), t.ints([0, 2]).to(device)
    assert torch.equal(ops.prefix_attention(q, cache, table, ctx, groups, t.ints([-1]).to(device)).isnan(), want.isnan())      # nothing shared
    with pytest.raises(IndexError, match="pages of group 0 differ"):
        ops.prefix_attention(q, cache, table, ctx, groups, t.ints([16]).to(device))


def test_checked_inputs(monkeypatch):
    monkeypatch.setattr(ops.quant_kv._pkg, "_checking", lambda x: True)
    check_checked("cpu")


def check_one_norm(device, four):
    """Weights for the queries alone, and for the keys alone."""
    case = ("mxfp4", 128, 8, 2, 16, 64, True, [1030 if four else 5], [1040 if four else 20])
    for which in (0, 1):
        (qkv, pos, seq, table, cs, wq, wk), cache = t.write_case(*case, device=device)
        wq, wk = (wq, None) if which == 0 else (None, wk)
        q = ops.norm_rope_kv_quant(qkv, pos, seq, table, cs, cache, 8, wq, wk)
        x = qkv.cpu().view(len(pos), -1, 128)
        want = plain.norm_rotation(x[:, :8], None if wq is None else wq.cpu(), 1e-6, cs.cpu(), pos.cpu())
        assert ((q.double().cpu() - want).abs() <= t.HALF * want.abs() + 2 ** -20 * want.abs().amax(-1, keepdim=True)).all()
        p, o = table.cpu()[0, pos.cpu().long() // 16].long(), pos.cpu().long() % 16
        codes, scales = plain.quantise(plain.norm_rotation(x[-9:, 8:10], None if wk is None else wk.cpu(), 1e-6, cs.cpu(), pos.cpu()[-9:]), "mxfp4")
        assert torch.equal(plain.whole_codes(cache)[0][p, :, o][-9:], codes) and torch.equal(cache.ks.cpu()[p, :, o][-9:].long(), scales)


def test_one_norm():
    check_one_norm("cpu", False)
