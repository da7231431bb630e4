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

# Forms of a sequence's own keys: (hq, hkv, page, contexts, tokens, keys that the table has room for at least)
OWN = {
    "16 rows": (8, 2, 16, [500, 33, 200], None, 0),
    "16 rows, pieces": (8, 2, 16, [1500, 700], None, 0),
    "32 rows": (64, 32, 16, [90, 40, 130], [60, 20, 60], 0),
    "32 rows, pieces": (64, 32, 16, [390, 40, 530], [60, 20, 60], 5000),
    "256 rows": (64, 64, 16, [300, 200], [150, 112], 0),
    "256 rows, pieces": (64, 64, 16, [300, 200], [150, 112], 2048),
    "256 rows, longest first": (64, 64, 16, [300, 140, 200], [150, 140, 100], 0),
}
# and of what groups share: (hq, hkv, page, shared pages of each group, sequences of each, own tokens, tokens of each, sequences before and behind, keys that the table has room for)
SHARED = {
    "16 rows": (8, 2, 16, [30], [6], [1, 20, 16, 33, 2, 40], None, 1, 0),
    "32 rows": (8, 1, 16, [30], [40], [1 + i % 29 for i in range(40)], None, 1, 0),
    "128 rows": (32, 16, 16, [20], [100], [1 + i % 29 for i in range(100)], None, 1, 0),
    "256 rows": (64, 32, 16, [20], [60], [1 + i % 29 for i in range(60)], None, 1, 0),
}


def widened(table, keys, page):
    wide = torch.zeros(table.shape[0], max(table.shape[1], -(-keys // page)), dtype=torch.int32, device=table.device)
    wide[:, :table.shape[1]] = table
    return wide


def own_case(form, kind, D):
    hq, hkv, page, ctx, lens, keys = OWN[form]
    q, cache, table, ctx, q_start = t.attention_case(kind, D, hq, hkv, page, ctx, lens, DEV, tail=3)
    return q, cache, table, ctx, q_start, widened(table, keys, page)


def shared_case(form, kind, D):
    *case, keys = SHARED[form]
    (q, table, ctx, groups, prefix, q_start), cache = g.prefix_case(kind, D, *case)
    return q, cache, table, ctx, groups, prefix, q_start, widened(table, keys, case[2])


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
    seen = torch.zeros(q.shape[0], dtype=torch.bool)
    for i in range(start[0], start[1]):
        seen[i] = int(ctx[0]) - start[1] + i >= 9
    assert seen[start[0]:start[1]].all()                         # tokens 2 and 9 are before all of them
    m.check_bytes_of_no_number(q, cache, table, ctx, q_start, lambda x: ops.quant_attention(x, cache, wide, ctx, q_start), 0, seen)


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("form", SHARED)
def test_bytes_of_no_number_in_a_prefix(form, D):
    q, cache, table, ctx, groups, prefix, q_start, wide = shared_case(form, "mxfp4", D)
    seen = torch.zeros(q.shape[0], dtype=torch.bool)
    seen[int(groups[0]):int(groups[1])] = True                   # the one group's rows, a token each
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
