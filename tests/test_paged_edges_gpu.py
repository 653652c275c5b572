"""Attention over pages where keys, values and scores are not finite, and where pages are missing in many places (paged_reference.py)."""
import pytest
import torch

import paged_reference as ref
from sequence_reference import assert_within
from test_paged_gpu import cache, ints, normal, trees

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


# new, cached, heads, kv_heads, width, page, window, sinks, a tree: items taken whole, cut into parts, of one tile of rows and of two
LOW = [
    ([1], [60], 2, 1, 64, 16, None, 0, False),
    ([1], [4000], 8, 2, 64, 16, None, 0, False),
    ([1] * 80, [300] * 80, 8, 8, 64, 16, None, 0, False),
    ([1, 1], [20000, 9000], 4, 1, 128, 64, None, 0, False),
    ([300, 5], [1000, 3000], 4, 2, 64, 32, None, 0, False),
    ([300], [1000], 3, 1, 128, 16, 150, 5, False),
    ([30, 200], [700, 2500], 4, 2, 64, 16, None, 0, True),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,cached,heads,kv,width,page,window,sinks,drafted", LOW)
def test_scores_of_minus_infinity(new, cached, heads, kv, width, page, window, sinks, drafted, dtype, cuda):
    """Infinite keys against queries below zero.  A row that sees nothing else is not a number, as the softmax of such scores is not; one that sees finite scores too is what these make
    it, wherever they lie; one that sees nothing is zeros."""
    from f3m_b200 import paged, sequence
    plan, lens = sequence.SequencePlan(new), ints(cached)
    kp, vp, table = cache(1, cached, new, kv, width, page, dtype)
    q, parents = -normal(2, sum(new), heads, width, dtype=dtype, scale=0.3).abs() - 0.1, trees(3, new) if drafted else None
    run = lambda k, t: paged.paged_attention(plan, q, k, vp, t, lens, window, sinks, parents)  # noqa: E731
    assert run(torch.full_like(kp, float("inf")), table).isnan().all()
    assert (run(kp, torch.full_like(table, -1)) == 0).all()
    # of some pages all keys: as if these were missing, but for rows that see nothing else
    for low in (lambda p: p < 3, lambda p: p % 3 == 1, lambda p: p >= 2):
        k2, t2 = kp.clone(), table.clone()
        for b in range(len(new)):
            for p in filter(low, range(-(-(cached[b] + new[b]) // page))):
                k2[table[b, p].long()], t2[b, p] = float("inf"), -1
        want = ref.attention(q, kp, vp, t2, cached, new, window, sinks, parents)
        none = (run(kp, t2) == 0).all(-1).all(-1)          # rows that see no finite score
        got = run(k2, table)
        assert got[none].isnan().all()
        assert_within(got[~none], tuple(x[~none] for x in want))
