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


@pytest.mark.parametrize("dtype", TYPES)
def test_one_bad_value_among_missing_pages(dtype, cuda):
    """Long caches where each tile of keys has a missing page, so that all are looked through: a value that is not finite costs the tiles next to it, not the whole of a part."""
    from f3m_b200 import paged, sequence
    n, kv, width, page, most = 32, 8, 128, 16, 1024
    kp, vp = normal(20, 256, page, kv, width, dtype=dtype), normal(21, 256, page, kv, width, dtype=dtype)
    table = (torch.arange(n * most, device="cuda").view(n, most) * 37 % 255).int()      # pages are shared, the last one is one sequence's
    table[:, 3::8] = -1
    table[:, most - 1:] = torch.arange(n, device="cuda")[:, None].int()
    plan, lens = sequence.SequencePlan([1] * n), ints([16 * most - 1] * n)
    q = normal(22, n, 4 * kv, width, dtype=dtype)

    def timed():
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            out = paged.paged_attention(plan, q, kp, vp, table, lens)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return out, min(times)

    clean, fast = timed()
    assert torch.isfinite(clean).all()
    table[5, 500], table[9, 0] = 255, 255
    vp[255, 7, 2, 11], vp[255, 3, 6, 100] = float("nan"), float("-inf")
    kp[255] = 0.0
    got, slow = timed()
    assert got[[5, 9], 8:12, 11].isnan().all() and (got[[5, 9], 24:28, 100] == float("-inf")).all()
    others = [b for b in range(n) if b not in (5, 9)]
    assert torch.equal(got[others], clean[others])
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[[5, 9], 8:12, 11] = rest[[5, 9], 24:28, 100] = False
    assert torch.isfinite(got[rest]).all()
    assert slow < 5 * fast, (slow, fast)


# new, cached, heads, kv_heads, width, page, window, sinks, a tree: items cut into parts; two tiles of rows
BAD = [
    ([1], [6000], 8, 2, 64, 16, None, 0, False),
    ([1], [6000], 8, 2, 128, 16, 700, 3, False),
    ([250], [130], 4, 4, 64, 16, None, 0, False),
    ([300], [3000], 3, 1, 128, 32, 150, 5, False),
    ([200], [500], 2, 1, 64, 16, None, 0, True),
    ([250], [5000], 4, 2, 128, 16, 200, 7, True),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,cached,heads,kv,width,page,window,sinks,drafted", BAD)
def test_bad_values_reach_the_rows_that_see_them(new, cached, heads, kv, width, page, window, sinks, drafted, dtype, cuda):
    """One value that is not finite, of any kind of key: cached, at the window's edge, new, seen by rows of the second tile only.  Rows that see it have it in its column; all else is as before."""
    from f3m_b200 import paged, sequence
    plan, lens, n, c = sequence.SequencePlan(new), ints(cached), new[0], cached[0]
    kp, vp, table = cache(30, cached, new, kv, width, page, dtype)
    q, parents = normal(31, n, heads, width, dtype=dtype, scale=0.5), trees(32, new) if drafted else None
    run = lambda v, t: paged.paged_attention(plan, q, kp, v, t, lens, window, sinks, parents)  # noqa: E731
    table[0, min(c // page, 20)] = -1           # tiles with a missing page are looked through
    clean = run(vp, table)
    assert torch.isfinite(clean).all()
    depths, above = ref.tree(None if parents is None else parents.tolist(), n)
    w = window or 1 << 40
    for s in (0, 2, c - (window or 50) + 1, c - 1, c, c + n // 3, c + n - 1, c + 5 * n // 6, c // 2):
        if not 0 <= s < c + n or int(table[0, s // page]) < 0:
            continue
        pos = s if s < c else c + depths[s - c]
        sees = torch.tensor([(s < c or s - c in above[i]) and (c + depths[i] - pos < w or pos < sinks) for i in range(n)], device="cuda")
        partly = not bool(sees.all())
        for bad in (float("inf"), float("nan")):
            v2 = vp.clone()
            v2[table[0, s // page].long(), s % page, kv - 1, 9] = bad
            got, group = run(v2, table), heads // kv
            mine = torch.zeros_like(got, dtype=torch.bool)
            mine[sees, heads - group:, 9] = True
            assert not torch.isfinite(got[mine]).any(), (s, bad)
            if partly:
                assert (got[mine] == bad).all() or got[mine].isnan().all()
            assert torch.equal(got[~mine], clean[~mine]), (s, bad)


def test_a_scale_of_zero_weighs_all_alike(cuda):
    """Also where products of queries and keys are as large as FP32 has them."""
    from f3m_b200 import paged, sequence
    dtype, new, cached = torch.bfloat16, [3], [300]
    kp, vp, table = cache(40, cached, new, 1, 64, 16, dtype)
    q = normal(41, 3, 2, 64, dtype=dtype) * 1e17
    plain = ref.attention(q, kp, vp, table, cached, new, scale=0.0)
    got = paged.paged_attention(sequence.SequencePlan(new), q, kp * 1e17, vp, table, ints(cached), scale=0.0)
    # the bound counts an exponent's error by the size of the products, which a scale of zero takes out
    assert_within(got, plain)


def test_every_call_reports_a_wait_that_ran_out(cuda):
    """The word that a kernel would set, set by hand: the next call is refused, whichever it is, enqueues nothing, and the one behind it runs."""
    from f3m_b200 import _lib, paged, sequence as sq
    word = _lib.lib().f3m_seqs_error_word()
    new, cached = [5, 20], [200, 17]
    plan, lens, n = sq.SequencePlan(new), ints(cached), 25
    kp, vp, table = cache(50, cached, new, 2, 64, 16, torch.bfloat16, garbage=0.0)
    k, q = normal(51, n, 2, 64, dtype=torch.bfloat16), normal(52, n, 4, 64, dtype=torch.bfloat16)
    x, ld, state = normal(53, n, 16, dtype=torch.float32), -normal(54, n, 16, dtype=torch.float32).abs(), torch.ones(n, 16, device="cuda")
    out, _ = sq.gated_recurrence(plan, x, ld)
    calls = [lambda: paged.paged_append(plan, k, k, kp, vp, table, lens), lambda: paged.paged_attention(plan, q, kp, vp, table, lens),
             lambda: paged.paged_keep(kp, vp, table, lens, ints([[3], [4]]), ints([1, 1])), lambda: sq.gated_recurrence(plan, x, ld), lambda: sq.gated_recurrence_grad(plan, ld, out, x),
             lambda: sq.gated_recurrence_step(x, ld, state)]
    before = kp.clone(), vp.clone()
    for call in calls:
        torch.cuda.synchronize()
        assert word[0] == 0
        word[0] = 1
        with pytest.raises(_lib.F3MError, match="gave up"):
            call()
        torch.cuda.synchronize()
        assert word[0] == 0 and bool((state == 1).all()) and torch.equal(kp, before[0]) and torch.equal(vp, before[1])
    for call in calls:
        call()
    torch.cuda.synchronize()
    assert word[0] == 0
