"""The paged cache against its definitions in 64 bits (paged_reference.py)."""
import random

import pytest
import torch

import paged_reference as ref
from sequence_reference import assert_within

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def normal(seed, *shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def ints(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


def trees(seed, new):
    rng = random.Random(seed)
    return ints([-1 if i == 0 or rng.random() < 0.05 else rng.randrange(max(0, i - 6), i) for n in new for i in range(n)])


def cache(seed, lengths, new, kv, width, page, dtype, garbage=float("nan"), spare=2):
    """Pages in any order; what holds no token holds garbage.  k_pages, v_pages, table"""
    rng = random.Random(seed)
    need = [-(-(max(c, 0) + n) // page) for c, n in zip(lengths, new)]
    pool, most = sum(need) + spare, max(need) + 1
    order = list(range(pool))
    rng.shuffle(order)
    kp, vp = normal(seed + 1, pool, page, kv, width, dtype=dtype), normal(seed + 2, pool, page, kv, width, dtype=dtype)
    empty = torch.ones(pool, page, dtype=torch.bool)
    rows = []
    for c, n, m in zip(lengths, new, need):
        mine = [order.pop() for _ in range(m)]
        for s in range(max(c, 0) + n):
            empty[mine[s // page], s % page] = False
        rows.append(mine + [order[0] if order else 0] * (most - m))       # behind the last page: one that holds garbage
    kp[empty.cuda()], vp[empty.cuda()] = garbage, garbage
    return kp, vp, ints(rows)


# new, cached, heads, kv_heads, width, page, window, sinks, a tree
CASES = [
    ([1], [0], 1, 1, 64, 16, None, 0, False),
    ([1], [127], 2, 2, 64, 16, None, 0, False),
    ([1], [128], 4, 1, 128, 128, None, 0, False),
    ([3, 0, 1, 2], [128, 5, 0, 1000], 4, 2, 64, 64, None, 0, False),
    ([1] * 9, [0, 1, 5, 300, 700, 129, 2000, 40, 63], 16, 2, 128, 32, 257, 3, False),
    ([300, 17], [513, 1], 3, 1, 128, 64, 100, 5, False),
    ([300], [513], 8, 2, 64, 256, 5000, 5000, False),
    ([130, 257, 1], [0, 7, 900], 6, 2, 96, 16, 130, 140, False),
    ([9], [1500], 8, 2, 64, 16, None, 0, True),
    ([32, 25, 1, 0, 64], [1000, 127, 0, 50, 4097], 16, 4, 128, 64, None, 0, True),
    ([60, 33], [500, 100], 12, 4, 80, 32, 20, 4, True),
    ([256, 100], [129, 0], 2, 1, 128, 128, None, 0, True),
    ([256], [700], 5, 1, 104, 8, 30, 710, True),
    ([40, 3], [90, 2000], 128, 1, 8, 16, None, 0, True),
    ([5, 7], [300, 1], 48, 3, 32, 512, 64, 1, True),
    ([77], [3000], 7, 7, 64, 1024, None, 0, True),
    ([2], [20000], 8, 8, 128, 64, None, 0, True),
    # items cut anywhere, several to a CTA: short ones and long ones, one tile of rows and two side by side
    ([1] * 40, [(997 * b) % 3100 for b in range(40)], 16, 8, 128, 64, None, 0, False),
    ([3, 1] * 100, [(89 * b) % 300 for b in range(200)], 8, 4, 64, 16, None, 0, True),
    ([400, 1, 30, 200], [5000, 3000, 1, 9000], 16, 4, 128, 64, None, 0, False),
    ([250, 40, 256], [6000, 100, 3000], 8, 4, 64, 32, None, 0, True),
    ([700], [12000], 12, 4, 96, 128, 4000, 700, False),
    ([512, 256], [2000, 2300], 8, 8, 128, 128, 1500, 3, False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,cached,heads,kv,width,page,window,sinks,drafted", CASES)
def test_paged_attention(new, cached, heads, kv, width, page, window, sinks, drafted, dtype, cuda):
    from f3m_b200 import paged, sequence
    kp, vp, table = cache(1, cached, new, kv, width, page, dtype)
    q = normal(5, sum(new), heads, width, dtype=dtype, scale=1.5)
    parents = trees(6, new) if drafted else None
    want = ref.attention(q, kp, vp, table, cached, new, window, sinks, parents)
    got = paged.paged_attention(sequence.SequencePlan(new), q, kp, vp, table, ints(cached), window, sinks, parents)
    assert_within(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("drafted", [False, True])
def test_only_what_is_seen_is_read(drafted, dtype, cuda):
    """Between the sinks and the window pages may be gone, or hold another's garbage."""
    from f3m_b200 import paged, sequence
    new, cached, window, sinks, page = [40, 1, 130], [900, 431, 2000], 100, 5, 16
    kp, vp, table = cache(11, cached, new, 2, 64, page, dtype)
    for b, c in enumerate(cached):      # the first new token is at position c
        for s in range(-(-sinks // page), (c - window + 1) // page):
            kp[table[b, s].long()], vp[table[b, s].long()] = float("nan"), float("inf")
            if s % 3 < 2:
                table[b, s] = -1 if s % 3 else 1 << 30
    q = normal(15, sum(new), 4, 64, dtype=dtype)
    parents = trees(16, new) if drafted else None
    want = ref.attention(q, kp, vp, table, cached, new, window, sinks, parents)
    assert_within(paged.paged_attention(sequence.SequencePlan(new), q, kp, vp, table, ints(cached), window, sinks, parents), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [8, 64, 256])
def test_missing_pages_lengths_and_parents_out_of_range(page, dtype, cuda):
    """A number that is no page holds no tokens, rows that see none are zeros; lengths and parents are held in their range."""
    from f3m_b200 import paged, sequence
    new, cached = [5, 4, 3, 1, 6], [300, 0, 10, 700, 3]
    kp, vp, table = cache(21, cached, new, 2, 64, page, dtype, garbage=0.0)
    table[0, 0], table[0, 2 if table.shape[1] > 2 else 0] = -1, kp.shape[0]
    table[1] = -7                        # nothing is left of the second sequence
    said = ints([300, -5, 10, 1 << 30, 3])      # the second's is 0; the fourth's all that the table holds, which leaves no place for a new token
    q = normal(25, sum(new), 6, 64, dtype=dtype)
    parents = ints([-1, 0, 5, -9, 2, 0, 0, 0, 0, 7, 2, 1, 1 << 30, -1, 0, 1, 2, 3, 4])
    for p in (None, parents):
        want = ref.attention(q, kp, vp, table, said.tolist(), new, None, 0, p)
        got = paged.paged_attention(sequence.SequencePlan(new), q, kp, vp, table, said, parents=p)
        assert_within(got, want)
        assert (got[5:9] == 0).all()
    none = torch.zeros(len(new), 0, device="cuda", dtype=torch.int32)
    assert (paged.paged_attention(sequence.SequencePlan(new), q, kp, vp, none, said) == 0).all()
    assert (paged.paged_attention(sequence.SequencePlan(new), q, kp[:0], vp[:0], table, said) == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_siblings_that_are_not_numbers(dtype, cuda):
    """A branch that is not finite reaches its own tokens and no others; a cached key that is not reaches all that see it."""
    from f3m_b200 import paged, sequence
    new, cached, page = [12], [200], 16
    plan, parents = sequence.SequencePlan(new), ints([-1, 0, 0, 1, 2, 3, 4, 5, 6, 0, 9, 2])
    kp, vp, table = cache(31, cached, new, 2, 64, page, dtype)
    q = normal(35, 12, 8, 64, dtype=dtype)
    clean = paged.paged_attention(plan, q, kp, vp, table, ints(cached), parents=parents)
    below = [2, 4, 6, 8, 11]
    others = [i for i in range(12) if i not in below]
    s = cached[0] + 2
    for k_bad, v_bad in ((float("nan"), None), (None, float("nan")), (None, float("inf")), (float("inf"), None)):
        k2, v2 = kp.clone(), vp.clone()
        at = (table[0, s // page].long(), s % page)
        if k_bad is not None:
            k2[at] = k_bad
        if v_bad is not None:
            v2[at[0], at[1], :, 3] = v_bad
        got = paged.paged_attention(plan, q, k2, v2, table, ints(cached), parents=parents)
        assert torch.equal(got[others], clean[others]), (k_bad, v_bad)
        if v_bad is not None:
            assert (got[below][..., 3] == v_bad).all() if v_bad == v_bad else got[below][..., 3].isnan().all()
            rest = [c for c in range(64) if c != 3]
            assert torch.equal(got[below][..., rest], clean[below][..., rest])
        elif k_bad != k_bad:
            assert got[below].isnan().all()
    k2 = kp.clone()
    k2[table[0, 3].long(), 5, 1] = float("nan")
    got = paged.paged_attention(plan, q, k2, vp, table, ints(cached), parents=parents)
    assert torch.equal(got[:, :4], clean[:, :4]) and got[:, 4:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_exponents_and_scales(dtype, cuda):
    """Rows whose largest weight comes first, last, and rises tile by tile; a negative scale, one of zero."""
    from f3m_b200 import paged, sequence
    cached, new, page = [700], [40], 32
    kp, vp, table = cache(41, cached, new, 1, 64, page, dtype)
    q = torch.ones(40, 2, 64, device="cuda", dtype=dtype)
    for slope in (0.05, -0.05, 0.5):
        for s in range(740):
            kp[table[0, s // page].long(), s % page] = s * slope
        for scale in (0.125, -0.125, 0.0):
            want = ref.attention(q, kp, vp, table, cached, new, 400, 7, None, scale)
            assert_within(paged.paged_attention(sequence.SequencePlan(new), q, kp, vp, table, ints(cached), 400, 7, scale=scale), want, f"{slope} {scale}")


@pytest.mark.parametrize("dtype", TYPES)
def test_views(dtype, cuda):
    """Pages with heads before tokens, keys and values of a page side by side, queries of a joint projection, heads before tokens, starting off 16 bytes."""
    from f3m_b200 import paged, sequence
    cached, new, kv, w, page = [77, 300], [4, 1], 2, 64, 32
    plan, lens = sequence.SequencePlan(new), ints(cached)
    kp, vp, table = cache(51, cached, new, kv, w, page, dtype)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kp, vp)]
    both = torch.stack([kp, vp], 1)
    joint = normal(55, 5, 3, 4, w, dtype=dtype)
    flat = normal(56, 5 * 4 * w + 1, dtype=dtype)
    for q in (joint[:, 1], normal(57, 4, 5, w, dtype=dtype).transpose(0, 1), flat[1:].view(5, 4, w)):
        want = ref.attention(q, kp, vp, table, cached, new)
        for k, v in ((kp, vp), heads_first, (both[:, 0], both[:, 1])):
            assert_within(paged.paged_attention(plan, q, k, v, table, lens), want)
    wide = torch.full((2, 2 * table.shape[1]), -1, device="cuda", dtype=torch.int32)
    for t in (wide[:, ::2], wide[:, :table.shape[1]]):
        t.copy_(table)
        assert_within(paged.paged_attention(plan, q, kp, vp, t, lens), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,columns,interleaved", [(64, 64, False), (128, 64, True), (80, 80, False), (96, 32, False), (32, 16, True), (104, 96, True)])
@pytest.mark.parametrize("drafted", [False, True])
def test_append(width, columns, interleaved, drafted, dtype, cuda):
    """Written tokens, and all others as they were; queries turned likewise."""
    from f3m_b200 import paged, sequence
    new, cached, heads, kv, page = [5, 0, 1, 130, 33], [0, 9, 64, 1000, 100000], 6, 2, 32
    plan, n = sequence.SequencePlan(new), sum(new)
    kp, vp, table = cache(61, cached, new, kv, width, page, dtype, garbage=0.5)
    k, v, q = (normal(65 + i, n, h, width, dtype=dtype) for i, h in enumerate((kv, kv, heads)))
    parents = trees(68, new) if drafted else None
    rotation = paged.Rotation(columns, interleaved=interleaved)
    freq = [10000.0 ** (-2 * i / columns) for i in range(columns // 2)]
    pos, r0, want_k, want_v = [], 0, kp.clone(), vp.clone()
    for c, m in zip(cached, new):
        pos += [c + d for d in ref.tree(None if parents is None else parents[r0:r0 + m].tolist(), m)[0]]
        r0 += m
    pos = torch.tensor(pos)
    k_pages, v_pages = kp.clone(), vp.clone()
    got_q = paged.paged_append(plan, k, v, k_pages, v_pages, table, ints(cached), rotation, parents, q)
    assert_within(got_q, ref.rotate(q, pos, columns, freq, interleaved), "q")
    turned, bound = ref.rotate(k, pos, columns, freq, interleaved)
    r0 = 0
    for b, (c, m) in enumerate(zip(cached, new)):
        page_of, row, there = ref.places(range(c, c + m), table[b], page, kp.shape[0])
        assert there.all()
        at = (page_of.cuda(), row.cuda())
        assert_within(k_pages[at], (turned[r0:r0 + m], bound[r0:r0 + m]), "k")
        want_k[at], want_v[at] = k_pages[at], v[r0:r0 + m]
        r0 += m
    assert torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)
    # without a rotation, without queries
    assert paged.paged_append(plan, k, v, k_pages, v_pages, table, ints(cached)) is None
    r0 = 0
    for b, (c, m) in enumerate(zip(cached, new)):
        page_of, row, _ = ref.places(range(c, c + m), table[b], page, kp.shape[0])
        want_k[page_of.cuda(), row.cuda()] = k[r0:r0 + m]
        r0 += m
    assert torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)


def test_append_far_positions_and_frequencies(cuda):
    """Angles two billion positions away; frequencies of one's own, above a turn and below zero."""
    from f3m_b200 import paged, sequence
    dtype, page, width, c = torch.float16, 1 << 20, 64, (1 << 31) - (1 << 24)
    plan = sequence.SequencePlan([3])
    table = torch.full((1, 2040), -1, device="cuda", dtype=torch.int32)
    kp = torch.zeros(1, page, 1, width, device="cuda", dtype=dtype)
    vp = torch.zeros_like(kp)
    table[0, c // page] = 0
    k, v = normal(71, 3, 1, width, dtype=dtype), normal(72, 3, 1, width, dtype=dtype)
    freq = [3.7 * (-0.9) ** i for i in range(32)]
    q = paged.paged_append(plan, k, v, kp, vp, table, ints([c + 5]), paged.Rotation(64, frequencies=freq), q=k)
    # the reference's own angles are rounded to 2^-53 of some 2^33
    turned, bound = ref.rotate(k, torch.arange(c + 5, c + 8), 64, freq, False)
    assert_within(q, (turned, bound + 2.0 ** -19))
    assert torch.equal(kp[0, 5:8], q) and torch.equal(vp[0, 5:8], v) and (kp[0, 8:] == 0).all() and (kp[0, :5] == 0).all()


@pytest.mark.parametrize("page", [8, 64])
def test_append_writes_only_places_that_are_there(page, cuda):
    from f3m_b200 import paged, sequence
    new, cached = [20, 3, 7], [10, 4, 0]
    plan, n = sequence.SequencePlan(new), sum(new)
    kp, vp, table = cache(81, cached, new, 2, 32, page, torch.bfloat16, garbage=0.25)
    k, v = normal(85, n, 2, 32, dtype=torch.bfloat16), normal(86, n, 2, 32, dtype=torch.bfloat16)
    table[0, 1], table[1] = -1, kp.shape[0]
    said = ints([10, 4, 1 << 30])       # the third's tokens lie behind the table
    k2, v2 = kp.clone(), vp.clone()
    paged.paged_append(plan, k, v, k2, v2, table, said)
    page_of, row, there = ref.places(range(10, 30), table[0], page, kp.shape[0])
    at = (page_of[there].cuda(), row[there].cuda())
    kp[at], vp[at] = k[:20][there.cuda()], v[:20][there.cuda()]
    assert torch.equal(k2, kp) and torch.equal(v2, vp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,page", [(64, 16), (128, 8), (24, 128)])
def test_keep(width, page, dtype, cuda):
    from f3m_b200 import paged
    cached, new, kv = [100, 0, 31, 7, 500], [64, 20, 9, 5, 30], 3
    kp, vp, table = cache(91, cached, new, kv, width, page, dtype, garbage=2.0)
    paths = [[0, 2, 3, 7, 8, 9, 20, 21, 22, 40, 63], [3, 4, 19], [], [1], list(range(30))]
    most = 31
    kept = ints([p + [-3] * (most - len(p)) for p in paths])
    k2, v2 = kp.clone(), vp.clone()
    paged.paged_keep(k2, v2, table, ints(cached), kept, ints([11, 3, 0, 1, 30]))
    for b, path in enumerate(paths):
        to = ref.places([cached[b] + j for j in range(len(path))], table[b], page, kp.shape[0])
        source = ref.places([cached[b] + m for m in path], table[b], page, kp.shape[0])
        for x in (kp, vp):
            x[to[0].cuda(), to[1].cuda()] = x[source[0].cuda(), source[1].cuda()].clone()
    assert torch.equal(k2, kp) and torch.equal(v2, vp)


def test_keep_leaves_what_it_cannot_move(cuda):
    """Values that no path has, counts out of range, pages that are missing, the same token twice."""
    from f3m_b200 import paged
    cached, new, page = [20, 20, 3], [12, 12, 12], 8
    kp, vp, table = cache(101, cached, new, 1, 16, page, torch.bfloat16, garbage=2.0)
    table[1, 3] = -1                     # tokens 24..31 of the second: new 4..11
    kept = ints([[2, 0, -1, 9, 9, 1 << 30], [1, 2, 6, 3, 8, 9], [5, 6, 7, 8, 9, 10]])
    k2, v2 = kp.clone(), vp.clone()
    paged.paged_keep(k2, v2, table, ints(cached), kept, ints([99, 6, -4]))
    for b, moves in enumerate(([(0, 2), (3, 9), (4, 9)], [(0, 1), (1, 2)], [])):
        for j, m in moves:
            for x in (kp, vp):
                s, d = cached[b] + m, cached[b] + j
                x[table[b, d // page].long(), d % page] = x[table[b, s // page].long(), s % page]
    assert torch.equal(k2, kp) and torch.equal(v2, vp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 4)])
def test_prompt_draft_keep_and_go_on(window, sinks, dtype, cuda):
    """A prompt in chunks, a drafted tree, its accepted path kept, another token: the outputs of attention over the whole text, as if it had been known from the start."""
    from f3m_b200 import paged, sequence as sq
    heads, kv, w, page, text = 4, 2, 64, 16, [300, 40]
    path = [0, 2, 5]                     # of the tree, accepted: tokens text..text + 2 of the whole
    total = [t + len(path) + 1 for t in text]
    q, k, v = (normal(110 + i, sum(total), h, w, dtype=dtype) for i, h in enumerate((heads, kv, kv)))
    rotation = paged.Rotation(w)
    ends = [0, total[0]]
    pages = -(-(max(total) + 10) // page)
    kp = torch.full((2 * pages, page, kv, w), float("nan"), device="cuda", dtype=dtype)
    vp, table, lengths = kp.clone(), torch.randperm(2 * pages, device="cuda").int().view(2, pages), ints([0, 0])

    def rows(x, parts):
        return torch.cat([x[e + a:e + b] for e, (a, b) in zip(ends, parts)])

    outs = [[], []]

    def go(parts, parents=None, fill=None):
        new = [b - a for a, b in parts] if fill is None else [len(f) for f in fill]
        plan = sq.SequencePlan(new)
        qq, kk, vv = ((rows(x, parts) if fill is None else torch.cat([torch.cat([x[e + t + path.index(i)][None] if i in path else normal(999 + i, 1, *x.shape[1:], dtype=dtype)
                                                                                  for i in f]) for e, t, f in zip(ends, text, fill)])) for x in (q, k, v))
        qq = paged.paged_append(plan, kk, vv, kp, vp, table, lengths, rotation, parents, qq)
        out = paged.paged_attention(plan, qq, kp, vp, table, lengths, window, sinks, parents)
        return list(torch.split(out, new))

    for a, b in ((0, 33), (33, 40), (40, 300)):
        parts = [(min(a, t), min(b, t)) for t in text]
        for o, x in zip(outs, go(parts)):
            o.append(x)
        lengths += ints([y - x for x, y in parts])
    drafted = go(None, ints([-1, 0, 0, 1, 1, 2, 2] * 2), [list(range(7))] * 2)
    for o, x in zip(outs, drafted):
        o.append(x[path])
    paged.paged_keep(kp, vp, table, lengths, ints([path] * 2), ints([3, 3]))
    lengths += 3
    for o, x in zip(outs, go([(t + 3, t + 4) for t in text])):
        o.append(x)
    got = torch.cat([torch.cat(o) for o in outs])
    # the same through window_attention, on keys and queries that were turned one by one
    pos = torch.cat([torch.arange(t) for t in total])
    freq = [10000.0 ** (-2 * i / w) for i in range(w // 2)]
    qt, kt = (ref.rotate(x, pos, w, freq, False)[0].to(dtype) for x in (q, k))
    plain, _ = sq.window_attention(sq.SequencePlan(total), qt, kt, v, window or 1 << 30, sinks)
    # roundings of turned keys and queries to the type differ in one of many
    err = (got.double() - plain.double()).norm() / plain.double().norm()
    assert err < 4 * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", TYPES)
def test_calls_repeat_and_replay(dtype, cuda):
    """The same bits again, on another stream, and from two captured graphs at once whose lengths, tables and trees move on."""
    from f3m_b200 import paged, sequence as sq
    new, kv, heads, w, page = [7, 1, 20], 2, 8, 64, 16
    plan, rotation = sq.SequencePlan(new), paged.Rotation(w)
    data = []
    for i, cached in enumerate(([900, 5, 130], [100, 700, 2])):
        kp, vp, table = cache(120 + i, [1000, 1000, 1000], new, kv, w, page, dtype)
        data.append([normal(130 + i, 28, heads, w, dtype=dtype), normal(140 + i, 28, kv, w, dtype=dtype), normal(150 + i, 28, kv, w, dtype=dtype), kp, vp, table, ints(cached),
                     trees(160 + i, new), ints([[0, 2, 4], [0, 0, 0], [1, 3, 17]]), ints([3, 1 + i, 3])])

    def run(q, k, v, kp, vp, table, lens, parents, kept, counts):
        q = paged.paged_append(plan, k, v, kp, vp, table, lens, rotation, parents, q)
        out = paged.paged_attention(plan, q, kp, vp, table, lens, None, 0, parents)
        paged.paged_keep(kp, vp, table, lens, kept, counts)
        return q, out

    clone = lambda d: [t.clone() for t in d]  # noqa: E731
    copies = [clone(d) for d in data]
    first = [run(*d) for d in copies]
    for _ in range(10):
        d = clone(data[0])
        for a, b in zip(run(*d) + (d[3], d[4]), first[0] + (copies[0][3], copies[0][4])):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    side, held = [torch.cuda.Stream(), torch.cuda.Stream()], [clone(data[0]) for _ in range(2)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for s, h in zip(side, held):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(run(*h))
        graphs.append(g)
    for _ in range(3):
        for h, d in zip(held, (data[1], data[0])):
            for a, b in zip(h, d):
                a.copy_(b)
        torch.cuda.synchronize()
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, h, i in ((outs[0], held[0], 1), (outs[1], held[1], 0)):
            for a, b in zip(o + (h[3], h[4]), first[i] + (copies[i][3], copies[i][4])):
                assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def test_versions_move_on(cuda):
    """What autograd saved before pages were written is known to be stale."""
    from f3m_b200 import paged, sequence as sq
    kp, vp, table = cache(170, [3], [1], 1, 16, 8, torch.float16)
    k = normal(171, 1, 1, 16, dtype=torch.float16)
    before = kp._version, vp._version
    paged.paged_append(sq.SequencePlan([1]), k, k, kp, vp, table, ints([3]))
    assert kp._version > before[0] and vp._version > before[1]
    before = kp._version
    paged.paged_keep(kp, vp, table, ints([3]), ints([[0]]), ints([1]))
    assert kp._version > before


def test_nothing_to_do(cuda):
    from f3m_b200 import paged, sequence as sq
    kp, vp, table = cache(180, [3, 4], [0, 0], 1, 16, 8, torch.float16)
    none = torch.zeros(0, 2, 16, device="cuda", dtype=torch.float16)
    for new, t, lens in (([0, 0], table, [3, 4]), ([], table[:0], [])):
        plan, lens = sq.SequencePlan(new), ints(lens)
        assert paged.paged_append(plan, none[:, :1], none[:, :1], kp, vp, t, lens, q=none).shape == (0, 2, 16)
        assert paged.paged_attention(plan, none, kp, vp, t, lens).shape == (0, 2, 16)
        paged.paged_keep(kp, vp, t, lens, torch.zeros(len(new), 0, device="cuda", dtype=torch.int32), torch.zeros(len(new), device="cuda", dtype=torch.int32))


def test_refusals(cuda):
    from f3m_b200 import paged, sequence as sq
    dtype = torch.bfloat16
    new, cached = [2, 1], [10, 20]
    plan, lens = sq.SequencePlan(new), ints(cached)
    kp, vp, table = cache(190, cached, new, 2, 32, 16, dtype)
    q, k = normal(191, 3, 4, 32, dtype=dtype), normal(192, 3, 2, 32, dtype=dtype)
    par = ints([-1, 0, -1])
    att = lambda **o: paged.paged_attention(**{**dict(plan=plan, q=q, k_pages=kp, v_pages=vp, page_table=table, lengths=lens), **o})  # noqa: E731
    app = lambda **o: paged.paged_append(**{**dict(plan=plan, k=k, v=k, k_pages=kp, v_pages=vp, page_table=table, lengths=lens), **o})  # noqa: E731
    long = sq.SequencePlan([300, 1])
    many = normal(193, 301, 4, 32, dtype=dtype)
    for call in (lambda: att(q=q[:2]), lambda: att(q=q[:, :3]), lambda: att(q=q[..., :24]), lambda: att(k_pages=kp[:, :12], v_pages=vp[:, :12]), lambda: att(k_pages=kp[:, :4], v_pages=vp[:, :4]),
                 lambda: att(v_pages=vp[:-1]), lambda: att(k_pages=kp[..., ::2], v_pages=vp[..., ::2]), lambda: att(plan=sq.SequencePlan([3])), lambda: att(window=0), lambda: att(sinks=-1),
                 lambda: att(plan=long, q=many, parents=ints([-1] * 301)), lambda: att(q=normal(194, 3, 258, 32, dtype=dtype)), lambda: att(page_table=table[0]),
                 lambda: att(k_pages=kp[:1].expand(4, -1, -1, -1), v_pages=vp[:4]), lambda: app(v=k[:2]), lambda: app(k=q, v=q), lambda: app(q=q[:2]), lambda: app(rotation=paged.Rotation(48)),
                 lambda: paged.Rotation(24), lambda: paged.Rotation(144), lambda: paged.Rotation(32, frequencies=[1.0]), lambda: paged.Rotation(32, base=-1.0),
                 lambda: paged.Rotation(32, device="cpu"), lambda: paged.paged_keep(kp, vp, table, lens, ints([1, 2]), ints([1, 1]))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: att(lengths=lens.long()), lambda: att(page_table=table.long()), lambda: att(page_table=table[:1]), lambda: att(parents=par[:2]), lambda: att(parents=par.long()),
                 lambda: att(q=q.half()), lambda: att(q=q.float(), k_pages=kp.float(), v_pages=vp.float()), lambda: app(parents=par.cpu()),
                 lambda: paged.paged_keep(kp, vp, table, lens, ints([[0], [0]]), ints([1]))):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: att(q=q.clone().requires_grad_(True)), lambda: app(k=k.clone().requires_grad_(True)),
                 lambda: paged.paged_keep(kp.clone().requires_grad_(True), vp, table, lens, ints([[0], [0]]), ints([1, 1]))):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(RuntimeError):          # the library's own check
        att(scale=float("inf"))


def test_pages_behind_two_billion_elements(cuda):
    """Sequences whose pages lie at the end of arrays of more than 2^31 elements: the bits that they have in small ones."""
    from f3m_b200 import paged, sequence as sq
    new, cached, page, kv, w, dtype = [3, 20], [700, 129], 256, 8, 128, torch.bfloat16
    plan, rotation, lens = sq.SequencePlan(new), paged.Rotation(w), ints(cached)
    kp, vp, table = cache(200, cached, new, kv, w, page, dtype, garbage=0.0)
    pool = (1 << 31) // (page * kv * w) + 5 + kp.shape[0]
    big = [torch.empty(pool, page, kv, w, device="cuda", dtype=dtype) for _ in range(2)]
    far = table + (pool - kp.shape[0])
    for x, y in zip(big, (kp, vp)):
        x[-kp.shape[0]:] = y
    k, v, q = normal(201, 23, kv, w, dtype=dtype), normal(202, 23, kv, w, dtype=dtype), normal(203, 23, 32, w, dtype=dtype)
    parents, kept, counts = trees(204, new), ints([[0, 2], [3, 7]]), ints([2, 2])
    outs = []
    for a, b, t in ((kp, vp, table), (*big, far)):
        qq = paged.paged_append(plan, k, v, a, b, t, lens, rotation, parents, q)
        outs.append(paged.paged_attention(plan, qq, a, b, t, lens, parents=parents))
        paged.paged_keep(a, b, t, lens, kept, counts)
    assert torch.equal(*outs) and all(torch.equal(x[-kp.shape[0]:], y) for x, y in zip(big, (kp, vp)))


def test_outputs_between_other_data(cuda):
    """The C entries turn queries in place, and write rows that lie between others, and nothing else."""
    import ctypes as C

    from f3m_b200 import _lib, paged, sequence as sq
    new, cached, page, kv, heads, w, dtype = [5, 40], [300, 64], 64, 2, 6, 64, torch.float16
    plan, rotation, lens, n = sq.SequencePlan(new), paged.Rotation(w), ints(cached), 45
    kp, vp, table = cache(210, cached, new, kv, w, page, dtype)
    k, v, q = normal(211, n, kv, w, dtype=dtype), normal(212, n, kv, w, dtype=dtype), normal(213, n, heads, w, dtype=dtype)
    want_q = paged.paged_append(plan, k, v, kp, vp, table, lens, rotation, q=q)
    want = paged.paged_attention(plan, want_q, kp, vp, table, lens)
    c, held = paged._cache(kp, vp, table, lens)
    rows = lambda t: _lib.Rows(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
    L, stream, wide = _lib.lib(), torch.cuda.current_stream().cuda_stream, normal(214, heads + 1, n, 2 * w, dtype=dtype)
    out = wide[1:, :, w:].transpose(0, 1)
    before = wide.clone()
    assert L.f3m_paged_append(plan._ref, 2, C.byref(c), rows(k), rows(v), None, rotation._ref, heads, rows(q), rows(q), stream) == 0
    need = L.f3m_paged_attention_workspace_bytes(plan._ref, C.byref(c), heads)
    ws = torch.full((need + 64,), 0xa5, device="cuda", dtype=torch.uint8)
    assert L.f3m_paged_attention(plan._ref, 2, C.byref(c), heads, 0x7fffffff, 0, w ** -0.5, None, rows(q), rows(out), ws.data_ptr(), need, stream) == 0
    assert torch.equal(q, want_q) and torch.equal(out, want) and (ws[need:] == 0xa5).all()
    before[1:, :, w:] = wide[1:, :, w:]
    assert torch.equal(wide, before)


def test_calls_from_several_host_threads(cuda):
    """Each thread on its own stream, all at once: the bits of the calls alone."""
    import threading

    from f3m_b200 import paged, sequence as sq
    new, dtype = [6, 1, 30], torch.bfloat16
    plan, jobs, got = sq.SequencePlan(new), [], [None] * 4
    x, ld = normal(225, 5000, 512, dtype=dtype), -normal(226, 5000, 512, dtype=dtype).abs() * 0.1
    line = sq.SequencePlan([5000])
    for i in range(4):
        cached = [500 * (i + 1), 3000, 17 * i]
        kp, vp, table = cache(220 + i, cached, new, 2, 64, 32, dtype)
        jobs.append((normal(230 + i, 37, 8, 64, dtype=dtype), kp, vp, table, ints(cached)))
    want = [paged.paged_attention(plan, *j) for j in jobs]
    h = sq.gated_recurrence(line, x, ld)
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got[i] = (paged.paged_attention(plan, *jobs[i]), *sq.gated_recurrence(line, x, ld))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b) and torch.equal(a[1], h[0]) and torch.equal(a[2], h[1])
