"""Kernel products over sequences: repeated calls at uneven widths, batches of very uneven lengths, small gradients, values that are not numbers."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def normal(seed, *shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


@pytest.mark.parametrize("width_k,width_v", [(128, 64), (64, 128), (128, 128), (128, 8), (64, 64)])
def test_many_calls_of_attention_with_a_decay(width_k, width_v, cuda):
    """The weights of a tile may be ready before the products ask for those of the tile before, most easily where width_v is small and width_k
    is not: the same bits from call to call, and no wait runs out."""
    from f3m_b200 import sequence as sq
    lengths, h = [6000, 1, 2300, 130], 16
    n = sum(lengths)
    q, k = normal(1, n, h, width_k, dtype=torch.bfloat16), normal(2, n, h, width_k, dtype=torch.bfloat16)
    v, do = normal(3, n, h, width_v, dtype=torch.bfloat16), normal(4, n, h, width_v, dtype=torch.bfloat16)
    state, dfinal = (normal(5 + i, len(lengths), h, width_k, width_v, dtype=torch.float32) for i in range(2))
    ld = -torch.exp2(-torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / 2)
    plan = sq.SequencePlan(lengths)

    def calls():
        return sq.decay_attention(plan, q, k, v, ld, state) + sq.decay_attention_grad(plan, q, k, v, ld, do, state, dfinal)

    first = calls()
    for _ in range(100):
        assert all(torch.equal(x, y) for x, y in zip(calls(), first))
    want = ref.decay(q[:, :1], k[:, :1], v[:, :1], ld[:1].tolist(), lengths, state[:, :1], dout=do[:, :1], dfinal=dfinal[:, :1])
    for name, x in zip(("out", "final", "dq", "dk", "dv", "dstate"), first):
        ref.assert_within(x[:, :1], want[name], name)


# lengths, heads, kv_heads, width, window, sinks: walks over sinks that are cut, of few sequences among many, at the front, the end and between
UNEVEN = [
    ([3000] + [64] * 60, 8, 2, 64, 128, 8),
    ([64] * 30 + [3300, 0, 1, 1700] + [130] * 20, 8, 2, 128, 100, 200),
    ([5, 0, 4100], 12, 1, 32, 129, 300),
    ([2900, 2900, 64, 3100], 16, 2, 80, 300, 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,kv_heads,width,window,sinks", UNEVEN)
def test_window_gradients_of_uneven_batches(lengths, heads, kv_heads, width, window, sinks, dtype, cuda):
    from f3m_b200 import sequence as sq
    n = sum(lengths)
    q, do = normal(1, n, heads, width, dtype=dtype), normal(2, n, heads, width, dtype=dtype)
    k, v = normal(3, n, kv_heads, width, dtype=dtype), normal(4, n, kv_heads, width, dtype=dtype)
    plan = sq.SequencePlan(lengths)
    want = ref.window(q, k, v, lengths, window, sinks, dout=do)
    out, lse = sq.window_attention(plan, q, k, v, window, sinks)
    first = sq.window_attention_grad(plan, q, k, v, out, lse, do, window, sinks)
    for name, x in zip(("dq", "dk", "dv"), first):
        ref.assert_within(x, want[name], name)
    again = sq.window_attention_grad(plan, q, k, v, out, lse, do, window, sinks)
    assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_window_gradients_of_thousands_of_short_sequences(cuda):
    """One document beside 2000 short ones: a workspace no larger than the arrays, and the gradients that each has by itself."""
    from f3m_b200 import sequence as sq
    lengths, h, hk, w, window, sinks = [16384] + [64] * 2000, 32, 8, 128, 128, 4
    n = sum(lengths)
    q, do = normal(1, n, h, w, dtype=torch.bfloat16), normal(2, n, h, w, dtype=torch.bfloat16)
    k, v = normal(3, n, hk, w, dtype=torch.bfloat16), normal(4, n, hk, w, dtype=torch.bfloat16)

    def both(plan, at):
        x = [y[at] for y in (q, k, v, do)]
        out, lse = sq.window_attention(plan, *x[:3], window, sinks)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        got = sq.window_attention_grad(plan, *x[:3], out, lse, x[3], window, sinks)
        torch.cuda.synchronize()
        return got, torch.cuda.max_memory_allocated() - held - sum(y.numel() * 2 for y in got)

    got, room = both(sq.SequencePlan(lengths), slice(0, n))
    assert room < q.numel() * 2
    for at, few in ((slice(0, 16384), [16384]), (slice(16384, 16384 + 6400), [64] * 100), (slice(n - 64, n), [64])):
        want, _ = both(sq.SequencePlan(few), at)
        for x, y in zip(got, want):     # parts may be cut otherwise: sums in FP32, rounded once
            assert torch.allclose(x[at].float(), y.float(), rtol=2 ** -7, atol=1e-4)


def scaled_up(f, dout, up, **also):
    """What f gives for dout (and dfinal) times `up`, a power of two, scaled back: gradients are linear in them, and so are bounds that do not depend
    on their size.  What is rounded to fp16 in the end may be subnormal: half of 2^-24."""
    want = f(dout.double() * up, **{n: x.double() * up for n, x in also.items() if x is not None})
    return {n: (value / up, bound / up + 2.0 ** -25) for n, (value, bound) in want.items()}


@pytest.mark.parametrize("size", [2.0 ** 8, 1.0, 2.0 ** -10, 2.0 ** -13, 2.0 ** -15])
def test_window_gradients_of_any_size_in_fp16(size, cuda):
    """dS is a weight times a difference, far below dout: it keeps its bits where dout does, in each sequence by itself."""
    from f3m_b200 import sequence as sq
    lengths, h, hk, w, window, sinks = [900, 130, 400], 4, 2, 64, 512, 4
    n = sum(lengths)
    q, k, v = (normal(i, n, g, w, dtype=torch.float16) for i, g in enumerate((h, hk, hk)))
    do = normal(3, n, h, w, dtype=torch.float32)
    do[:900] *= size
    do[1030:] *= 64 * size if size < 1 else 1
    do = do.half()
    do[900:1030] = 0
    plan = sq.SequencePlan(lengths)
    out, lse = sq.window_attention(plan, q, k, v, window, sinks)
    got = sq.window_attention_grad(plan, q, k, v, out, lse, do, window, sinks)
    for at, up in ((slice(0, 900), 1 / size), (slice(900, 1030), 1.0), (slice(1030, n), 1 / (64 * size) if size < 1 else 1.0)):
        q1, k1, v1, d1 = (x[at] for x in (q, k, v, do))
        want = scaled_up(lambda d: ref.window(q1, k1, v1, [q1.shape[0]], window, sinks, dout=d), d1, up)
        for name, x in zip(("dq", "dk", "dv"), got):
            ref.assert_within(x[at], want[name], f"{name} at {size}")


def test_captured_gradients_in_fp16_take_their_range_from_each_replay(cuda):
    from f3m_b200 import sequence as sq
    lengths, h, w = [333, 129], 2, 64
    n = sum(lengths)
    plan = sq.SequencePlan(lengths)
    q, k, v, do = (normal(i, n, h, w, dtype=torch.float16) for i in range(4))

    def train():
        out, lse = sq.window_attention(plan, q, k, v, 100, 3)
        return sq.window_attention_grad(plan, q, k, v, out, lse, do, 100, 3)

    train()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = train()
    for size in (1.0, 2.0 ** 9, 2.0 ** -13, 1.0):
        do.copy_(normal(9, n, h, w, dtype=torch.float16, scale=size))
        v.copy_(normal(10, n, h, w, dtype=torch.float16, scale=min(1.0, 1 / size)))
        g.replay()
        assert all(torch.equal(x, y) for x, y in zip(train(), res)), size


@pytest.mark.parametrize("carried", [False, True])
@pytest.mark.parametrize("size", [2.0 ** 6, 1.0, 2.0 ** -10, 2.0 ** -13, 2.0 ** -15])
def test_decay_gradients_of_any_size_in_fp16(size, carried, cuda):
    """Weights and states that small gradients go into keep their bits where these do, in each sequence and head by itself; in one range and in several."""
    from f3m_b200 import sequence as sq
    h, wk, wv, lengths = 2, 64, 80, [2500, 0, 300]
    n, log_decay = sum(lengths), [-0.02, -0.4]
    ld = torch.tensor(log_decay, device="cuda")
    q, k, v, do = normal(1, n, h, wk, dtype=torch.float16), normal(2, n, h, wk, dtype=torch.float16), normal(3, n, h, wv, dtype=torch.float16), normal(4, n, h, wv, dtype=torch.float32)
    state = normal(5, 3, h, wk, wv, dtype=torch.float32) if carried else None
    dfinal = normal(6, 3, h, wk, wv, dtype=torch.float32) * size if carried else None
    do[:, 0] *= size
    do[:, 1] *= size * 2 ** 4
    do = do.half()
    if carried:
        dfinal[:, 1] *= 2 ** 4
    plan = sq.SequencePlan(lengths)
    got = sq.decay_attention_grad(plan, q, k, v, ld, do, state, dfinal)
    for a in range(h):
        one = slice(a, a + 1)
        want = scaled_up(lambda d, dfinal=None: ref.decay(q[:, one], k[:, one], v[:, one], log_decay[one], lengths, None if state is None else state[:, one], dout=d, dfinal=dfinal),
                         do[:, one], 1 / (size * 2 ** (4 * a)), dfinal=None if dfinal is None else dfinal[:, one])
        for name, x in zip(("dq", "dk", "dv", "dstate"), got):
            ref.assert_within(x[:, one], want[name], f"{name}, head {a} at {size}")


@pytest.mark.parametrize("dtype", TYPES)
def test_a_key_that_is_not_a_number_reaches_all_that_see_it(dtype, cuda):
    """Wherever the key stands in its tile, and in tiles that are seen whole."""
    from f3m_b200 import sequence as sq
    n, h, w, window = 512, 1, 64, 300
    plan = sq.SequencePlan([n])
    q, k, v, do = (normal(40 + i, n, h, w, dtype=dtype) for i in range(4))
    out, lse = sq.window_attention(plan, q, k, v, window)
    i = torch.arange(n, device="cuda")
    for j in (*range(128, 144), 255):
        bad = k.clone()
        bad[j] = float("nan")
        sees = (i >= j) & (i - j < window)
        got = sq.window_attention(plan, q, bad, v, window)
        assert got[0][sees].isnan().all() and got[1][0, sees].isnan().all(), j
        dq, dk, dv = sq.window_attention_grad(plan, q, bad, v, out, lse, do, window)
        assert dq[sees].isnan().all() and dk[j].isnan().all() and dv[j].isnan().all(), j
    inf = k.clone()
    inf[:] = float("inf")
    assert not torch.isfinite(sq.window_attention(plan, q.abs() * -1, inf, v, window)[0]).any()      # every exponent -inf: no row is a mean of values


@pytest.mark.parametrize("dtype", TYPES)
def test_a_decay_that_is_not_a_number_is_not_one(dtype, cuda):
    from f3m_b200 import sequence as sq
    lengths, h, w = [300, 20], 2, 64
    n = sum(lengths)
    plan = sq.SequencePlan(lengths)
    q, k, v, do = (normal(50 + i, n, h, w, dtype=dtype) for i in range(4))
    good = torch.tensor([-0.1, -0.1], device="cuda")
    ld = torch.tensor([float("nan"), -0.1], device="cuda")
    got = sq.decay_attention(plan, q, k, v, ld) + sq.decay_attention_grad(plan, q, k, v, ld, do)
    want = sq.decay_attention(plan, q, k, v, good) + sq.decay_attention_grad(plan, q, k, v, good, do)
    for x, y in zip(got, want):
        assert x[:, 0].isnan().all() and torch.equal(x[:, 1], y[:, 1])
    s = normal(60, 3, h, w, w, dtype=torch.float32)
    out = sq.decay_attention_step(q[:3], k[:3], v[:3], ld, s)
    assert out[:, 0].isnan().all() and s[:, 0].isnan().all() and torch.isfinite(out[:, 1]).all() and torch.isfinite(s[:, 1]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("capacity", [200, 5000])
def test_a_step_does_not_lose_what_is_not_a_number(capacity, dtype, cuda):
    """A seen key or value that is not a number, among finite ones, in a part of its own, and as a part's only keys; in a cache taken whole and in parts."""
    from f3m_b200 import sequence as sq
    h, w = 4, 64
    q = normal(1, 1, h, w, dtype=dtype)
    kc, vc = normal(2, 1, capacity, 2, w, dtype=dtype), normal(3, 1, capacity, 2, w, dtype=dtype)
    lens = torch.tensor([capacity], dtype=torch.int32, device="cuda")
    assert torch.isfinite(sq.window_attention_step(q, kc, vc, lens, capacity)).all()
    for at in (slice(0, 1), slice(capacity - 1, capacity), slice(capacity // 2, capacity // 2 + 3), slice(0, capacity // 2), slice(0, capacity)):
        for which in (0, 1):
            x = [kc.clone(), vc.clone()]
            x[which][:, at, 0] = float("nan")
            got = sq.window_attention_step(q, *x, lens, capacity)
            assert got[:, :2].isnan().all() and torch.isfinite(got[:, 2:]).all(), (at, which)
    far = kc.clone()
    far[:, :64] = float("nan")         # and where what is finite weighs far more
    far[:, 64:] = 60 * q[:, :1].sign()
    assert sq.window_attention_step(q[:, :1].repeat(1, 4, 1), far, vc, lens, capacity, scale=1.0).isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (4, 2), (2, 2)])
def test_what_is_not_finite_stays_with_the_tiles_that_see_it(heads, kv_heads, dtype, cuda):
    """Tiles of 128 queries whose window ends before a token's tile, or begins behind it, do not notice what it holds."""
    from f3m_b200 import sequence as sq
    n, w, window, sinks = 900, 64, 130, 3
    plan = sq.SequencePlan([n])
    q, k, v = normal(1, n, heads, w, dtype=dtype), normal(2, n, kv_heads, w, dtype=dtype), normal(3, n, kv_heads, w, dtype=dtype)
    want, lse = sq.window_attention(plan, q, k, v, window, sinks)
    i = torch.arange(n, device="cuda")
    for t in range(1, 7):       # tile 0 holds the sinks: it is seen by all
        for worst in (float("nan"), float("inf")):
            kk, vv = k.clone(), v.clone()
            vv[128 * t + 5] = worst
            kk[128 * t + 77] = worst
            got, l = sq.window_attention(plan, q, kk, vv, window, sinks)
            # a tile of queries sees tile t of keys if one of its queries, from 128 tile to 128 tile + 127, sees one of its keys
            tile = i // 128
            sees = (tile >= t) & (128 * tile - (128 * t + 127) < window)
            assert torch.equal(got[~sees], want[~sees]) and torch.equal(l[:, ~sees], lse[:, ~sees]), t
            assert got[128 * t + 77].isnan().all()


def test_a_step_at_the_end_of_the_longest_cache(cuda):
    """Numbers of keys whose sum with a part's length passes 2^31: the last part's keys, which weigh all."""
    from f3m_b200 import sequence as sq
    cap, w, last, dtype = 0x7fffff00, 8, 100, torch.bfloat16
    cache = torch.zeros(1, cap, 1, w, device="cuda", dtype=dtype)          # keys and values are the same
    cache[0, -last:, 0] = 2 + normal(1, last, w, dtype=dtype, scale=0.25)
    q = torch.full((1, 1, w), 8.0, device="cuda", dtype=dtype)
    got = sq.window_attention_step(q, cache, cache, torch.tensor([cap], dtype=torch.int32, device="cuda"), cap)
    kd = cache[0, -last:, 0].double()
    weights = torch.exp(kd @ q[0, 0].double() * w ** -0.5 - 40)            # the others have exp(-40) each
    want = weights @ kd / (weights.sum() + (cap - last) * torch.exp(torch.tensor(-40.0, dtype=torch.float64, device="cuda")))
    del cache
    # the weights and the output are rounded to 16 bits; the row sum adds 2^31 numbers in FP32, which may fall below its last place
    ref.assert_within(got[0, 0], (want, (3 * ref.half_step(dtype) + 1e-4) * want.abs()))


def test_every_call_reports_a_wait_that_ran_out(cuda):
    """The word that a kernel would set, set by hand: the next call is refused, whichever it is, enqueues nothing, and the one behind it runs."""
    from f3m_b200 import _lib, sequence as sq
    word = _lib.lib().f3m_seqs_error_word()
    n, h, w = 40, 2, 64
    plan, ld = sq.SequencePlan([n]), torch.tensor([-0.1, -0.2], device="cuda")
    x = normal(1, n, h, w, dtype=torch.bfloat16)
    lens, state = torch.full((n,), 1, dtype=torch.int32, device="cuda"), torch.ones(n, h, w, w, device="cuda")
    out, lse = sq.window_attention(plan, x, x, x, 10)
    calls = [lambda: sq.window_attention(plan, x, x, x, 10), lambda: sq.window_attention_grad(plan, x, x, x, out, lse, x, 10),
             lambda: sq.window_attention_step(x, x[:, None], x[:, None], lens, 10), lambda: sq.decay_attention(plan, x, x, x, ld),
             lambda: sq.decay_attention_grad(plan, x, x, x, ld, x), lambda: sq.decay_attention_step(x, x, x, ld, state)]
    for call in calls:
        torch.cuda.synchronize()
        assert word[0] == 0
        word[0] = 1
        with pytest.raises(_lib.F3MError, match="gave up"):
            call()
        assert word[0] == 0 and bool((state == 1).all())
    for call in calls:
        call()
    torch.cuda.synchronize()
    assert word[0] == 0


def test_calls_from_several_host_threads(cuda):
    """Each thread on its own stream, all at once: the bits of the calls alone."""
    import threading
    from f3m_b200 import sequence as sq
    lengths, h, w = [2500, 17, 400], 4, 64
    n = sum(lengths)
    ld = torch.tensor([-0.01, -0.1, -0.3, 0.0], device="cuda")
    plan = sq.SequencePlan(lengths)
    kc, vc = normal(8, 2, 3000, 2, w, dtype=torch.float16), normal(9, 2, 3000, 2, w, dtype=torch.float16)
    lens = torch.tensor([3000, 2000], dtype=torch.int32, device="cuda")

    def calls(seed):
        q, k, v, do = (normal(seed + i, n, h, w, dtype=torch.float16) for i in range(4))
        out, lse = sq.window_attention(plan, q, k[:, :2], v[:, :2], 300, 5)
        a = sq.window_attention_grad(plan, q, k[:, :2], v[:, :2], out, lse, do, 300, 5)
        s = normal(seed, 2, h, w, w, dtype=torch.float32)
        step = sq.decay_attention_step(q[:2], k[:2], v[:2], ld, s)
        return (out, lse, s, step) + a + sq.decay_attention(plan, q, k, v, ld) + sq.decay_attention_grad(plan, q, k, v, ld, do) + (sq.window_attention_step(q[:2], kc, vc, lens, 2500, 3),)

    want = {seed: calls(seed) for seed in range(100, 140, 10)}
    torch.cuda.synchronize()
    wrong = []

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = calls(seed)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(x, y) for x, y in zip(got, want[seed])):
                        wrong.append(seed)
        except Exception as e:      # noqa: BLE001  (a thread's failure has to reach the test)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in want]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong, wrong


@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_prompts_and_gradients_behind_two_billion_elements(dtype, cuda):
    """The last sequence of arrays of more than 2^31 elements: the bits it has by itself."""
    from f3m_b200 import sequence as sq
    w, h, last = 128, 16, 300
    n = 2 ** 31 // (h * w) + 4000
    plan, alone = sq.SequencePlan([n - last, last]), sq.SequencePlan([last])
    q = torch.zeros(n, h, w, device="cuda", dtype=dtype)
    k, v = (torch.zeros(n, 1, w, device="cuda", dtype=dtype) for _ in range(2))
    q[-last:], k[-last:], v[-last:] = (normal(i, last, x.shape[1], w, dtype=dtype) for i, x in enumerate((q, k, v)))
    do = q.flip(2)
    t = [x[-last:].clone() for x in (q, k, v, do)]
    want, wl = sq.window_attention(alone, *t[:3], 100, 3)
    wg = sq.window_attention_grad(alone, *t[:3], want, wl, t[3], 100, 3)
    out, lse = sq.window_attention(plan, q, k, v, 100, 3)
    assert torch.equal(out[-last:], want) and torch.equal(lse[:, -last:], wl) and not out[:-last].any()
    got = sq.window_attention_grad(plan, q, k, v, out, lse, do, 100, 3)
    for x, y in zip(got, wg):
        ref.assert_within(x[-last:], (y.double(), y.double().abs() * 2 ** -7 + 1e-5))      # walks over sinks may be cut otherwise
    del got, out, lse, k, v
    ld = -torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / 50
    state = normal(7, 2, h, w, w, dtype=torch.float32)
    want, wf = sq.decay_attention(alone, t[0], t[0], t[3], ld, state[1:])
    out, final = sq.decay_attention(plan, q, q, do, ld, state)
    u = ref.half_step(dtype)
    ref.assert_within(out[-last:], (want.double(), 2 * u * want.double().abs() + 4 * u * want.double().abs().max()))       # states may be joined between ranges
    ref.assert_within(final[1:], (wf.double(), 1e-5 * wf.double().abs().max().expand_as(wf)))
    del out
    got = sq.decay_attention_grad(plan, q, q, do, ld, do, state)
    for x, y in zip(got[:3], sq.decay_attention_grad(alone, t[0], t[0], t[3], ld, t[3], state[1:])[:3]):
        ref.assert_within(x[-last:], (y.double(), 2 * u * y.double().abs() + 4 * u * y.double().abs().max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [128, 72])
def test_outputs_between_other_data(width, dtype, cuda):
    """The C entries write rows that lie between others, heads before tokens or behind them, and nothing else: the bits of dense outputs.  States that are not
    asked for are not needed."""
    from f3m_b200 import _lib, sequence as sq
    from f3m_b200._lib import Rows, check
    L, kind, lengths, h, hk, w = _lib.lib(), {torch.bfloat16: 1, torch.float16: 2}[dtype], [300, 0, 131, 1], 4, 2, width
    n, scale, stream = sum(lengths), width ** -0.5, torch.cuda.current_stream().cuda_stream
    plan, ld = sq.SequencePlan(lengths), torch.tensor([-0.1, -0.01, 0.0, -2.0], device="cuda")
    q, do = normal(1, n, h, w, dtype=dtype), normal(2, n, h, w, dtype=dtype)
    k, v = normal(3, n, h, w, dtype=dtype), normal(4, n, h, w, dtype=dtype)
    k2, v2 = k[:, :hk], v[:, :hk]
    lens, state0 = torch.tensor([200, 17, 0], dtype=torch.int32, device="cuda"), normal(5, 3, h, w, w, dtype=torch.float32)
    cache = normal(6, 3, 256, hk, w, dtype=dtype)
    rows = lambda t: Rows(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
    held = []

    def place(tokens, heads, order):
        """(tokens, heads, w) rows inside a larger array of sevens"""
        if order:
            a = torch.full((heads + 1, tokens + 3, w + 24), 7.0, device="cuda", dtype=dtype)
            x = a[:heads, 2:2 + tokens, 8:8 + w].transpose(0, 1)
        else:
            a = torch.full((tokens + 2, 3, heads, w + 8), 7.0, device="cuda", dtype=dtype)
            x = a[1:1 + tokens, 1, :, :w]
        held.append((a, x))
        return x

    def work(n):
        return torch.empty(max(n, 16), device="cuda", dtype=torch.uint8)

    out, lse = sq.window_attention(plan, q, k2, v2, 100, 3)
    grads = sq.window_attention_grad(plan, q, k2, v2, out, lse, do, 100, 3)
    dec, final = sq.decay_attention(plan, q, k, v, ld)
    step = sq.window_attention_step(q[:3], cache, cache, lens, 150, 2)
    state = state0.clone()
    dstep = sq.decay_attention_step(q[:3], k[:3], v[:3], ld, state)
    for order in (False, True):
        held.clear()
        x, l2 = place(n, h, order), torch.empty_like(lse)
        check(L.f3m_window_attention(plan._ref, kind, h, hk, w, 100, 3, scale, rows(q), rows(k2), rows(v2), rows(x), l2.data_ptr(), stream), "")
        assert torch.equal(x, out) and torch.equal(l2, lse)
        d = [place(n, g, order) for g in (h, hk, hk)]
        need = L.f3m_window_attention_grad_workspace_bytes(plan._ref, h, hk, w, 100, 3)
        ws = work(need)
        check(L.f3m_window_attention_grad(plan._ref, kind, h, hk, w, 100, 3, scale, rows(q), rows(k2), rows(v2), rows(x), l2.data_ptr(), rows(do), *map(rows, d),
                                          ws.data_ptr(), need, stream), "")
        assert all(torch.equal(a, b) for a, b in zip(d, grads))
        x, need = place(n, h, order), L.f3m_decay_attention_workspace_bytes(plan._ref, h, w, w)
        ws, f = work(need), torch.empty_like(final)
        check(L.f3m_decay_attention(plan._ref, kind, h, w, w, ld.data_ptr(), scale, rows(q), rows(k), rows(v), None, rows(x), f.data_ptr(), ws.data_ptr(), need, stream), "")
        assert torch.equal(x, dec) and torch.equal(f, final)
        # without the last state it is carried in two parts, and out may round otherwise
        x = place(n, h, order)
        check(L.f3m_decay_attention(plan._ref, kind, h, w, w, ld.data_ptr(), scale, rows(q), rows(k), rows(v), None, rows(x), None, ws.data_ptr(), need, stream), "")
        want = ref.decay(q, k, v, ld.tolist(), lengths, dout=do)
        ref.assert_within(x, want["out"])
        d = [place(n, h, order) for _ in range(3)]
        check(L.f3m_decay_attention_grad(plan._ref, kind, h, w, w, ld.data_ptr(), scale, rows(q), rows(k), rows(v), None, rows(do), None, *map(rows, d), None,
                                         ws.data_ptr(), need, stream), "")
        for name, a in zip(("dq", "dk", "dv"), d):
            ref.assert_within(a, want[name], name)
        x, need = place(3, h, order), L.f3m_window_attention_step_workspace_bytes(3, h, hk, w, 256, 150, 2)
        ws = work(need)
        check(L.f3m_window_attention_step(3, kind, h, hk, w, 256, 150, 2, scale, rows(q), rows(cache[0]), cache.stride(0), rows(cache[0]), cache.stride(0), lens.data_ptr(),
                                          rows(x), ws.data_ptr(), need, stream), "")
        assert torch.equal(x, step)
        x, s = place(3, h, order), state0.clone()
        check(L.f3m_decay_attention_step(3, kind, h, w, w, ld.data_ptr(), scale, rows(q), rows(k), rows(v), s.data_ptr(), rows(x), stream), "")
        assert torch.equal(x, dstep) and torch.equal(s, state)
        for a, x in held:
            x.fill_(7.0)
            assert bool((a == 7.0).all())
