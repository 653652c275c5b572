"""The gated recurrence where inputs and states are infinite: what the definition makes of them, wherever a run or a tile begins."""
import pytest
import torch

from test_recurrence_gpu import inputs, states

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
INF, NAN = float("inf"), float("nan")


def definition(x, ld, lengths, state):
    """h of every token and behind the last ones, in 64 bits"""
    a, hs, last, t = torch.exp(ld.double().clamp(max=0)), torch.empty_like(x, dtype=torch.float64), [], 0
    for s, n in enumerate(lengths):
        h = state[s].double()
        for _ in range(n):
            hs[t] = h = a[t] * h + x[t].double()
            t += 1
        last.append(h)
    return hs, torch.stack(last)


def same_kind(got, want, what=""):
    """Infinite, of which sign, or not a number, in the same places"""
    for is_ in (torch.isnan, torch.isposinf, torch.isneginf):
        bad = is_(got) != is_(want)
        assert not bad.any(), (what, is_.__name__, bad.nonzero()[:5].tolist())


def infinite(seed, lengths, dtype, channels=40):
    """x, log_decay, state.  Decays of all speeds, by channel: none, slow, products that leave FP32's range within a tile, within a run; no memory at all here and there"""
    n = sum(lengths)
    x, ld = inputs(seed, n, channels, dtype)
    st = states(seed + 1, len(lengths), channels)
    for c, d in enumerate((0.0, -1e-3, -0.1, -0.3, -0.6, -2.0, -8.0, -60.0)):
        ld[:, c::8] = d
    ld[37::100, 32:] = -INF
    x[::7, 16:24] = 0.0
    for c in range(channels):
        kind = c // 8
        if kind in (0, 4):
            st[:, c] = INF if c % 2 else -INF
        if kind in (1, 4):
            x[(61 * c) % n, c] = INF
        if kind == 2:
            x[(29 * c) % n, c] = -INF
        if kind == 3:
            st[:, c], x[(150 + c) % n, c] = INF, -INF
    return x, ld, st


LENGTHS = [[3], [1500], [129, 1, 700, 16]]


@pytest.mark.parametrize("dtype", TYPES)
def test_steps_from_infinite_states(dtype, cuda):
    from f3m_b200 import sequence as sq
    n = 60
    x, ld, st = infinite(1, [1] * n, dtype)
    ld[::9, ::3] = 0.0
    want, _ = definition(x, ld, [1] * n, st)
    got = sq.gated_recurrence_step(x, ld, st)
    same_kind(got, want)
    same_kind(st, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", LENGTHS)
def test_infinite_inputs_and_states(lengths, dtype, cuda):
    from f3m_b200 import sequence as sq
    x, ld, st = infinite(2, lengths, dtype)
    out, final = sq.gated_recurrence(sq.SequencePlan(lengths), x, ld, st)
    want, last = definition(x, ld, lengths, st)
    same_kind(out, want, "out")
    same_kind(final, last, "final")
    # channels without any: the bits of a call by themselves
    x2, ld2 = inputs(2, sum(lengths), 40, dtype)
    clean = sq.gated_recurrence(sq.SequencePlan(lengths), x2, ld2)
    x2[0, 3], st2 = INF, torch.zeros_like(st)
    st2[:, 7] = -INF
    rest = [c for c in range(40) if c not in (3, 7)]
    for a, b in zip(sq.gated_recurrence(sq.SequencePlan(lengths), x2, ld2, st2), clean):
        assert torch.equal(a[:, rest], b[:, rest])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", LENGTHS)
def test_infinite_gradients(lengths, dtype, cuda):
    """The recurrence from the end: what flows back through a token is a_t (dout_t + ..)."""
    from f3m_b200 import sequence as sq
    do, ld, df = infinite(3, lengths, dtype)
    out = inputs(4, sum(lengths), 40, dtype)[0]
    dx, _, dstate = sq.gated_recurrence_grad(sq.SequencePlan(lengths), ld, out, do, None, df)
    want, flows, r0 = torch.empty_like(do, dtype=torch.float64), [], 0
    a = torch.exp(ld.double().clamp(max=0))
    for s, n in enumerate(lengths):
        c = df[s].double()
        for t in range(r0 + n - 1, r0 - 1, -1):
            want[t] = do[t].double() + c
            c = a[t] * want[t]
        flows.append(c)
        r0 += n
    same_kind(dx, want, "dx")
    same_kind(dstate, torch.stack(flows), "dstate")


@pytest.mark.parametrize("dtype", TYPES)
def test_decays_that_are_zero_in_float32(dtype, cuda):
    """exp(-200) is: what was infinite is not a number behind it, wherever that token lies, in prompts as in steps; what was finite is forgotten."""
    from f3m_b200 import sequence as sq
    n, c = 700, 16
    plan = sq.SequencePlan([n])
    for at in (0, 5, 127, 128, 300, 699):
        x, ld = inputs(5, n, c, dtype)
        st = states(6, 1, c)
        ld[at, :8] = -200.0
        st[:, ::2] = INF
        out, final = sq.gated_recurrence(plan, x, ld, st)
        assert (out[:at, ::2] == INF).all() and out[at:, :8:2].isnan().all() and (out[at:, 8::2] == INF).all() and torch.isfinite(out[:, 1::2]).all()
        assert torch.equal(out[at, 1:8:2], x[at, 1:8:2])
        same_kind(final[0], out[-1])
        h = st[:, :].clone()
        sq.gated_recurrence_step(x[at:at + 1], ld[at:at + 1], h)
        same_kind(h[0], out[at])


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_before_an_infinite_one_keep_their_bits(dtype, cuda):
    """Forward those before it, backward those behind it; and calls with infinite numbers repeat their bits."""
    from f3m_b200 import sequence as sq
    n, c = 1900, 72
    plan = sq.SequencePlan([n])
    x, ld = inputs(7, n, c, dtype)
    do = inputs(8, n, c, dtype)[0]
    out, _ = sq.gated_recurrence(plan, x, ld)
    dx, dl, _ = sq.gated_recurrence_grad(plan, ld, out, do)
    for at in (0, 5, 640, 700, 1899):
        for bad in (INF, -INF, NAN):
            x2, do2 = x.clone(), do.clone()
            x2[at, 3::5], do2[at, 1::4] = bad, bad
            o, f = sq.gated_recurrence(plan, x2, ld)
            assert torch.equal(o[:at], out[:at]) and not torch.isfinite(o[at:, 3::5]).any() and not torch.isfinite(f[0, 3::5]).any()
            gx, gl, gs = sq.gated_recurrence_grad(plan, ld, out, do2)
            assert torch.equal(gx[at + 1:], dx[at + 1:]) and torch.equal(gl[at + 1:], dl[at + 1:]) and not torch.isfinite(gx[:at + 1, 1::4]).any() and not torch.isfinite(gs[0, 1::4]).any()
            for _ in range(5):
                again = sq.gated_recurrence(plan, x2, ld) + sq.gated_recurrence_grad(plan, ld, out, do2)
                assert all(torch.equal(a.nan_to_num(7.0, 8.0, 9.0), b.nan_to_num(7.0, 8.0, 9.0)) for a, b in zip(again, (o, f, gx, gl, gs)))
