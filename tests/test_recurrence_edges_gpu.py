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
