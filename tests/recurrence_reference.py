"""The gated recurrence in 64 bits, token by token, and how far a kernel's roundings may take it.

Every function returns, for each output, (value, bound).  A step a h + x is off by two roundings to FP32 of sums whose absolute values are `mass`, and by what a itself is off:
next to 1, where it is 1 + (a - 1), a - 1 relative to itself; further below, an exponential of 2^-22 whose argument is rounded to FP32.  2^-22 + 2^-19 (1 - a) a step covers both, and also
a state that is carried over many tokens in one product instead.  Errors decay as h does.  Outputs are rounded once (`u`, `tiny`), and dlog_decay is taken from rounded outputs.
"""
import torch

from sequence_reference import half_step, tiny


def _walk(a, x, state):
    """h, its bound, and the state behind the last token with its own; rows are tokens"""
    h, mass, err = state, state.abs(), torch.zeros_like(state)
    hs, es = torch.empty_like(x), torch.empty_like(x)
    for t in range(x.shape[0]):
        h = a[t] * h + x[t]
        mass = a[t] * mass + x[t].abs()
        err = a[t] * err + (2.0 ** -22 + 2.0 ** -19 * (1 - a[t])) * mass
        hs[t], es[t] = h, err
    return hs, es, h, err


def recurrence(x, log_decay, lengths, state=None, dout=None, dfinal=None):
    u, w0 = (half_step(x.dtype), tiny(x.dtype)) if x.dtype != torch.float32 else (2.0 ** -24, 0.0)
    z = lambda *s: torch.zeros(2, *s, device=x.device, dtype=torch.float64)  # noqa: E731
    got = {"out": z(*x.shape), "final": z(len(lengths), x.shape[1])}
    if dout is not None:
        got |= {"dx": z(*x.shape), "dlog": z(*x.shape), "dstate": z(len(lengths), x.shape[1])}
    a_all, r0 = torch.exp(log_decay.double().clamp(max=0)), 0

    def note(name, at, val, err):
        got[name][0][at], got[name][1][at] = val, u * val.abs() + (1 + u) * err + w0

    for s, n in enumerate(lengths):
        at, S = slice(r0, r0 + n), state[s].double() if state is not None else torch.zeros(x.shape[1], device=x.device, dtype=torch.float64)
        a = a_all[at]
        hs, es, last, err = _walk(a, x[at].double(), S)
        note("out", at, hs, es)
        got["final"][0][s], got["final"][1][s] = last, err + 2.0 ** -24 * last.abs()
        if dout is not None:
            D = dfinal[s].double() if dfinal is not None else torch.zeros_like(S)
            nxt = torch.cat([a[1:], torch.ones_like(a[:1])]) if n else a       # what enters behind the last token is not decayed
            g, ge, _, _ = _walk(nxt.flip(0), dout[at].double().flip(0), D)
            g, ge = g.flip(0), ge.flip(0)
            note("dx", at, g, ge)
            before = torch.cat([S[None], hs[:-1]]) if n else hs
            off = torch.cat([torch.zeros_like(S)[None], u * hs[:-1].abs() + (1 + u) * es[:-1] + w0]) if n else hs
            on = (log_decay[at] <= 0).double()
            note("dlog", at, on * g * a * before, on * (a * (ge * before.abs() + g.abs() * off + ge * off) + 2.0 ** -20 * (g * a * before).abs()))
            d0, e0 = (a[0] * g[0], a[0] * ge[0]) if n else (D, torch.zeros_like(D))
            got["dstate"][0][s], got["dstate"][1][s] = d0, e0 + 2.0 ** -20 * d0.abs()
        r0 += n
    return {k: tuple(v) for k, v in got.items()}
