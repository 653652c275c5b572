"""The kernel products over sequences in 64 bits, written from their definitions, and how far a kernel's 16-bit roundings may take it.

Every function returns, for each output, (value, bound): the bound counts half a step of the type (`u`) for each rounding that the
kernels make -- of the outputs, of the weights that go into a matrix product, of the carried state as an operand -- times the sum of the
absolute values of what is rounded, and 1e-5 times that sum for arithmetic in FP32 (sums of a few thousand terms and an exponential
of 2^-22).  Numbers below FP32's smallest normal one, 2^-126, may be flushed or rounded to a multiple of 2^-149.  In fp16 a weight below 2^-14 is off by up to half of 2^-24 instead (`tiny`).  A weight
2^x with x below -125 may be taken as 2^-125 (where the exponential is a polynomial, its exponent stays in the normal range): FLOOR.
"""
import math

import torch

FP32 = 1e-5
FLOOR = 2.0 ** -125


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t == torch.float16 else 0.0


def split(x, lengths):
    return torch.split(x, list(lengths))


def seen(n, window, sinks, device):
    i, j = torch.arange(n, device=device)[:, None], torch.arange(n, device=device)[None, :]
    return (j <= i) & ((i - j < window) | (j < sinks))


def window(q, k, v, lengths, window, sinks, scale=None, dout=None):
    u, w0, t = half_step(q.dtype), tiny(q.dtype) + FLOOR, q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    names = ["out", "lse"] + (["dq", "dk", "dv"] if dout is not None else [])
    got = {n: ([], []) for n in names}
    for s, (qs, ks, vs) in enumerate(zip(split(q, lengths), split(k, lengths), split(v, lengths))):
        qd = qs.double().transpose(0, 1)
        kd, vd = (x.double().transpose(0, 1).repeat_interleave(group, 0) for x in (ks, vs))
        x = (qd @ kd.mT) * t
        m = seen(qs.shape[0], window, sinks, q.device).double()
        x = x.masked_fill(m == 0, -math.inf)
        lse = torch.logsumexp(x, -1) if x.shape[-1] else x.new_zeros(x.shape[:2])
        p = torch.exp(x - lse[..., None])
        # an exponent is an FP32 sum of products: a weight is off by that, relative to itself
        fp32 = FP32 + 2.0 ** -22 * abs(t) * (qd.abs() @ kd.abs().mT).amax(-1, keepdim=True) if x.shape[-1] else FP32
        o, mass = p @ vd, p @ vd.abs()
        # a weight's error against the row's largest, of which the row sum is at least one
        got["out"][0].append(o.transpose(0, 1))
        got["out"][1].append((u * o.abs() + (u + fp32) * mass + w0 * (m @ vd.abs())).transpose(0, 1))
        got["lse"][0].append(lse)
        got["lse"][1].append(FP32 * (1 + lse.abs() + (qd.abs() @ kd.abs().mT).amax(-1) * abs(t) if x.shape[-1] else lse))
        if dout is None:
            continue
        g = split(dout, lengths)[s].double().transpose(0, 1)
        dp, delta = g @ vd.mT, (g * o).sum(-1, keepdim=True)
        ds = p * (dp - delta) * t
        # delta is taken from the rounded out; dp and delta are FP32 sums
        slack = p * abs(t) * (u * (g.abs() * (o.abs() + mass)).sum(-1, keepdim=True) + FP32 * (g.abs() @ vd.abs().mT + (g * o).abs().sum(-1, keepdim=True)))
        e = (u + fp32) * ds.abs() + slack + w0 * m
        ep = (u + fp32) * p + w0 * m
        shared = lambda y: y.reshape(k.shape[1], group, *y.shape[1:]).sum(1)  # noqa: E731
        for name, val, err in (("dq", ds @ kd, e @ kd.abs()), ("dk", shared(ds.mT @ qd), shared(e.mT @ qd.abs())),
                               ("dv", shared(p.mT @ g), shared(ep.mT @ g.abs()))):
            got[name][0].append(val.transpose(0, 1))
            got[name][1].append((u * val.abs() + err + tiny(q.dtype)).transpose(0, 1))
    return {n: tuple(torch.cat(z, 1 if n == "lse" else 0) for z in got[n]) for n in names}


def window_step(q, kc, vc, lengths, window, sinks, scale=None):
    u, w0, t = half_step(q.dtype), tiny(q.dtype), q.shape[2] ** -0.5 if scale is None else scale
    group, cap = q.shape[1] // kc.shape[2], kc.shape[1]
    out, bound = torch.zeros(2, *q.shape, device=q.device, dtype=torch.float64)
    for b, n in enumerate(lengths):
        n = min(max(n, 0), cap)
        j = torch.arange(n, device=q.device)
        j = j[(n - 1 - j < window) | (j < sinks)]
        if n == 0:
            continue
        kd, vd = (x[b, j].double().repeat_interleave(group, 1) for x in (kc, vc))
        p = torch.softmax(torch.einsum("hd,khd->hk", q[b].double(), kd) * t, 1)
        fp32 = FP32 + 2.0 ** -22 * abs(t) * torch.einsum("hd,khd->hk", q[b].double().abs(), kd.abs()).amax(1)[:, None]
        out[b], mass = torch.einsum("hk,khd->hd", p, vd), torch.einsum("hk,khd->hd", p, vd.abs())
        bound[b] = u * out[b].abs() + (u + fp32) * mass + w0 * vd.abs().sum(0)
    return out, bound


def _run(a, b, c, decay, start, use, upd, undecayed):
    """One head's product on one sequence, a (n, wb), b (n, wb), c (n, wc), start (wb, wc): outputs, the last state, and the sums of
    absolute values that bound their roundings."""
    n = a.shape[0]
    i = torch.arange(n, device=a.device, dtype=torch.float64)
    apart = i[:, None] - i[None, :]
    L = (decay ** apart.clamp(min=0)).tril()
    steps = decay ** (i + (0 if undecayed else 1))
    x = L * (a @ b.T) * use * upd
    o = x @ c + steps[:, None] * (a @ start) * use
    # the state is carried as sums of absolute values too: it is rounded where it becomes an operand
    mass = ((L * (a.abs() @ b.abs().T)) @ c.abs() * abs(use * upd)) + steps[:, None] * (a.abs() @ start.abs()) * abs(use)
    left = decay ** (n - 1 - i + (1 if undecayed else 0))
    last = (left[:, None] * b).T @ c * upd + decay ** n * start
    last_mass = (left[:, None] * b.abs()).T @ c.abs() * abs(upd) + decay ** n * start.abs()
    return o, mass, last, last_mass, (left[:, None] * b.abs()).sum(0)[:, None] + c.abs().sum(0)[None]


def decay(q, k, v, log_decay, lengths, state=None, scale=None, dout=None, dfinal=None):
    u, w0, t = half_step(q.dtype), tiny(q.dtype), q.shape[2] ** -0.5 if scale is None else scale
    heads, wk, wv = q.shape[1], q.shape[2], v.shape[2]
    total = q.shape[0]
    z = lambda *s: torch.zeros(2, *s, device=q.device, dtype=torch.float64)  # noqa: E731
    got = {"out": z(total, heads, wv), "final": z(len(lengths), heads, wk, wv)}
    if dout is not None:
        got |= {"dq": z(total, heads, wk), "dk": z(total, heads, wk), "dv": z(total, heads, wv), "dstate": z(len(lengths), heads, wk, wv)}
    r0 = 0

    def note(name, at, val, mass):
        # the outputs, the weights of a tile and the carried state are rounded; weights below the type's smallest are off by `tiny` each
        got[name][0][at] = val
        got[name][1][at] = u * val.abs() + (2 * u + FP32) * mass + w0 * 1000

    def note_state(name, at, val, mass, ones):
        # an operand is split into a head and a tail: what is lost is half a step of half a step
        got[name][0][at] = val
        got[name][1][at] = (u * u + FP32) * mass + w0 * ones

    for s, n in enumerate(lengths):
        rows = slice(r0, r0 + n)
        for h in range(heads):
            qd, kd, vd = (x[rows, h].double() for x in (q, k, v))
            g = min(1.0, math.exp(min(0.0, float(log_decay[h]))))
            S = state[s, h].double() if state is not None else torch.zeros(wk, wv, device=q.device, dtype=torch.float64)
            o, m, last, lm, ones = _run(qd, kd, vd, g, S, t, 1.0, False)
            note("out", (rows, h), o, m)
            note_state("final", (s, h), last, lm, ones)
            if dout is None:
                continue
            D = dfinal[s, h].double() if dfinal is not None else torch.zeros_like(S)
            gd = dout[rows, h].double()
            o, m, *_ = _run(gd, vd, kd, g, S.T, t, 1.0, False)
            note("dq", (rows, h), o, m)
            o, m, *_ = _run(vd.flip(0), gd.flip(0), qd.flip(0), g, D.T, 1.0, t, True)
            note("dk", (rows, h), o.flip(0), m.flip(0))
            o, m, last, lm, ones = _run(kd.flip(0), qd.flip(0), gd.flip(0), g, D, 1.0, t, True)
            note("dv", (rows, h), o.flip(0), m.flip(0))
            note_state("dstate", (s, h), last, lm, ones)
        r0 += n
    return {n: tuple(x) for n, x in got.items()}


def assert_within(got, want, what=""):
    value, bound = want
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = (got.double() - value).abs()
    bad = ~(off <= bound + 2.0 ** -126)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / bound.clamp(min=1e-30)).max()):.3g} of the bound"
