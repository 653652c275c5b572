"""The paged cache in 64 bits, written from its definitions, and how far a kernel's roundings may take it (as sequence_reference.py counts them)."""
import math

import torch

from sequence_reference import FLOOR, FP32, half_step, tiny


def tree(parents, n):
    """Depths of n new tokens, and for each the set of itself and those above it; parents None: one after the other"""
    depths, above = [], []
    for i in range(n):
        p = i - 1 if parents is None else int(parents[i])
        p = p if 0 <= p < i else -1
        depths.append(depths[p] + 1 if p >= 0 else 0)
        above.append((above[p] if p >= 0 else set()) | {i})
    return depths, above


def places(slots, table_row, page_tokens, pages):
    """(page, row) of each token of a sequence that has a place, and which have"""
    slots = torch.as_tensor(slots, dtype=torch.long)
    col = slots // page_tokens
    inside = col < len(table_row)
    page = torch.where(inside, table_row.long().cpu()[col.clamp(max=max(len(table_row) - 1, 0))] if len(table_row) else col * 0 - 1, col * 0 - 1)
    return page, slots % page_tokens, inside & (page >= 0) & (page < pages)


def attention(q, k_pages, v_pages, table, lengths, new, window=None, sinks=0, parents=None, scale=None):
    """(value, bound); lengths: tokens before the new ones, new: numbers of new tokens"""
    pages, page_tokens, kv, width = k_pages.shape
    u, w0, t = half_step(q.dtype), tiny(q.dtype) + FLOOR, width ** -0.5 if scale is None else scale
    group, w, cap = q.shape[1] // kv, 1 << 40 if window is None else window, table.shape[1] * page_tokens
    out, bound = torch.zeros(2, *q.shape, device=q.device, dtype=torch.float64)
    r0 = 0
    for b, (c, n) in enumerate(zip(lengths, new)):
        c = min(max(int(c), 0), cap)
        depths, above = tree(None if parents is None else parents[r0:r0 + n].tolist(), n)
        if n == 0:
            continue
        page, row, there = places(range(c + n), table[b], page_tokens, pages)
        pos = torch.tensor(list(range(c)) + [c + d for d in depths])
        apart = pos[c:, None] - pos[None]
        seen = (apart < w) | (pos < sinks)
        among = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            among[i, list(above[i])] = True
        seen[:, c:] &= among
        seen &= there
        used = seen.any(0)
        seen = seen[:, used].to(q.device)
        kd, vd = (x[page[used].to(q.device), row[used].to(q.device)].double() for x in (k_pages, v_pages))
        qd = q[r0:r0 + n].double()
        for h in range(q.shape[1]):
            kh, vh = kd[:, h // group], vd[:, h // group]
            x = (qd[:, h] @ kh.T * t).masked_fill(~seen, -math.inf)
            some = seen.any(1, keepdim=True)
            p = torch.where(some, torch.softmax(x, 1) if x.shape[1] else x, torch.zeros_like(x)).nan_to_num()
            fp32 = FP32 + 2.0 ** -22 * abs(t) * ((qd[:, h].abs() @ kh.abs().T).amax(1, keepdim=True) if x.shape[1] else 0.0)
            o, mass = p @ vh, p @ vh.abs()
            out[r0:r0 + n, h] = o
            bound[r0:r0 + n, h] = u * o.abs() + (u + fp32) * mass + w0 * (seen.double() @ vh.abs())
        r0 += n
    return out, bound


def rotate(x, pos, columns, frequencies, interleaved):
    """(value, bound) of rows x (tokens, heads, width) at positions pos"""
    y, u = x.double().clone(), half_step(x.dtype)
    half = columns // 2
    a, b = (slice(0, columns, 2), slice(1, columns, 2)) if interleaved else (slice(0, half), slice(half, columns))
    angle = pos.to(x.device).double()[:, None] * torch.tensor(frequencies, dtype=torch.float64, device=x.device)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    p, q = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = p * cos - q * sin, p * sin + q * cos
    mass = torch.zeros_like(y)
    mass[..., a] = mass[..., b] = p.abs() + q.abs()
    # an output's rounding; cosines and sines of FP32 (their own 2^-22, and a part of a turn rounded to 2^-25), two products and a sum
    return y, u * y.abs() + 2.0 ** -20 * mass + tiny(x.dtype)
