"""A cache of keys and values in pages: new tokens appended, rotated on the way, their attention over it, accepted paths of drafted trees.

The products are those of `sequence.window_attention`; what is different is where the keys lie and which ones a new token sees.  Definitions, limits and what is asked
of the arrays stand in include/f3m.h.

    k_pages, v_pages                                   # (pages, page_tokens, kv_heads, width), bf16 or fp16: the program's own, written in place
    page_table                                         # (n, most) int32: the pages of each sequence, in order
    lengths                                            # (n) int32: tokens in the cache, without the new ones
    plan = SequencePlan([9, 1, 33])                    # new tokens of each sequence: one, a chunk of a prompt, or a tree of drafted ones
    rotation = Rotation(width)

    q = paged_append(plan, k, v, k_pages, v_pages, page_table, lengths, rotation, parents, q=q)
    out = paged_attention(plan, q, k_pages, v_pages, page_table, lengths, window=None, sinks=0, parents=parents)
    paged_keep(k_pages, v_pages, page_table, lengths, kept, counts)      # after a tree was looked at: its accepted path moves to the front
    lengths += counts

New tokens are packed, as in `sequence`: row t of q, k, v is token t of all sequences laid end to end.  Token i of a sequence is token lengths + i of its cache.  Without
`parents` new tokens follow one another; `parents` (tokens) int32 makes them a tree: the number, among the sequence's new tokens, of the token before each one, -1 where
that is the cache's last.  A new token sees the cache, itself and those above it; its position is the cache's length plus its depth.  The tokens of a cache that is one array
(n, capacity, kv_heads, width) are pages too: `cache.view(n * capacity // 128, 128, kv_heads, width)`.  For one new token of each sequence over such an array `sequence.window_attention_step`
needs no plan and no table; `paged_attention` shares long caches more evenly (32 sequences up to 16384, 32 heads on 8, width 128: 177 us, 235).

A plan holds the numbers of new tokens.  Making one copies a table from host memory and waits for that: a program whose numbers change from step to step keeps a plan for each that comes
up -- one new token for n sequences, drafts of one size (a draft that came out shorter may be filled up: what is appended behind a sequence's kept tokens is written over by the next call).

No call with a plan in hand waits for the GPU: lengths, tables, parents and paths are read there, and all that they say is held within the arrays.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import Cache, Pages, RotationTable, Rows, check
from .sequence import SequencePlan, _check_plan, _check_width, _needs_grad, _new, _On, _pointer, _read, _refuse_tangents, _type_of, _window_numbers

_NO_ROWS = Rows(None, 0, 0)


class Rotation:
    """Turns of the first `columns` columns, a multiple of 16, by position: pair i by base^(-2 i / columns) radians a position, or by frequencies[i] where these
    are given.  Pair i is columns (i, i + columns / 2), or (2 i, 2 i + 1) if interleaved.  Kept for any number of calls on any stream of the device (as long as any graph that holds one of them)."""

    def __init__(self, columns: int, base: float = 10000.0, interleaved: bool = False, frequencies: Optional[Sequence[float]] = None, device="cuda:0"):
        if columns < 16 or columns > _lib.MAX_WIDTH or columns % 16:
            raise ValueError(f"{columns} columns: not a multiple of 16 in 16..{_lib.MAX_WIDTH}")
        if frequencies is None:
            if not (base > 0 and math.isfinite(base)):
                raise ValueError(f"base {base}")
            frequencies = [base ** (-2 * i / columns) for i in range(columns // 2)]
        frequencies = [float(f) for f in frequencies]
        if len(frequencies) != columns // 2 or not all(math.isfinite(f) for f in frequencies):
            raise ValueError(f"{columns // 2} finite frequencies are needed")
        self.columns, self.interleaved = int(columns), bool(interleaved)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("Rotation needs a CUDA device: the engine has no CPU path")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        # turns a position, modulo one, in 2^-64: an integer product by the position is exact
        words = [round(math.fmod(f / (2 * math.pi), 1.0) * 2 ** 64) % 2 ** 64 for f in frequencies]
        self.turns = torch.tensor([w - 2 ** 64 if w >= 2 ** 63 else w for w in words], dtype=torch.int64).to(self.device)    # blocks: it has ended
        self._home = torch.cuda.current_stream(self.device).cuda_stream
        self._table = RotationTable(self.turns.data_ptr(), self.columns, int(self.interleaved))
        self._ref = C.byref(self._table)


def _pages(t: torch.Tensor, shape, what: str) -> Pages:
    (ps, ts, hs, cs), (pages, _, heads, width), at = t.stride(), shape, t.data_ptr()
    if pages < 2:
        if pages == 0:
            return Pages(None, 0, 0, 0)
        ps = 0
    if heads == 1:
        hs = 0
    if cs != 1 or (at | 2 * (ps | ts | hs)) & 15 or ts < width or (hs < width and heads > 1) or (ps < width and pages > 1):
        raise ValueError(f"{what} is used in place: contiguous columns, strides multiples of 8 elements, data on 16 bytes")
    return Pages(at, ps, ts, hs)


def _numbers(t: torch.Tensor, shape, device, what: str) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.shape != shape or t.device != device:
        raise TypeError(f"{what} must be an int32 array {tuple(shape)} on {device}")
    return t


def _cache(k_pages, v_pages, page_table, lengths):
    """The library's view of a cache, and the arrays that it points to."""
    shape, device = k_pages.shape, k_pages.device
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} are (pages, page_tokens, kv_heads, width) arrays")
    pages, page_tokens, kv_heads, width = shape
    _check_width(width)
    if page_tokens < 8 or page_tokens & (page_tokens - 1):
        raise ValueError(f"pages of {page_tokens} tokens: not a power of two from 8 on")
    if kv_heads < 1:
        raise ValueError("a cache without key heads")
    if page_table.dim() != 2:
        raise ValueError("page_table is a (sequences, most) array")
    n, most = sizes = page_table.shape
    _numbers(page_table, sizes, device, "page_table")
    step, one = page_table.stride()
    if one != 1 and most > 1:
        page_table = page_table.contiguous()
        step = most
    lengths = _numbers(lengths, sizes[:1], device, "lengths").contiguous()
    c = Cache(_pages(k_pages, shape, "k_pages"), _pages(v_pages, shape, "v_pages"), pages, page_tokens, kv_heads, width, page_table.data_ptr(), step if n > 1 else most, most, n,
              lengths.data_ptr())
    return c, (page_table, lengths)


def _check_new(plan, c, first, parents):
    _check_plan(plan, first)
    if plan.sequences != c.sequences:
        raise ValueError(f"a plan of {plan.sequences} sequences, a cache of {c.sequences}")
    if parents is None:
        return None
    if plan.longest > _lib.TREE_MAX:
        raise ValueError(f"a tree of {plan.longest} tokens: at most {_lib.TREE_MAX}")
    return _numbers(parents, (plan.tokens,), first.device, "parents").contiguous()


def _check_rows(t, c, what, heads=None):
    if t.dim() != 3 or t.shape[2] != c.width or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{what} {tuple(t.shape)} does not match pages of {c.kv_heads} heads, width {c.width}")


def _written(*tensors):
    for t in tensors:
        torch.autograd.graph.increment_version(t)


def _no_gradient(what, *tensors):
    if _needs_grad(*tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")


def paged_append(plan: SequencePlan, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 lengths: torch.Tensor, rotation: Optional[Rotation] = None, parents: Optional[torch.Tensor] = None,
                 q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the new tokens' keys, rotated by their positions, and values (tokens, kv_heads, width) to their pages, in place.  Returns q (tokens, heads, width)
    rotated likewise, as a new array, or None without one.  Tokens whose page is missing, or lies behind the table, are not written; no two may have one place."""
    _refuse_tangents(k, v, k_pages, v_pages, q)
    kind = _type_of(k, v, k_pages, v_pages, *(() if q is None else (q,)))
    c, held = _cache(k_pages, v_pages, page_table, lengths)
    _check_rows(k, c, "k", c.kv_heads)
    if v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if q is not None:
        _check_rows(q, c, "q")
        if q.shape[0] != k.shape[0] or q.shape[1] < 1:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} do not match")
    parents = _check_new(plan, c, k, parents)
    if rotation is not None:
        if rotation.columns > c.width:
            raise ValueError(f"{rotation.columns} columns are rotated, the width is {c.width}")
        if rotation.device != k.device:
            raise ValueError(f"the rotation lies on {rotation.device}, the arrays on {k.device}")
    _no_gradient("paged_append", k, v, k_pages, v_pages, q)
    (k, rk), (v, rv) = _read(k), _read(v)
    heads, rq, out, ro = 0, _NO_ROWS, None, _NO_ROWS
    if q is not None:
        heads = q.shape[1]
        (q, rq), (out, ro) = _read(q), _new(q)
    with _On(k.device, plan) as stream:
        if rotation is not None and stream != rotation._home and not torch.cuda.is_current_stream_capturing():
            rotation.turns.record_stream(torch.cuda.current_stream(k.device))
        st = _lib.lib().f3m_paged_append(plan._ref, kind, C.byref(c), rk, rv, _pointer(parents), None if rotation is None else rotation._ref, heads, rq, ro, stream)
    check(st, "f3m_paged_append")
    _written(k_pages, v_pages)
    return out


def paged_attention(plan: SequencePlan, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                    window: Optional[int] = None, sinks: int = 0, parents: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of new tokens that the pages hold already (`paged_append`).  One at position p sees cached token j if p - j < window or j < sinks, and of itself and the new tokens
    above it, at positions p', those with p - p' < window or p' < sinks; window None is all.  q (tokens, heads, width), heads a multiple of the pages' kv_heads, at
    most 128 times; scale is 1/sqrt(width) unless given.  Returns out like q; a row that sees nothing, because its pages are missing, is zeros."""
    _refuse_tangents(q, k_pages, v_pages)
    kind = _type_of(q, k_pages, v_pages)
    c, held = _cache(k_pages, v_pages, page_table, lengths)
    _check_rows(q, c, "q")
    heads = q.shape[1]
    if heads < 1 or heads % c.kv_heads or heads // c.kv_heads > 128:
        raise ValueError(f"{heads} heads do not share {c.kv_heads} key heads evenly, at most 128 to one")
    parents = _check_new(plan, c, q, parents)
    _no_gradient("paged_attention", q, k_pages, v_pages)
    window, sinks, scale = _window_numbers(c.width, 0x7fffffff if window is None else window, sinks, scale)
    (q, rq), (out, ro) = _read(q), _new(q)
    L, ref = _lib.lib(), C.byref(c)
    need = L.f3m_paged_attention_workspace_bytes(plan._ref, ref, heads)
    ws = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
    with _On(q.device, plan) as stream:
        st = L.f3m_paged_attention(plan._ref, kind, ref, heads, window, sinks, scale, _pointer(parents), rq, ro, _pointer(ws), need, stream)
    check(st, "f3m_paged_attention")
    return out


def paged_keep(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, kept: torch.Tensor, counts: torch.Tensor) -> None:
    """Keeps a path of each tree: new token kept[b, j] of sequence b becomes token lengths[b] + j of the cache, for j < counts[b], in place.  kept (n, most), counts (n) int32;
    kept[b, j] >= j, as along any path from a root, others leave the place as it is.  `lengths` is the program's to move on: lengths += counts."""
    _refuse_tangents(k_pages, v_pages)
    kind = _type_of(k_pages, v_pages)
    c, held = _cache(k_pages, v_pages, page_table, lengths)
    if kept.dim() != 2:
        raise ValueError("kept is a (sequences, most) array")
    kept = _numbers(kept, (c.sequences, kept.shape[1]), k_pages.device, "kept").contiguous()
    counts = _numbers(counts, (c.sequences,), k_pages.device, "counts").contiguous()
    _no_gradient("paged_keep", k_pages, v_pages)
    with _On(k_pages.device) as stream:
        st = _lib.lib().f3m_paged_keep(kind, C.byref(c), kept.data_ptr(), kept.shape[1], kept.shape[1], counts.data_ptr(), stream)
    check(st, "f3m_paged_keep")
    _written(k_pages, v_pages)
