"""Kernel products over sequences: attention over a window with sinks, and linear attention with a decay for each head.

They are the engine's two products on a line of positions: `window_attention` sums every pair that is seen (as `engine.rbf_dense`
does, rows normalised), `decay_attention` sums near pairs one by one and far ones through moments (as `FFM` does, here exactly).
Definitions, limits and what is asked of the arrays stand in include/f3m.h.

    plan = SequencePlan([1021, 1, 4096])                     # lengths of the packed sequences; kept for any number of calls
    out, lse = window_attention(plan, q, k, v, window=1024, sinks=4)
    dq, dk, dv = window_attention_grad(plan, q, k, v, out, lse, dout, window=1024, sinks=4)
    out = window_attention_step(q, k_cache, v_cache, lengths, window=1024, sinks=4)     # one new token of each sequence

    out, state = decay_attention(plan, q, k, v, log_decay)
    dq, dk, dv, dstate = decay_attention_grad(plan, q, k, v, log_decay, dout)
    out = decay_attention_step(q, k, v, log_decay, state)                               # state updated in place

Prompts and training take packed arrays (tokens, heads, width), bf16 or fp16; a batch (n, tokens, heads, width) of equal lengths is
`x.flatten(0, 1)` with `SequencePlan([tokens] * n)`.  Columns have to be contiguous, token and head strides multiples of 8 elements
and data on 16 bytes -- views of a joint projection are; anything else is copied.  No call waits for the GPU.

`window_attention` and `decay_attention` are differentiable by q, k, v (and the states) when autograd is on.  Autograd's bookkeeping of a
leaf belongs to the stream that first used it, so a graph that is differentiated by autograd is not captured: the two refuse that, and a
captured training step calls the gradient functions itself.  Forward-mode derivatives are refused.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import Rows, Seqs, check

_TYPES = {torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
_NO_ROWS = Rows(None, 0, 0)


class SequencePlan:
    """Where the sequences of a packed batch lie (f3m_seqs_layout): made from their lengths, a list of whole numbers or a CPU
    tensor, and kept for any number of products on any stream of the device (as long as any graph that holds one of them)."""

    def __init__(self, lengths: Sequence[int], device="cuda:0"):
        host = np.ascontiguousarray(lengths.cpu().numpy() if torch.is_tensor(lengths) else lengths)
        if host.size == 0:
            host = host.reshape(0).astype(np.int64)
        if host.ndim != 1 or host.dtype.kind not in "iu":
            raise ValueError("lengths must be a list of whole numbers")
        if host.size and (host.min() < 0 or host.max() > 0x7fffffff):
            raise ValueError("lengths must lie between 0 and 2^31 - 1")
        host = host.astype(np.int32)
        self.lengths = tuple(int(n) for n in host)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("SequencePlan needs a CUDA device: the engine has no CPU path")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._seqs = Seqs()
        L = _lib.lib()
        check(L.f3m_seqs_layout(host.ctypes.data, host.size, C.byref(self._seqs), None), "f3m_seqs_layout")
        table = np.zeros(max(4, self._seqs.table_words), dtype=np.int32)
        check(L.f3m_seqs_layout(host.ctypes.data, host.size, C.byref(self._seqs), table.ctypes.data), "f3m_seqs_layout")
        self.table = torch.from_numpy(table).to(self.device)      # a copy that blocks: it has ended when this returns
        self._home = torch.cuda.current_stream(self.device).cuda_stream
        self._seqs.table = self.table.data_ptr()
        self._ref = C.byref(self._seqs)
        self.tokens, self.sequences, self.longest = int(self._seqs.tokens), int(self._seqs.sequences), int(self._seqs.longest)


class _On:
    """The device of the arrays made current for a call, where it is not already, and its current stream.  A plan's table belongs to the stream
    that it was made on: another one's use of it is noted, so that its memory is not handed on before that has ended."""
    __slots__ = ("index", "guard", "plan")

    def __init__(self, device, plan=None):
        self.index, self.guard, self.plan = device.index, None, plan

    def __enter__(self) -> int:
        if torch.cuda.current_device() != self.index:
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        stream = torch._C._cuda_getCurrentRawStream(self.index)
        if self.plan is not None and stream != self.plan._home and not torch.cuda.is_current_stream_capturing():
            self.plan.table.record_stream(torch.cuda.current_stream(self.index))
        return stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _read(t: torch.Tensor) -> Tuple[torch.Tensor, Rows]:
    """t (tokens, heads, width), or a dense copy of it where the library could not read it in place, and the library's view of that."""
    (ts, hs, cs), (tokens, heads, width), at = t.stride(), t.shape, t.data_ptr()
    if tokens == 1:
        ts = heads * width
    if heads == 1:
        hs = width
    if cs != 1 or (at | 2 * ts | 2 * hs) & 15 or ts < width or hs < width:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        at, ts, hs = t.data_ptr(), heads * width, width
    return t, Rows(at, ts, hs)


def _cache(t: torch.Tensor, what: str) -> Tuple[Rows, int]:
    """The library's view of a cache (n, capacity, heads, width), which is read in place, and the stride of its sequences."""
    (ss, ts, hs, cs), (n, tokens, heads, width), at = t.stride(), t.shape, t.data_ptr()
    if t.numel() == 0:
        return _NO_ROWS, 0
    if n == 1:
        ss = 0
    if tokens == 1:
        ts = heads * width
    if heads == 1:
        hs = width
    if cs != 1 or (at | 2 * ss | 2 * ts | 2 * hs) & 15 or ts < width or hs < width or (n > 1 and ss < width):
        raise ValueError(f"{what} is read in place: contiguous columns, strides multiples of 8 elements, data on 16 bytes")
    return Rows(at, ts, hs), ss


def _new(t: torch.Tensor) -> Tuple[torch.Tensor, Rows]:
    """A dense array like t and the library's view of it."""
    y = torch.empty_like(t, memory_format=torch.contiguous_format)
    _, heads, width = y.shape
    return y, Rows(y.data_ptr(), heads * width, width)


def _type_of(q: torch.Tensor, *others: torch.Tensor) -> int:
    if not q.is_cuda:
        raise ValueError("the engine has no CPU path: q must be a CUDA tensor")
    if q.dtype not in _TYPES:
        raise TypeError(f"{q.dtype}: only torch.bfloat16 and torch.float16 are built")
    for t in others:
        if t.dtype != q.dtype:
            raise TypeError(f"arrays of {q.dtype} and {t.dtype} in one call")
        if t.device != q.device:
            raise ValueError(f"arrays on {q.device} and {t.device} in one call")
    return _TYPES[q.dtype]


def _check_width(*widths: int):
    for w in widths:
        if w < 8 or w > _lib.MAX_WIDTH or w % 8:
            raise ValueError(f"width {w} is not a multiple of 8 in 8..{_lib.MAX_WIDTH}")


def _check_plan(plan: SequencePlan, q: torch.Tensor):
    if q.device != plan.device:
        raise ValueError(f"the plan lies on {plan.device}, the arrays on {q.device}")
    if q.shape[0] != plan.tokens:
        raise ValueError(f"arrays of {q.shape[0]} tokens, a plan of {plan.tokens}")


def _shape(t: torch.Tensor, shape, what: str):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, not {tuple(shape)}")


def _window_numbers(width: int, window: int, sinks: int, scale: Optional[float]) -> Tuple[int, int, float]:
    if window < 1 or sinks < 0:
        raise ValueError(f"window {window}, sinks {sinks}: at least one key has to be seen")
    return min(int(window), 0x7fffffff), min(int(sinks), 0x7fffffff), width ** -0.5 if scale is None else float(scale)


def _refuse_capture(what: str):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} is differentiated by autograd while a graph is captured: call {what}_grad there, on tensors "
                           "that need no gradient")


def _refuse_tangents(*tensors):
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the products over sequences have no forward-mode derivatives")


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---------------------------------------------------------------------------------------------------------------------
# window attention
# ---------------------------------------------------------------------------------------------------------------------
def _check_qkv(plan, q, k, v):
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3:
        raise ValueError("q, k, v are (tokens, heads, width) arrays")
    _check_plan(plan, q)
    _check_width(qs[2])
    if ks[0] != qs[0] or ks[2] != qs[2] or v.shape != ks:
        raise ValueError(f"q {tuple(qs)}, k {tuple(ks)} and v {tuple(v.shape)} do not match")
    if ks[1] < 1 or qs[1] % ks[1]:
        raise ValueError(f"{qs[1]} heads do not share {ks[1]} key heads evenly")


def window_attention(plan: SequencePlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
                     scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Token i of a sequence sees token j <= i if i - j < window or j < sinks: out_i = sum_j w_ij v_j / sum_j w_ij, w_ij = exp(scale q_i.k_j).
    q (tokens, heads, width), k and v (tokens, kv_heads, width) with heads a multiple of kv_heads; scale is 1/sqrt(width) unless given.
    Returns out like q and lse (heads, tokens) float32, the logs of the row sums."""
    _refuse_tangents(q, k, v)
    if _needs_grad(q, k, v):
        _refuse_capture("window_attention")
        return _WindowAttention.apply(plan, q, k, v, window, sinks, scale)
    return _window_forward(plan, q, k, v, window, sinks, scale)


def _window_forward(plan, q, k, v, window, sinks, scale):
    kind = _type_of(q, k, v)
    _check_qkv(plan, q, k, v)
    window, sinks, scale = _window_numbers(q.shape[2], window, sinks, scale)
    tokens, heads, width = q.shape
    (q, rq), (k, rk), (v, rv), (out, ro) = _read(q), _read(k), _read(v), _new(q)
    lse = torch.empty((heads, tokens), device=q.device, dtype=torch.float32)
    with _On(q.device, plan) as stream:
        st = _lib.lib().f3m_window_attention(plan._ref, kind, heads, k.shape[1], width, window, sinks, scale, rq, rk, rv, ro, lse.data_ptr(), stream)
    check(st, "f3m_window_attention")
    return out, lse


def window_attention_grad(plan: SequencePlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                          dout: torch.Tensor, window: int, sinks: int = 0, scale: Optional[float] = None
                          ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of sum(out * dout), from what window_attention returned for the same arguments."""
    _refuse_tangents(q, k, v, out, lse, dout)
    kind = _type_of(q, k, v, out, dout)
    _check_qkv(plan, q, k, v)
    _shape(out, q.shape, "out")
    _shape(dout, q.shape, "dout")
    _shape(lse, (q.shape[1], q.shape[0]), "lse")
    if lse.dtype != torch.float32 or lse.device != q.device:
        raise TypeError("lse must be the float32 array that window_attention returned")
    window, sinks, scale = _window_numbers(q.shape[2], window, sinks, scale)
    heads, lse = q.shape[1], lse.contiguous()
    (q, rq), (k, rk), (v, rv), (out, ro), (dout, rg) = _read(q), _read(k), _read(v), _read(out), _read(dout)
    (dq, wq), (dk, wk), (dv, wv) = _new(q), _new(k), _new(v)
    L = _lib.lib()
    need = L.f3m_window_attention_grad_workspace_bytes(plan._ref, heads, k.shape[1], q.shape[2], window, sinks)
    ws = torch.empty(need, device=q.device, dtype=torch.uint8)
    with _On(q.device, plan) as stream:
        st = L.f3m_window_attention_grad(plan._ref, kind, heads, k.shape[1], q.shape[2], window, sinks, scale, rq, rk, rv, ro, lse.data_ptr(), rg,
                                         wq, wk, wv, ws.data_ptr(), need, stream)
    check(st, "f3m_window_attention_grad")
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, q, k, v, window, sinks, scale):
        out, lse = _window_forward(plan, q, k, v, window, sinks, scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.rest = (plan, window, sinks, scale)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        _refuse_capture("window_attention")
        q, k, v, out, lse = ctx.saved_tensors
        plan, window, sinks, scale = ctx.rest
        return (None,) + window_attention_grad(plan, q, k, v, out, lse, dout, window, sinks, scale) + (None,) * 3


def window_attention_step(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, window: int, sinks: int = 0,
                          scale: Optional[float] = None) -> torch.Tensor:
    """One new token for each of n sequences, 65535 at most.  q (n, heads, width); k_cache, v_cache (n, capacity, kv_heads, width) hold the tokens so far,
    the new one at lengths - 1 among them; lengths (n) int32 on the device, taken as 0..capacity.  Returns out like q; a sequence of length
    0 gets zeros."""
    _refuse_tangents(q, k_cache, v_cache)
    kind = _type_of(q, k_cache, v_cache)
    if q.dim() != 3 or k_cache.dim() != 4:
        raise ValueError("q is a (n, heads, width) array, k_cache and v_cache are (n, capacity, kv_heads, width) arrays")
    n, heads, width = q.shape
    _check_width(width)
    _shape(k_cache, (n, k_cache.shape[1], k_cache.shape[2], width), "k_cache")
    _shape(v_cache, k_cache.shape, "v_cache")
    capacity, kv_heads = k_cache.shape[1], k_cache.shape[2]
    if kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads do not share {kv_heads} key heads evenly")
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (n,) or lengths.device != q.device:
        raise TypeError("lengths must be an int32 array (n) on the device of q")
    if _needs_grad(q, k_cache, v_cache):
        raise RuntimeError("window_attention_step has no gradient: call it under torch.no_grad()")
    window, sinks, scale = _window_numbers(width, window, sinks, scale)
    lengths = lengths.contiguous()
    (q, rq), (out, ro), (rk, sk), (rv, sv) = _read(q), _new(q), _cache(k_cache, "k_cache"), _cache(v_cache, "v_cache")
    L = _lib.lib()
    need = L.f3m_window_attention_step_workspace_bytes(n, heads, kv_heads, width, capacity, window, sinks)
    ws = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
    with _On(q.device) as stream:
        st = L.f3m_window_attention_step(n, kind, heads, kv_heads, width, capacity, window, sinks, scale, rq, rk, sk, rv, sv, lengths.data_ptr(), ro,
                                         _pointer(ws), need, stream)
    check(st, "f3m_window_attention_step")
    return out


# ---------------------------------------------------------------------------------------------------------------------
# attention with a decay
# ---------------------------------------------------------------------------------------------------------------------
def _check_decay(q, k, v, log_decay):
    if q.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k, v are (tokens, heads, width) arrays")
    _check_width(q.shape[2], v.shape[2])
    _shape(k, q.shape, "k")
    _shape(v, (q.shape[0], q.shape[1], v.shape[2]), "v")
    _shape(log_decay, (q.shape[1],), "log_decay")
    if log_decay.dtype != torch.float32 or log_decay.device != q.device:
        raise TypeError("log_decay must be a float32 array (heads) on the device of q")


def _check_state(t, n, q, v, what):
    if t is None:
        return None
    _shape(t, (n, q.shape[1], q.shape[2], v.shape[2]), what)
    if t.dtype != torch.float32 or t.device != q.device:
        raise TypeError(f"{what} must be a float32 array on the device of q")
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _pointer(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


def decay_attention(plan: SequencePlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                    state: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """S_t = exp(log_decay) S_(t-1) + k_t v_t^T, out_t = scale q_t S_t along every sequence.  q, k (tokens, heads, width_k), v (tokens, heads,
    width_v), log_decay (heads) float32, at most 0; state (sequences, heads, width_k, width_v) float32 is the state before the first token
    (zeros unless given); scale is 1/sqrt(width_k) unless given.  Returns out like v and the state behind the last token, as a new array."""
    _refuse_tangents(q, k, v, log_decay, state)
    if _needs_grad(q, k, v, log_decay, state):
        if log_decay.requires_grad:
            raise RuntimeError("decay_attention has no gradient by log_decay: the decay is a constant")
        _refuse_capture("decay_attention")
        return _DecayAttention.apply(plan, q, k, v, log_decay, state, scale)
    return _decay_forward(plan, q, k, v, log_decay, state, scale)


def _decay_workspace(plan, q, v):
    need = _lib.lib().f3m_decay_attention_workspace_bytes(plan._ref, q.shape[1], q.shape[2], v.shape[2])
    return need, (torch.empty(need, device=q.device, dtype=torch.uint8) if need else None)


def _decay_forward(plan, q, k, v, log_decay, state, scale):
    kind = _type_of(q, k, v)
    _check_decay(q, k, v, log_decay)
    _check_plan(plan, q)
    state = _check_state(state, plan.sequences, q, v, "state")
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    log_decay, heads = log_decay.contiguous(), q.shape[1]
    (q, rq), (k, rk), (v, rv), (out, ro) = _read(q), _read(k), _read(v), _new(v)
    final = torch.empty((plan.sequences, heads, q.shape[2], v.shape[2]), device=q.device, dtype=torch.float32)
    need, ws = _decay_workspace(plan, q, v)
    with _On(q.device, plan) as stream:
        st = _lib.lib().f3m_decay_attention(plan._ref, kind, heads, q.shape[2], v.shape[2], log_decay.data_ptr(), scale, rq, rk, rv, _pointer(state), ro,
                                            final.data_ptr(), _pointer(ws), need, stream)
    check(st, "f3m_decay_attention")
    return out, final


def decay_attention_grad(plan: SequencePlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, dout: torch.Tensor,
                         state: Optional[torch.Tensor] = None, dfinal: Optional[torch.Tensor] = None, scale: Optional[float] = None
                         ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv, dstate) of sum(out * dout) + sum(final * dfinal) for (out, final) = decay_attention(plan, q, k, v, log_decay,
    state, scale); dfinal is zero unless given."""
    _refuse_tangents(q, k, v, log_decay, dout, state, dfinal)
    kind = _type_of(q, k, v, dout)
    _check_decay(q, k, v, log_decay)
    _check_plan(plan, q)
    _shape(dout, v.shape, "dout")
    state = _check_state(state, plan.sequences, q, v, "state")
    dfinal = _check_state(dfinal, plan.sequences, q, v, "dfinal")
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    log_decay, heads = log_decay.contiguous(), q.shape[1]
    (q, rq), (k, rk), (v, rv), (dout, rg) = _read(q), _read(k), _read(v), _read(dout)
    (dq, wq), (dk, wk), (dv, wv) = _new(q), _new(k), _new(v)
    dstate = torch.empty((plan.sequences, heads, q.shape[2], v.shape[2]), device=q.device, dtype=torch.float32)
    need, ws = _decay_workspace(plan, q, v)
    with _On(q.device, plan) as stream:
        st = _lib.lib().f3m_decay_attention_grad(plan._ref, kind, heads, q.shape[2], v.shape[2], log_decay.data_ptr(), scale, rq, rk, rv, _pointer(state),
                                                 rg, _pointer(dfinal), wq, wk, wv, dstate.data_ptr(), _pointer(ws), need, stream)
    check(st, "f3m_decay_attention_grad")
    return dq, dk, dv, dstate


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, q, k, v, log_decay, state, scale):
        out, final = _decay_forward(plan, q, k, v, log_decay, state, scale)
        ctx.save_for_backward(q, k, v, log_decay, state)
        ctx.plan, ctx.scale = plan, scale
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        _refuse_capture("decay_attention")
        q, k, v, log_decay, state = ctx.saved_tensors
        dq, dk, dv, dstate = decay_attention_grad(ctx.plan, q, k, v, log_decay, dout, state, dfinal, ctx.scale)
        return None, dq, dk, dv, None, dstate if state is not None else None, None


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                         scale: Optional[float] = None) -> torch.Tensor:
    """One new token for each of n sequences: q, k (n, heads, width_k), v (n, heads, width_v); state (n, heads, width_k, width_v) float32,
    contiguous, is updated in place.  Returns out like v."""
    _refuse_tangents(q, k, v, log_decay, state)
    kind = _type_of(q, k, v)
    _check_decay(q, k, v, log_decay)
    _shape(state, (q.shape[0], q.shape[1], q.shape[2], v.shape[2]), "state")
    if state.dtype != torch.float32 or state.device != q.device or not state.is_contiguous() or state.data_ptr() % 16:
        raise TypeError("state must be a contiguous float32 array on the device of q that starts on 16 bytes: it is updated in place")
    if _needs_grad(q, k, v, log_decay, state):
        raise RuntimeError("decay_attention_step has no gradient: call it under torch.no_grad()")
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    log_decay = log_decay.contiguous()
    (q, rq), (k, rk), (v, rv), (out, ro) = _read(q), _read(k), _read(v), _new(v)
    n, heads, width = q.shape
    with _On(q.device) as stream:
        st = _lib.lib().f3m_decay_attention_step(n, kind, heads, width, v.shape[2], log_decay.data_ptr(), scale, rq, rk, rv, state.data_ptr(), ro, stream)
    check(st, "f3m_decay_attention_step")
    torch.autograd.graph.increment_version(state)
    return out
