"""What the kernel products over sequences check before they touch a GPU: the table of tiles, arguments of the C entries."""
import ctypes as C

import numpy as np
import pytest
import torch

from f3m_b200 import _lib, sequence
from f3m_b200._lib import Rows, Seqs


def layout(lengths):
    L, s = _lib.lib(), Seqs()
    host = np.array(lengths, dtype=np.int32)
    assert L.f3m_seqs_layout(host.ctypes.data, len(lengths), C.byref(s), None) == 0
    table = np.full(s.table_words, -1, dtype=np.int32)
    assert L.f3m_seqs_layout(host.ctypes.data, len(lengths), C.byref(s), table.ctypes.data) == 0
    return s, table.reshape(-1, 4)


@pytest.mark.parametrize("lengths", [[1], [0], [128, 129, 0, 1, 5000], [7] * 40])
def test_layout(lengths):
    s, t = layout(lengths)
    assert (s.tokens, s.sequences, s.empty, s.longest) == (sum(lengths), len(lengths), lengths.count(0), max(lengths))
    first = np.cumsum(lengths) - lengths
    tiles = [(first[i], n, a, i) for i, n in enumerate(lengths) for a in range(0, n, 128)]
    assert s.tiles == len(tiles) and len(t) == 3 * len(tiles) + len(lengths) + s.pairs
    by = [t[k * s.tiles:(k + 1) * s.tiles] for k in range(3)]
    assert by[0].tolist() == [list(map(int, x)) for x in tiles]
    for b in by[1:]:
        assert sorted(b.tolist()) == sorted(by[0].tolist())
    assert (np.diff(by[1][:, 2]) <= 0).all() and (np.diff(by[2][:, 1] - by[2][:, 2]) <= 0).all()
    at = 0
    even = [r for r in by[1].tolist() if r[2] % 256 == 0]
    assert s.pairs == len(even) == sum(-(-n // 256) for n in lengths) and t[3 * s.tiles + len(lengths):].tolist() == even
    for i, row in enumerate(t[3 * s.tiles:3 * s.tiles + len(lengths)].tolist()):
        n = -(-lengths[i] // 128)
        assert row == [first[i], lengths[i], at, n]
        at += n


def test_layout_refusals():
    L, s = _lib.lib(), Seqs()
    for bad in ([-1], [2 ** 31 - 1, 2 ** 31 - 1]):
        host = np.array(bad, dtype=np.int32)
        assert L.f3m_seqs_layout(host.ctypes.data, len(bad), C.byref(s), None) in (1, 4)
        assert L.f3m_last_error()
    for bad in ([1.5], [[1, 2]], [-1], [2 ** 31]):
        with pytest.raises(ValueError):
            sequence.SequencePlan(bad)
    with pytest.raises(ValueError):
        sequence.SequencePlan([1], device="cpu")


def test_argument_checks_of_the_entries():
    """Every call here is refused before anything is launched: the pointers are never followed."""
    L = _lib.lib()
    s, t = layout([100, 30])
    buf = np.zeros(64, dtype=np.uint8)
    base = buf.ctypes.data + (-buf.ctypes.data) % 16
    s.table = base
    ok = Rows(base, 128, 64)        # 130 tokens, 2 heads, width 64

    def window(q=ok, k=ok, v=ok, out=ok, type=1, heads=2, kv=2, width=64, window=4, sinks=0, scale=0.1, lse=base, seqs=s):
        return L.f3m_window_attention(C.byref(seqs), type, heads, kv, width, window, sinks, scale, q, k, v, out, lse, None)

    none = Rows(None, 128, 64)
    assert window(type=3) == 5 and window(width=60) == 5 and window(width=136) == 5 and window(width=0) == 5
    assert window(heads=3) == 1 and window(kv=0) == 1 and window(heads=0, kv=1) == 1
    assert window(window=0) == 1 and window(sinks=-1) == 1 and window(scale=float("inf")) == 1
    assert window(q=none) == 1 and window(out=none) == 1 and window(lse=None) == 1
    assert window(q=Rows(base + 2, 128, 64)) == 1 and window(k=Rows(base, 132, 64)) == 1 and window(v=Rows(base, 128, -64)) == 1
    assert window(out=Rows(base, 64, 64)) == 1 and b"overlap" in L.f3m_last_error()
    assert window(out=Rows(base, 128, 0)) == 1
    bad = Seqs(None, 130, 2, 0, 3, 2, 100, 0)
    assert window(seqs=bad) == 1

    def grad(ws=base, have=1 << 20, dk=ok):
        return L.f3m_window_attention_grad(C.byref(s), 1, 2, 2, 64, 4, 0, 0.1, ok, ok, ok, ok, base, ok, ok, dk, ok, ws, have, None)

    need = L.f3m_window_attention_grad_workspace_bytes(C.byref(s), 2, 2, 64, 4, 0)
    assert need > 0 and grad(have=need - 1) == 7 and grad(ws=None) == 1 and grad(ws=base + 4) == 1 and grad(dk=Rows(base, 8, 64)) == 1

    def step(n=2, cap=100, lens=base, ws=base, have=1 << 40, k=ok, seq=12800):
        return L.f3m_window_attention_step(n, 1, 2, 2, 64, cap, 50, 0, 0.1, ok, k, seq, ok, seq, lens, ok, ws, have, None)

    assert step(n=-1) == 1 and step(cap=-1) == 1 and step(cap=1 << 31) == 1 and step(lens=None) == 1 and step(k=none) == 1 and step(seq=4) == 1

    def decay(q=ok, state_in=None, state_out=None, ld=base, wk=64, ws=base, have=1 << 40):
        return L.f3m_decay_attention(C.byref(s), 1, 2, wk, 64, ld, 0.1, q, ok, ok, state_in, ok, state_out, ws, have, None)

    assert decay(q=none) == 1 and decay(ld=None) == 1 and decay(wk=12) == 5 and decay(state_in=base + 4) == 1
    assert decay(state_in=base, state_out=base) == 1 and b"same array" in L.f3m_last_error()
    assert L.f3m_decay_attention_step(2, 1, 2, 64, 64, base, 0.1, ok, ok, ok, None, ok, None) == 1
    assert L.f3m_decay_attention_step(2, 1, 2, 64, 64, base, float("nan"), ok, ok, ok, base, ok, None) == 1


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        sequence.window_attention_step(x, x[:, None], x[:, None], torch.ones(4, dtype=torch.int32), 4)
    with pytest.raises(ValueError):
        sequence.decay_attention_step(x, x, x, torch.zeros(2), torch.zeros(4, 2, 64, 64))


def test_gradient_workspace_of_uneven_batches():
    """Sums of parts of walks over the keys that hold sinks take room where a walk is cut, not for every sequence beside the longest."""
    L = _lib.lib()

    def need(lengths, heads, kv, width, window, sinks):
        s, _ = layout(lengths)
        rows = 2 * 4 * sum(lengths) * heads
        return L.f3m_window_attention_grad_workspace_bytes(C.byref(s), heads, kv, width, window, sinks) - rows

    # 2 x 148 CTAs' worth of parts and as many again where lengths fall badly, dk and dv of 128 keys each, in FP32
    most = 4 * 148 * 2 * 128 * 128 * 4 + (1 << 20)
    assert need([16384] + [64] * 2000, 32, 8, 128, 128, 4) < most
    assert need([32768] + [64] * 1000, 32, 8, 128, 1024, 16) < most
    assert need([32768] + [128] * 500, 32, 4, 128, 256, 4) < most
    assert need([65536], 32, 8, 128, 512, 65536) < most
    assert need([64] * 5000, 32, 8, 128, 128, 4) < 1 << 20            # no walk is cut
    assert need([16384] + [64] * 2000, 32, 8, 128, 128, 0) < 1 << 20


def test_forward_mode_derivatives_are_refused():
    """A tangent would be dropped without a word: the library takes addresses."""
    from torch.autograd import forward_ad
    x, ld, state = torch.ones(4, 2, 64, dtype=torch.bfloat16), torch.zeros(2), torch.zeros(4, 2, 64, 64)
    lens, lse = torch.ones(4, dtype=torch.int32), torch.zeros(2, 4)
    calls = [lambda d: sequence.window_attention(None, x, d, x, 4), lambda d: sequence.window_attention_grad(None, x, x, x, x, lse, d, 4),
             lambda d: sequence.window_attention_step(d, x[:, None], x[:, None], lens, 4), lambda d: sequence.decay_attention(None, x, x, d, ld),
             lambda d: sequence.decay_attention_grad(None, d, x, x, ld, x), lambda d: sequence.decay_attention_step(x, d, x, ld, state)]
    with forward_ad.dual_level():
        dual, plain = forward_ad.make_dual(x, torch.ones_like(x)), 0
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
        with pytest.raises(RuntimeError, match="forward-mode"):
            sequence.decay_attention(None, x, x, x, ld, forward_ad.make_dual(state, state))
        for call in calls:                      # without a tangent it is the CPU that is refused, as ever
            with pytest.raises((ValueError, RuntimeError)) as e:
                call(x)
            plain += "forward-mode" not in str(e.value)
        assert plain == len(calls)
