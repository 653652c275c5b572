"""What the paged cache and the gated recurrence check before they touch a GPU, and their references against each other."""
import ctypes as C

import numpy as np
import pytest
import torch

import paged_reference
import recurrence_reference
from f3m_b200 import _lib, paged, sequence
from f3m_b200._lib import Cache, Pages, RotationTable, Rows, Seqs


def layout(lengths):
    L, s = _lib.lib(), Seqs()
    host = np.array(lengths, dtype=np.int32)
    assert L.f3m_seqs_layout(host.ctypes.data, len(lengths), C.byref(s), None) == 0
    return s


@pytest.fixture
def base():
    buf = np.zeros(64, dtype=np.uint8)
    yield buf.ctypes.data + (-buf.ctypes.data) % 16


def test_entries_of_the_paged_cache(base):
    """Every call here is refused before anything is launched: the pointers are never followed."""
    L, s = _lib.lib(), layout([100, 30])
    s.table = base
    kv = Rows(base, 128, 64)                       # 130 tokens, 2 heads, width 64

    def cache(**o):
        d = dict(k=Pages(base, 2048, 128, 64), v=Pages(base, 2048, 128, 64), pages=10, page_tokens=16, kv_heads=2, width=64, table=base, table_stride=20, table_pages=20, sequences=2,
                 lengths=base)
        return Cache(*{**d, **o}.values())

    def attend(c=None, type=1, heads=4, window=9, sinks=0, scale=0.1, parents=None, q=Rows(base, 256, 64), out=Rows(base, 256, 64), ws=base, have=1 << 40, seqs=s):
        return L.f3m_paged_attention(C.byref(seqs), type, C.byref(c or cache()), heads, window, sinks, scale, parents, q, out, ws, have, None)

    assert attend(type=3) == 5 and attend(cache(width=60)) == 5 and attend(cache(page_tokens=12)) == 5 and attend(cache(page_tokens=4)) == 5 and attend(cache(page_tokens=0)) == 5
    assert attend(cache(kv_heads=0)) == 1 and attend(cache(lengths=None)) == 1 and attend(cache(table=None)) == 1 and attend(cache(pages=-1)) == 1
    assert attend(cache(table_pages=1 << 28)) == 1 and attend(cache(table_pages=(1 << 27) - 17)) == 4 and attend(cache(sequences=3)) == 1
    assert attend(cache(k=Pages(None, 2048, 128, 64))) == 1 and attend(cache(v=Pages(base, 2044, 128, 64))) == 1 and attend(cache(k=Pages(base + 8, 2048, 128, 64))) == 1
    assert attend(heads=3) == 1 and attend(heads=0) == 1 and attend(heads=258) == 5 and attend(window=0) == 1 and attend(sinks=-1) == 1 and attend(scale=float("nan")) == 1
    assert attend(q=Rows(None, 256, 64)) == 1 and attend(out=Rows(base, 64, 64)) == 1
    assert attend(seqs=Seqs(None, 130, 2, 0, 3, 2, 100, 0)) == 1
    long = layout([257, 1])
    long.table = base
    assert attend(parents=base, seqs=long) == 5
    need = L.f3m_paged_attention_workspace_bytes(C.byref(s), C.byref(cache()), 4)
    assert need == 0 or attend(have=need - 1) == 7 and attend(ws=None) == 1 and attend(ws=base + 4) == 1

    def append(c=None, k=kv, heads=0, q=kv, q_out=kv, rotation=None):
        return L.f3m_paged_append(C.byref(s), 1, C.byref(c or cache()), k, kv, None, None if rotation is None else C.byref(rotation), heads, q, q_out, None)

    assert append(k=Rows(base, 132, 64)) == 1 and append(heads=-1) == 1 and append(heads=2, q=Rows(None, 128, 64)) == 1 and append(heads=2, q_out=Rows(base, 256, 64)) == 1
    assert append(cache(k=Pages(base, 2048, 64, 64))) == 1 and b"overlap" in L.f3m_last_error() and append(cache(v=Pages(base, 0, 128, 64))) == 1
    assert append(rotation=RotationTable(base, 24, 0)) == 5 and append(rotation=RotationTable(base, 80, 0)) == 5 and append(rotation=RotationTable(base, 0, 0)) == 5
    assert append(rotation=RotationTable(None, 32, 0)) == 1 and append(rotation=RotationTable(base + 4, 32, 0)) == 1

    def keep(c=None, type=1, kept=base, stride=4, most=4, counts=base):
        return L.f3m_paged_keep(type, C.byref(c or cache()), kept, stride, most, counts, None)

    assert keep(type=0) == 5 and keep(kept=None) == 1 and keep(counts=None) == 1 and keep(most=-1) == 1 and keep(stride=-1) == 1 and keep(cache(v=Pages(base, 2048, 128, 0))) == 1


def test_entries_of_the_gated_recurrence(base):
    L, s = _lib.lib(), layout([100, 30])
    s.table = base
    ok = Rows(base, 64, 0)

    def forward(type=1, channels=64, x=ok, ld=ok, out=ok, state_in=None, state_out=None, ws=base, have=1 << 40):
        return L.f3m_gated_recurrence(C.byref(s), type, channels, x, ld, state_in, out, state_out, ws, have, None)

    assert forward(type=0) == 5 and forward(channels=60) == 5 and forward(channels=0) == 5 and forward(channels=1 << 21) == 5
    assert forward(x=Rows(None, 64, 0)) == 1 and forward(ld=Rows(base, 60, 0)) == 1 and forward(out=Rows(base, 56, 0)) == 1 and forward(x=Rows(base + 8, 64, 0)) == 1
    assert forward(state_in=base, state_out=base) == 1 and forward(state_out=base + 4) == 1 and forward(x=Rows(base, -64, 0)) == 1 and forward(type=3, x=Rows(base, 66, 0)) == 1
    need = L.f3m_gated_recurrence_workspace_bytes(C.byref(s), 64)
    assert need == 0 or forward(have=need - 1) == 7 and forward(ws=None) == 1

    def grad(ld=ok, out=ok, dout=ok, dx=ok, dl=ok, dstate_out=None, dstate_in=None, ws=base, have=1 << 40):
        return L.f3m_gated_recurrence_grad(C.byref(s), 2, 64, ld, out, dout, None, dstate_out, dx, dl, dstate_in, ws, have, None)

    bad = Rows(base, 32, 0)
    assert grad(dx=bad) == 1 and grad(dl=bad) == 1 and grad(out=Rows(None, 64, 0)) == 1 and grad(dstate_out=base, dstate_in=base) == 1 and (need == 0 or grad(have=need - 1) == 7)
    assert L.f3m_gated_recurrence_step(1, 1, 64, ok, ok, None, ok, None) == 1 and L.f3m_gated_recurrence_step(-1, 1, 64, ok, ok, base, ok, None) == 1


def test_cpu_tensors_and_tangents_are_refused():
    from torch.autograd import forward_ad
    x, ints = torch.ones(2, 1, 64, dtype=torch.bfloat16), lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    pages, y = torch.ones(3, 8, 1, 64, dtype=torch.bfloat16), torch.ones(2, 64)
    calls = [lambda d: paged.paged_append(None, d, x, pages, pages, ints(2, 1), ints(2)), lambda d: paged.paged_append(None, x, x, pages, pages, ints(2, 1), ints(2), q=d),
             lambda d: paged.paged_attention(None, d, pages, pages, ints(2, 1), ints(2))]
    more = [lambda d: sequence.gated_recurrence(None, d, y), lambda d: sequence.gated_recurrence(None, y, y, d), lambda d: sequence.gated_recurrence_grad(None, y, y, d),
            lambda d: sequence.gated_recurrence_step(y, d, y)]
    pool = [lambda d: paged.paged_keep(d, pages, ints(2, 1), ints(2), ints(2, 1), ints(2)), lambda d: paged.paged_attention(None, x, pages, d, ints(2, 1), ints(2))]
    for group, plain in ((calls, x), (more, y), (pool, pages)):
        for call in group:
            with pytest.raises(ValueError, match="CPU"):
                call(plain)
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(plain, torch.ones_like(plain)))


def test_reference_of_the_recurrence_against_differences():
    g = torch.Generator().manual_seed(1)
    lengths, c = [7, 0, 1, 12], 3
    x, ld = torch.randn(20, c, generator=g, dtype=torch.float64), -torch.rand(20, c, generator=g, dtype=torch.float64)
    st, do, df = torch.randn(4, c, generator=g, dtype=torch.float64), torch.randn(20, c, generator=g, dtype=torch.float64), torch.randn(4, c, generator=g, dtype=torch.float64)
    as_type = lambda t: t.float()  # noqa: E731
    x, ld, st, do, df = map(as_type, (x, ld, st, do, df))
    want = recurrence_reference.recurrence(x, ld, lengths, st, do, df)

    def loss(args):
        w = recurrence_reference.recurrence(args[0], args[1], lengths, args[2])
        return float((w["out"][0] * do).sum() + (w["final"][0] * df).sum())

    for i, name in enumerate(("dx", "dlog", "dstate")):
        along = torch.randn((x, ld, st)[i].shape, generator=g, dtype=torch.float64)
        up, down = ([y.double() + (sign * 1e-6 * along if j == i else 0) for j, y in enumerate((x, ld, st))] for sign in (1, -1))
        slope = (loss(up) - loss(down)) / 2e-6
        assert abs(slope - float((along * want[name][0]).sum())) < 1e-6 * (1 + float((along * want[name][0]).abs().sum()))


def test_reference_of_the_attention_sees_what_it_should():
    """A chain is the window's rule on one axis; a tree's path sees what the chain of its tokens would."""
    g = torch.Generator().manual_seed(2)
    kp, vp, q = (torch.randn(6, 8, 1, 16, generator=g).half() for _ in range(3))
    table, q = torch.tensor([[4, 2, 0, 5]], dtype=torch.int32), q.view(-1, 1, 16)[:6]
    chain, _ = paged_reference.attention(q[:3], kp, vp, table, [20], [3], 7, 2)
    rows = torch.tensor([4, 2, 0])
    k, v = (x[rows].reshape(24, 16)[:23].double() for x in (kp, vp))
    for i in range(3):
        j = [j for j in range(21 + i) if 20 + i - j < 7 or j < 2]
        p = torch.softmax(k[j] @ q[i, 0].double() / 4, 0)
        assert torch.allclose(p @ v[j], chain[i, 0])
    # tokens 0, 2, 5 of a tree in places 20, 22, 25, at positions 20, 21, 22
    parents = torch.tensor([-1, 0, 0, 1, 1, 2])
    got, _ = paged_reference.attention(q, kp, vp, table, [20], [6], 7, 2, parents)
    k2, v2 = kp.clone(), vp.clone()
    for place, source in ((21, 22), (22, 25)):
        for x, y in ((k2, kp), (v2, vp)):
            x[table[0, place // 8], place % 8] = y[table[0, source // 8], source % 8]
    path, _ = paged_reference.attention(q[[0, 2, 5]], k2, v2, table, [20], [3], 7, 2)
    assert torch.allclose(got[[0, 2, 5]], path)
