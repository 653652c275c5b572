"""Kernel products over sequences against their definitions in 64 bits (sequence_reference.py says how the bounds come about)."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def normal(seed, *shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


# lengths, heads, kv_heads, width, window, sinks: tiles cut anywhere, windows inside a tile and beyond the sequence, sinks inside the
# window, across a tile's end and behind the sequence; one head, shared heads in odd and even numbers; widths of half a tile and odd ones
WINDOWS = [
    ([1], 1, 1, 64, 1, 0),
    ([129], 2, 2, 64, 1, 0),
    ([128, 0, 1, 127], 4, 2, 64, 64, 0),
    ([300, 17], 3, 1, 128, 100, 5),
    ([700], 2, 1, 128, 5000, 0),
    ([700, 513], 6, 2, 128, 130, 140),
    ([640], 4, 4, 32, 257, 1),
    ([515, 2], 8, 1, 80, 129, 128),
    ([260], 5, 5, 8, 50, 300),
    ([1030], 2, 2, 104, 1, 1),
    ([900], 16, 2, 96, 384, 0),
    ([2300, 130, 900], 16, 2, 64, 200, 8),         # key tiles with sinks are cut into parts
    ([1700], 12, 3, 128, 128, 150),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,kv_heads,width,window,sinks", WINDOWS)
def test_window_attention_and_gradients(lengths, heads, kv_heads, width, window, sinks, dtype, cuda):
    from f3m_b200 import sequence as sq
    n = sum(lengths)
    q, do = normal(1, n, heads, width, dtype=dtype, scale=1.5), normal(2, n, heads, width, dtype=dtype)
    k, v = normal(3, n, kv_heads, width, dtype=dtype), normal(4, n, kv_heads, width, dtype=dtype)
    plan = sq.SequencePlan(lengths)
    want = ref.window(q, k, v, lengths, window, sinks, dout=do)
    out, lse = sq.window_attention(plan, q, k, v, window, sinks)
    ref.assert_within(out, want["out"], "out")
    ref.assert_within(lse, want["lse"], "lse")
    got = sq.window_attention_grad(plan, q, k, v, out, lse, do, window, sinks)
    for name, x in zip(("dq", "dk", "dv"), got):
        ref.assert_within(x, want[name], name)


@pytest.mark.parametrize("dtype", TYPES)
def test_window_attention_scale_and_views(dtype, cuda):
    """Views of one joint projection, heads before tokens, broadcast key heads, an array that starts off 16 bytes."""
    from f3m_b200 import sequence as sq
    lengths, h, w = [200, 131], 4, 64
    n = sum(lengths)
    plan = sq.SequencePlan(lengths)
    joint = normal(5, n, 3, h, w, dtype=dtype)
    q, k, v = joint[:, 0], joint[:, 1], joint[:, 2]
    do = normal(6, h, n, w, dtype=dtype).transpose(0, 1)
    for kk, vv in ((k, v), (k[:, :1].expand(n, h, w), v), (k[:, :2], v[:, 1:3])):
        want = ref.window(q, kk, vv, lengths, 70, 3, scale=0.3, dout=do)
        out, lse = sq.window_attention(plan, q, kk, vv, 70, 3, scale=0.3)
        ref.assert_within(out, want["out"])
        for name, x in zip(("dq", "dk", "dv"), sq.window_attention_grad(plan, q, kk, vv, out, lse, do, 70, 3, scale=0.3)):
            ref.assert_within(x, want[name], name)
    flat = normal(7, n * h * w + 1, dtype=dtype)
    odd = flat[1:].view(n, h, w)
    ref.assert_within(sq.window_attention(plan, odd, k, v, 70)[0], ref.window(odd, k, v, lengths, 70, 0)["out"])


@pytest.mark.parametrize("dtype", TYPES)
def test_window_attention_large_exponents(dtype, cuda):
    """Rows whose largest weight comes first, last, and rises tile by tile; a negative scale."""
    from f3m_b200 import sequence as sq
    n, h, w = 600, 2, 64
    plan = sq.SequencePlan([n])
    v = normal(11, n, h, w, dtype=dtype)
    q = torch.ones(n, h, w, device="cuda", dtype=dtype)
    for slope in (0.05, -0.05, 0.5):
        k = (torch.arange(n, device="cuda") * slope)[:, None, None].expand(n, h, w).to(dtype).contiguous()
        for scale in (0.125, -0.125):
            want = ref.window(q, k, v, [n], 400, 7, scale=scale)
            out, lse = sq.window_attention(plan, q, k, v, 400, 7, scale=scale)
            ref.assert_within(out, want["out"], f"slope {slope} scale {scale}")
            ref.assert_within(lse, want["lse"])


def test_a_sequence_does_not_reach_its_neighbours(cuda):
    """What is not finite in one sequence stays there, in the tiles that two sequences share in memory too."""
    from f3m_b200 import sequence as sq
    lengths, h, w = [100, 60, 300], 2, 64
    plan = sq.SequencePlan(lengths)
    q, k, v, do = (normal(20 + i, sum(lengths), h, w, dtype=torch.bfloat16) for i in range(4))
    ld = torch.tensor([-0.1, -0.01], device="cuda")
    bad = [x.clone() for x in (q, k, v, do)]
    for x in bad:
        x[100:160] = float("nan")
        x[110] = float("inf")
    keep = torch.ones(sum(lengths), dtype=torch.bool, device="cuda")
    keep[100:160] = False
    a, b = sq.window_attention(plan, q, k, v, 80, 2), sq.window_attention(plan, *bad[:3], 80, 2)
    assert torch.equal(a[0][keep], b[0][keep]) and torch.equal(a[1][:, keep], b[1][:, keep])
    ga, gb = sq.window_attention_grad(plan, q, k, v, *a, do, 80, 2), sq.window_attention_grad(plan, *bad[:3], *b, bad[3], 80, 2)
    for x, y in zip(ga, gb):
        assert torch.equal(x[keep], y[keep])
    a, b = sq.decay_attention(plan, q, k, v, ld), sq.decay_attention(plan, *bad[:3], ld)
    assert torch.equal(a[0][keep], b[0][keep]) and torch.equal(a[1][[0, 2]], b[1][[0, 2]])
    ga, gb = sq.decay_attention_grad(plan, q, k, v, ld, do), sq.decay_attention_grad(plan, *bad[:3], ld, bad[3])
    for x, y in zip(ga[:3], gb[:3]):
        assert torch.equal(x[keep], y[keep])
    assert torch.equal(ga[3][[0, 2]], gb[3][[0, 2]])


# n, capacity, heads, kv_heads, width, window, sinks
STEPS = [
    (1, 1, 1, 1, 64, 1, 0),
    (3, 40, 4, 2, 64, 16, 2),
    (5, 1000, 8, 1, 128, 100000, 0),
    (2, 5000, 32, 4, 128, 777, 4),
    (2, 3001, 6, 2, 80, 3001, 0),
    (4, 300, 20, 1, 8, 50, 200),
    (1, 70000, 16, 16, 96, 65000, 128),
    (70, 600, 2, 1, 32, 300, 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,capacity,heads,kv_heads,width,window,sinks", STEPS)
def test_window_attention_step(n, capacity, heads, kv_heads, width, window, sinks, dtype, cuda):
    from f3m_b200 import sequence as sq
    q = normal(1, n, heads, width, dtype=dtype, scale=2.0)
    kc, vc = normal(2, n, capacity, kv_heads, width, dtype=dtype), normal(3, n, capacity, kv_heads, width, dtype=dtype)
    lengths = [max(0, capacity - 97 * b * (b + 1) // 2) for b in range(n)]
    if n > 1:
        lengths[1] = capacity + 5           # taken as the capacity
    if n > 2:
        lengths[2] = -1                     # and this as an empty cache
    for b, x in enumerate(lengths):         # what lies behind the tokens is not read
        kc[b, max(0, min(x, capacity)):] = float("nan")
        vc[b, max(0, min(x, capacity)):] = float("inf")
    want = ref.window_step(q, kc, vc, lengths, window, sinks)
    got = sq.window_attention_step(q, kc, vc, torch.tensor(lengths, dtype=torch.int32, device="cuda"), window, sinks)
    ref.assert_within(got, want)


def test_window_attention_step_reads_only_what_is_seen(cuda):
    """Tokens between the sinks and the window may hold anything; a cache laid out heads first, one that starts inside another array."""
    from f3m_b200 import sequence as sq
    n, cap, h, w = 2, 900, 2, 64
    lens = torch.tensor([900, 431], dtype=torch.int32, device="cuda")
    q = normal(1, n, 4, w, dtype=torch.bfloat16)
    kc = normal(2, n + 1, h, cap, w, dtype=torch.bfloat16).transpose(1, 2)[1:]
    vc = normal(3, n, cap, h, 2 * w, dtype=torch.bfloat16)[..., w:]
    kc[0, 5:800], vc[0, 5:800] = float("nan"), float("nan")
    kc[1, 5:331], vc[1, 5:331] = float("nan"), float("nan")
    ref.assert_within(sq.window_attention_step(q, kc, vc, lens, 100, 5), ref.window_step(q, kc, vc, [900, 431], 100, 5))


def test_window_attention_step_far_into_a_cache(cuda):
    """Offsets beyond 2^31 elements and beyond 2^32 bytes."""
    from f3m_b200 import sequence as sq
    cap, h, w = 1_200_000, 16, 128
    kc = torch.zeros(1, cap, h, w, device="cuda", dtype=torch.bfloat16)
    vc = torch.zeros(1, cap, h, w, device="cuda", dtype=torch.bfloat16)
    kc[:, -500:], vc[:, -500:] = normal(1, 1, 500, h, w, dtype=torch.bfloat16), normal(2, 1, 500, h, w, dtype=torch.bfloat16)
    q = normal(3, 1, h, w, dtype=torch.bfloat16)
    got = sq.window_attention_step(q, kc, vc, torch.tensor([cap], dtype=torch.int32, device="cuda"), 300, 0)
    ref.assert_within(got, ref.window_step(q, kc, vc, [cap], 300, 0))


# lengths, heads, width_k, width_v, log_decay of the heads, with states
DECAYS = [
    ([1], 1, 64, 64, [-0.1], True),
    ([129], 2, 64, 64, [-0.5, 0.0], False),
    ([128, 0, 1, 127], 3, 128, 128, [-1e-3, -0.1, -3.0], True),
    ([700, 300], 2, 128, 64, [-0.02, -100.0], True),
    ([515], 2, 32, 128, [float("-inf"), -0.01], True),
    ([260, 17], 2, 80, 8, [-0.2, 1.0], True),
    ([1500], 1, 128, 128, [-0.004], True),
    ([130] * 7, 2, 96, 104, [-0.05, -0.7], False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,width_k,width_v,log_decay,carried", DECAYS)
def test_decay_attention_and_gradients(lengths, heads, width_k, width_v, log_decay, carried, dtype, cuda):
    from f3m_b200 import sequence as sq
    n = sum(lengths)
    q, k = normal(1, n, heads, width_k, dtype=dtype), normal(2, n, heads, width_k, dtype=dtype)
    v, do = normal(3, n, heads, width_v, dtype=dtype), normal(4, n, heads, width_v, dtype=dtype)
    ld = torch.tensor(log_decay, device="cuda")
    state = normal(5, len(lengths), heads, width_k, width_v, dtype=torch.float32) if carried else None
    dfinal = normal(6, len(lengths), heads, width_k, width_v, dtype=torch.float32) if carried else None
    plan = sq.SequencePlan(lengths)
    want = ref.decay(q, k, v, log_decay, lengths, state, dout=do, dfinal=dfinal)
    out, final = sq.decay_attention(plan, q, k, v, ld, state)
    ref.assert_within(out, want["out"], "out")
    ref.assert_within(final, want["final"], "final")
    for name, x in zip(("dq", "dk", "dv", "dstate"), sq.decay_attention_grad(plan, q, k, v, ld, do, state, dfinal)):
        ref.assert_within(x, want[name], name)


@pytest.mark.parametrize("heads,tokens", [(1, 6000), (2, 20000)])
def test_decay_attention_split_over_a_long_sequence(heads, tokens, cuda):
    """Few heads and many tokens: the work of a head is cut into ranges whose states are joined."""
    from f3m_b200 import sequence as sq
    lengths = [tokens - 777, 1, 776]
    q, k, v, do = (normal(i, tokens, heads, 64, dtype=torch.bfloat16) for i in range(4))
    log_decay = [-0.0005, -0.03][:heads]
    ld = torch.tensor(log_decay, device="cuda")
    state, dfinal = (normal(7 + i, 3, heads, 64, 64, dtype=torch.float32) for i in range(2))
    plan = sq.SequencePlan(lengths)
    out, final = sq.decay_attention(plan, q, k, v, ld, state)
    got = sq.decay_attention_grad(plan, q, k, v, ld, do, state, dfinal)
    again = sq.decay_attention_grad(plan, q, k, v, ld, do, state, dfinal)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    if tokens > 10000:        # the definition over all pairs, head by head: keep it to what fits
        want = ref.decay(q[:, :1], k[:, :1], v[:, :1], log_decay[:1], lengths, state[:, :1], dout=do[:, :1], dfinal=dfinal[:, :1])
        out, final, got = out[:, :1], final[:, :1], [x[:, :1] for x in got]
    else:
        want = ref.decay(q, k, v, log_decay, lengths, state, dout=do, dfinal=dfinal)
    ref.assert_within(out, want["out"], "out")
    ref.assert_within(final, want["final"], "final")
    for name, x in zip(("dq", "dk", "dv", "dstate"), got):
        ref.assert_within(x, want[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads,width_k,width_v", [(1, 1, 8, 8), (3, 2, 64, 128), (2, 5, 128, 128), (70, 3, 72, 104), (2, 2, 128, 24)])
def test_decay_attention_step(n, heads, width_k, width_v, dtype, cuda):
    from f3m_b200 import sequence as sq
    ld = -torch.rand(heads, device="cuda")
    ld[0] = float("-inf")
    q, k, v = normal(1, n, heads, width_k, dtype=dtype), normal(2, n, heads, width_k, dtype=dtype), normal(3, n, heads, width_v, dtype=dtype)
    state = normal(4, n, heads, width_k, width_v, dtype=torch.float32)
    S = state.double() * torch.exp(ld.double())[:, None, None] + k.double()[..., None] * v.double()[..., None, :]
    o, mass = torch.einsum("nhk,nhkv->nhv", q.double(), S) * width_k ** -0.5, torch.einsum("nhk,nhkv->nhv", q.double().abs(), S.abs()) * width_k ** -0.5
    version = state._version
    out = sq.decay_attention_step(q, k, v, ld, state)
    assert state._version > version
    ref.assert_within(state, (S, 1e-6 * (S.abs() + 1)), "state")
    ref.assert_within(out, (o, ref.half_step(dtype) * o.abs() + 1e-6 * mass + ref.tiny(dtype)), "out")


def test_many_calls_in_a_row(cuda):
    """The roles of a kernel's warps run apart from one another in ways that differ from call to call: the bits do not, and no wait runs out."""
    from f3m_b200 import sequence as sq
    tokens, h = 20011, 4
    lengths = [tokens - 300, 299, 1]
    q, k, v, do = (normal(i, tokens, h, 128, dtype=torch.bfloat16) for i in range(4))
    ld = torch.tensor([-0.001, -0.03, -0.2, 0.0], device="cuda")
    plan = sq.SequencePlan(lengths)

    def calls():
        out, lse = sq.window_attention(plan, q, k[:, :2], v[:, :2], 300, 5)
        return (out, lse) + sq.window_attention_grad(plan, q, k[:, :2], v[:, :2], out, lse, do, 300, 5) + sq.decay_attention(plan, q, k, v, ld) + sq.decay_attention_grad(plan, q, k, v, ld, do)

    first = calls()
    for _ in range(150):
        again = calls()
        assert all(torch.equal(x, y) for x, y in zip(again, first))


def test_steps_continue_a_prompt(cuda):
    """A prompt, then its answer token by token, as a model runs it: the same outputs as reading all of it at once."""
    from f3m_b200 import sequence as sq
    n, more, h, hk, w, window, sinks, dt = 300, 6, 4, 2, 64, 100, 4, torch.bfloat16
    q, k, v = normal(1, n + more, h, w, dtype=dt), normal(2, n + more, hk, w, dtype=dt), normal(3, n + more, hk, w, dtype=dt)
    kd, vd = k.repeat_interleave(h // hk, 1), v.repeat_interleave(h // hk, 1)
    ld = torch.tensor([-0.01, -0.1, -0.5, 0.0], device="cuda")
    want = ref.window(q, k, v, [n + more], window, sinks)["out"]
    want_d = ref.decay(q, kd, vd, ld.tolist(), [n + more])
    plan = sq.SequencePlan([n])
    cache = [torch.full((1, 512, hk, w), float("nan"), device="cuda", dtype=dt) for _ in range(2)]
    cache[0][0, :n], cache[1][0, :n] = k[:n], v[:n]
    ref.assert_within(sq.window_attention(plan, q[:n], k[:n], v[:n], window, sinks)[0], [x[:n] for x in want])
    out, state = sq.decay_attention(plan, q[:n], kd[:n], vd[:n], ld)
    ref.assert_within(out, [x[:n] for x in want_d["out"]])
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    for t in range(n, n + more):
        cache[0][0, t], cache[1][0, t] = k[t], v[t]
        length += 1
        ref.assert_within(sq.window_attention_step(q[t:t + 1], *cache, length, window, sinks), [x[t:t + 1] for x in want])
        out = sq.decay_attention_step(q[t:t + 1], kd[t:t + 1], vd[t:t + 1], ld, state)
        ref.assert_within(out, [x[t:t + 1] for x in want_d["out"]])
    ref.assert_within(state, want_d["final"])


def test_a_layer_of_both_is_differentiated(cuda):
    """Window attention feeding attention with a decay, differentiated by autograd: the gradients of the explicit calls; and one of them
    against differences of a 64-bit loss."""
    from f3m_b200 import sequence as sq
    lengths, h, w = [150, 40], 2, 64
    n = sum(lengths)
    plan, ld = sq.SequencePlan(lengths), torch.tensor([-0.05, -0.3], device="cuda")
    q, k, v, g = (normal(i, n, h, w, dtype=torch.float16, scale=0.5) for i in range(4))
    state = normal(9, 2, h, w, w, dtype=torch.float32)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    first, lse = sq.window_attention(plan, *leaves, 64, 2)
    s = state.clone().requires_grad_()
    out, final = sq.decay_attention(plan, leaves[0], leaves[1], first, ld, s)
    assert not lse.requires_grad
    ((out.float() * g.float()).sum() + 0.1 * final.sum()).backward()
    o1, l1 = sq.window_attention(plan, q, k, v, 64, 2)
    dq, dk, dv1, ds = sq.decay_attention_grad(plan, q, k, o1, ld, g, state, torch.full_like(state, 0.1))
    eq, ek, ev = sq.window_attention_grad(plan, q, k, v, o1, l1, dv1, 64, 2)
    for x, want in zip(leaves, (dq + eq, dk + ek, ev)):
        assert torch.allclose(x.grad.float(), want.float(), rtol=2 ** -10, atol=1e-6)     # autograd adds the two in 16 bits, once
    assert torch.equal(s.grad, ds)

    def loss(vv):
        o = ref.window(q, k, vv, lengths, 64, 2)["out"][0]
        r = ref.decay(q, k, o, ld.tolist(), lengths, state)
        return float((r["out"][0] * g.double()).sum() + 0.1 * r["final"][0].sum())

    direction = torch.randn(v.shape, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(3))
    eps = 1e-3
    slope = (loss(v.double() + eps * direction) - loss(v.double() - eps * direction)) / (2 * eps)
    along = float((leaves[2].grad.double() * direction).sum())
    # the loss is linear in v; what is left are the 16-bit roundings of first, dv1 and the gradient, of independent signs
    scale = float((leaves[2].grad.double().square() * direction.square()).sum().sqrt())
    assert abs(along - slope) <= 2 ** -11 * 8 * scale, (along, slope, scale)


def test_captured_calls(cuda):
    """Two graphs with calls of both kinds, replayed in turn on new inputs; a training step of explicit calls in one of them."""
    from f3m_b200 import sequence as sq
    lengths, h, w = [333, 129], 2, 64
    n = sum(lengths)
    plan, ld = sq.SequencePlan(lengths), torch.tensor([-0.05, -0.3], device="cuda")
    q, k, v, do = (normal(i, n, h, w, dtype=torch.bfloat16) for i in range(4))
    kc, vc = normal(7, 2, 2000, h, w, dtype=torch.bfloat16), normal(8, 2, 2000, h, w, dtype=torch.bfloat16)
    lens = torch.tensor([2000, 77], dtype=torch.int32, device="cuda")

    def train():
        out, lse = sq.window_attention(plan, q, k, v, 100, 3)
        return (out, lse) + sq.window_attention_grad(plan, q, k, v, out, lse, do, 100, 3)

    def serve():
        out, final = sq.decay_attention(plan, q, k, v, ld)
        return (out, final) + sq.decay_attention_grad(plan, q, k, v, ld, do) + (sq.window_attention_step(q[:2], kc, vc, lens, 1500, 3),)

    train(), serve()
    graphs = []
    for f in (train, serve):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = f()
        graphs.append((f, g, res))
    for seed in (11, 12):
        for i, x in enumerate((q, k, v, do)):
            x.copy_(normal(seed + 10 * i, n, h, w, dtype=torch.bfloat16))
        for _, g, _ in graphs:
            g.replay()
        graphs[0][1].replay()
        for f, _, res in graphs:
            assert all(torch.equal(x, y) for x, y in zip(f(), res))


def test_the_first_call_of_a_process_is_captured(cuda):
    """What the library makes once per process (its error word, the driver's entry point) may be made while a stream is captured."""
    import os
    import subprocess
    import sys
    code = """
import torch
from f3m_b200 import sequence as sq
plan = sq.SequencePlan([300])
q, k, v = (torch.randn(300, 2, 64, device="cuda").half() for _ in range(3))
ld = torch.tensor([-0.1, -0.01], device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a, b = sq.window_attention(plan, q, k, v, 100), sq.decay_attention(plan, q, k, v, ld)
g.replay()
c, d = sq.window_attention(plan, q, k, v, 100), sq.decay_attention(plan, q, k, v, ld)
assert all(torch.equal(x, y) for x, y in zip(a + b, c + d))
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_inference_mode_and_a_dropped_plan(cuda):
    """Under inference mode; and plans dropped while another stream still reads their tables."""
    from f3m_b200 import sequence as sq
    q, k, v = (normal(i, 5000, 2, 64, dtype=torch.bfloat16) for i in range(3))
    ld = torch.tensor([-0.1, -0.01], device="cuda")
    want = sq.window_attention(sq.SequencePlan([5000]), q, k, v, 700)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    with torch.inference_mode():
        for _ in range(20):
            plan = sq.SequencePlan([5000])
            with torch.cuda.stream(side):
                got.append(sq.window_attention(plan, q, k, v, 700))
            del plan
            torch.full((200, 4), 7, dtype=torch.int32, device="cuda")      # takes the table's memory, were it free
        state = torch.zeros(3, 2, 64, 64, device="cuda")
        sq.decay_attention_step(q[:3], k[:3], v[:3], ld, state)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for g in got for x, y in zip(g, want))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_scale_of_zero_and_large_inputs(dtype, cuda):
    """All weights equal; and exponents of some thousands, where each row has one weight or two."""
    from f3m_b200 import sequence as sq
    n, h, w = 333, 2, 64
    plan = sq.SequencePlan([n])
    q, k, v, do = (normal(30 + i, n, h, w, dtype=dtype) for i in range(4))
    for qq, scale in ((q, 0.0), (q * 40, 1.0)):
        want = ref.window(qq, k, v, [n], 90, 2, scale=scale, dout=do)
        out, lse = sq.window_attention(plan, qq, k, v, 90, 2, scale=scale)
        ref.assert_within(out, want["out"], "out")
        ref.assert_within(lse, want["lse"], "lse")
        for name, x in zip(("dq", "dk", "dv"), sq.window_attention_grad(plan, qq, k, v, out, lse, do, 90, 2, scale=scale)):
            if scale == 0.0 or name == "dv":
                ref.assert_within(x, want[name], name)
            else:
                assert torch.isfinite(x).all()


def test_autograd_refuses_capture(cuda):
    """Outside a graph it works before and after; nothing has been enqueued when it is refused."""
    from f3m_b200 import sequence as sq
    plan, ld = sq.SequencePlan([64]), torch.tensor([-0.1], device="cuda")
    x = normal(1, 64, 1, 64, dtype=torch.bfloat16).requires_grad_()
    eager = sq.window_attention(plan, x, x, x, 10)[0]
    for call in (lambda: sq.window_attention(plan, x, x, x, 10), lambda: sq.decay_attention(plan, x, x, x, ld)):
        g = torch.cuda.CUDAGraph()
        keep = torch.zeros(1, device="cuda")
        with torch.cuda.graph(g):
            keep += 1
            with pytest.raises(RuntimeError, match="captured"):
                call()
    eager.sum().backward()
    assert x.grad is not None


def test_another_stream(cuda):
    from f3m_b200 import sequence as sq
    lengths, h, w = [1000, 24], 4, 128
    n = sum(lengths)
    plan, ld = sq.SequencePlan(lengths), torch.full((h,), -0.02, device="cuda")
    q, k, v, do = (normal(i, n, h, w, dtype=torch.bfloat16) for i in range(4))

    def both():
        out, lse = sq.window_attention(plan, q, k, v, 300, 3)
        a = sq.window_attention_grad(plan, q, k, v, out, lse, do, 300, 3)
        o, f = sq.decay_attention(plan, q, k, v, ld)
        return (out, lse, o, f) + a + sq.decay_attention_grad(plan, q, k, v, ld, do)

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(both())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want))


def test_empty_batches(cuda):
    from f3m_b200 import sequence as sq
    e = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    ld = torch.zeros(2, device="cuda")
    state = normal(1, 2, 2, 64, 64, dtype=torch.float32)
    for plan in (sq.SequencePlan([]), sq.SequencePlan([0, 0])):
        out, lse = sq.window_attention(plan, e, e, e, 5)
        assert out.shape == e.shape and lse.shape == (2, 0)
        assert all(x.shape == e.shape for x in sq.window_attention_grad(plan, e, e, e, out, lse, e, 5))
        s = state if plan.sequences else None
        out, final = sq.decay_attention(plan, e, e, e, ld, s)
        assert out.shape == e.shape and (s is None or torch.equal(final, s))
        d = sq.decay_attention_grad(plan, e, e, e, ld, e, s, s)[3]
        assert s is None or torch.equal(d, s)
    _, final = sq.decay_attention(sq.SequencePlan([0, 0]), e, e, e, ld)
    assert not final.any()
    assert sq.window_attention_step(e, e[:, None], e[:, None], torch.empty(0, device="cuda", dtype=torch.int32), 4).shape == e.shape
    z = sq.window_attention_step(torch.ones(3, 2, 64, device="cuda", dtype=torch.float16), *[torch.empty(3, 0, 1, 64, device="cuda", dtype=torch.float16)] * 2,
                                 torch.ones(3, device="cuda", dtype=torch.int32), 4)
    assert z.shape == (3, 2, 64) and not z.any()
    assert sq.decay_attention_step(e, e, e, ld, torch.empty(0, 2, 64, 64, device="cuda")).shape == e.shape


def test_refusals(cuda):
    from f3m_b200 import sequence as sq
    from f3m_b200._lib import F3MError
    plan = sq.SequencePlan([4])
    x = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    ld = torch.zeros(2, device="cuda")
    with pytest.raises(TypeError):
        sq.window_attention(plan, x.float(), x.float(), x.float(), 4)
    with pytest.raises(TypeError):
        sq.window_attention(plan, x, x.half(), x, 4)
    with pytest.raises(ValueError):
        sq.window_attention(plan, x[:3], x[:3], x[:3], 4)
    with pytest.raises(ValueError):
        sq.window_attention(plan, x, x.cpu(), x, 4)
    with pytest.raises(ValueError):
        sq.window_attention(plan, x, x, x, 0)
    with pytest.raises(ValueError):
        sq.window_attention(plan, x, x, x, 4, -1)
    with pytest.raises(ValueError):
        sq.window_attention(plan, x.repeat(1, 1, 3), x.repeat(1, 1, 3), x.repeat(1, 1, 3), 4)     # 192 columns
    with pytest.raises(ValueError):
        sq.window_attention(plan, x[..., :60], x[..., :60], x[..., :60], 4)
    with pytest.raises(ValueError):
        sq.window_attention(plan, x.repeat(1, 2, 1)[:, :3], x, x, 4)                              # 3 heads on 2
    with pytest.raises(F3MError):
        sq.window_attention(plan, x, x, x, 4, 0, float("nan"))
    with pytest.raises(RuntimeError):
        sq.decay_attention(plan, x, x, x, ld.clone().requires_grad_())
    with pytest.raises(TypeError):
        sq.decay_attention(plan, x, x, x, ld.double())
    with pytest.raises(ValueError):
        sq.decay_attention(plan, x, x, x, ld, torch.zeros(2, 2, 64, 64, device="cuda"))
    with pytest.raises(TypeError):
        sq.decay_attention_step(x, x, x, ld, torch.zeros(4, 2, 64, 64, device="cuda", dtype=torch.float64))
    with pytest.raises(TypeError):
        sq.decay_attention_step(x, x, x, ld, torch.zeros(4, 2, 64, 128, device="cuda")[..., ::2])
    with pytest.raises(TypeError):
        sq.window_attention_step(x, x[:, None], x[:, None], torch.ones(4, device="cuda"), 4)
    with pytest.raises(RuntimeError):
        sq.decay_attention_step(x.clone().requires_grad_(), x, x, ld, torch.zeros(4, 2, 64, 64, device="cuda"))
    with pytest.raises(ValueError):
        sq.window_attention_step(x, torch.zeros(4, 9, 2, 65, device="cuda", dtype=torch.bfloat16)[..., 1:], torch.zeros(4, 9, 2, 64, device="cuda", dtype=torch.bfloat16),
                                 torch.ones(4, device="cuda", dtype=torch.int32), 4)
