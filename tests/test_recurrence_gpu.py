"""The gated recurrence against its definition in 64 bits (recurrence_reference.py says how the bounds come about)."""
import pytest
import torch

import recurrence_reference as ref
from sequence_reference import assert_within

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def inputs(seed, tokens, channels, dtype, slow=1e-3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, channels, device="cuda", generator=g)
    rate = slow ** torch.rand(channels, device="cuda", generator=g)
    ld = -rate * torch.sigmoid(torch.randn(tokens, channels, device="cuda", generator=g))
    return x.to(dtype), ld.to(dtype)


def states(seed, n, channels):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, channels, device="cuda", generator=g)


def check(lengths, x, ld, state=None, do=None, dfinal=None):
    from f3m_b200 import sequence as sq
    plan = sq.SequencePlan(lengths)
    want = ref.recurrence(x, ld, lengths, state, do, dfinal)
    out, final = sq.gated_recurrence(plan, x, ld, state)
    assert_within(out, want["out"], "out")
    assert_within(final, want["final"], "final")
    if do is not None:
        for name, y in zip(("dx", "dlog", "dstate"), sq.gated_recurrence_grad(plan, ld, out, do, state, dfinal)):
            assert_within(y, want[name], name)


# lengths around a tile, its parts and several of them; few channels, odd multiples of 8, more than a block's
SIZES = [
    ([1], 8),
    ([129], 64),
    ([0, 3, 0], 72),
    ([16, 17, 15, 1, 0, 31, 33, 127], 40),
    ([128, 256, 257, 1], 136),
    ([700, 1, 900], 264),
    ([2500], 16),
    ([300], 2056),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,channels", SIZES)
def test_recurrence_and_gradients(lengths, channels, dtype, cuda):
    n = sum(lengths)
    x, ld = inputs(1, n, channels, dtype)
    do = inputs(2, n, channels, dtype)[0]
    check(lengths, x, ld, None, do)
    check(lengths, x, ld, states(3, len(lengths), channels), do, states(4, len(lengths), channels))


@pytest.mark.parametrize("dtype", TYPES)
def test_recurrence_of_views(dtype, cuda):
    """Columns of a joint projection, a broadcast decay, rows that start off 16 bytes."""
    lengths, c = [200, 131], 48
    n = sum(lengths)
    joint = torch.cat(inputs(5, n, c, dtype) + inputs(6, n, c, dtype), 1)
    x, ld, do = joint[:, :c], joint[:, c:2 * c], joint[:, 2 * c:3 * c]
    check(lengths, x, ld, None, do)
    check(lengths, x, ld[:, :1].expand(n, c), None, do)
    check(lengths, x, ld[:1].expand(n, c), None, do[:1].expand(n, c))
    flat = torch.cat([x.reshape(-1)[:1], x.reshape(-1)])
    check(lengths, flat[1:].view(n, c), ld, None, do)


@pytest.mark.parametrize("dtype", TYPES)
def test_decays_at_their_ends(dtype, cuda):
    """No decay, none above 0, no memory at all, tiny and huge ones side by side; gradients are 0 where the decay is held at 0."""
    n, c = 400, 32
    x, ld = inputs(7, n, c, dtype)
    ld[:, 0], ld[:, 1], ld[:, 2], ld[:, 3] = 0.0, 0.5, float("-inf"), -1e-4
    ld[::50, 4], ld[::7, 5], ld[::3, 6], ld[:, 7] = float("-inf"), -30.0, 2.0, -0.5
    ld[:, 8], ld[:, 9] = -0.25, -80.0
    if dtype == torch.float16:      # sums without decay stay in fp16's range
        x *= 0.125
    check([n], x, ld, states(8, 1, c), inputs(9, n, c, dtype)[0], states(10, 1, c))


def test_long_sums_next_to_no_decay(cuda):
    """Sums over ten thousand tokens keep their bits where each decay is next to 1."""
    n, c = 10000, 8
    x = inputs(11, n, c, torch.float32)[0] + 1.0
    ld = torch.full((n, c), -1.3e-4, device="cuda")
    check([n], x, ld)


def test_a_sequence_does_not_reach_its_neighbours(cuda):
    from f3m_b200 import sequence as sq
    lengths, c = [100, 60, 300], 64
    plan = sq.SequencePlan(lengths)
    x, ld = inputs(12, sum(lengths), c, torch.bfloat16)
    do, st = inputs(13, sum(lengths), c, torch.bfloat16)[0], states(14, 3, c)
    keep = torch.ones(sum(lengths), dtype=torch.bool, device="cuda")
    keep[100:160] = False
    bad = [y.clone() for y in (x, ld, do)]
    for y in bad:
        y[100:160] = float("nan")
    st2 = st.clone()
    st2[1] = float("inf")
    a, b = sq.gated_recurrence(plan, x, ld, st), sq.gated_recurrence(plan, bad[0], bad[1], st2)
    assert torch.equal(a[0][keep], b[0][keep]) and torch.equal(a[1][[0, 2]], b[1][[0, 2]])
    assert b[0][100:160].isnan().all() and b[1][1].isnan().all()
    ga, gb = sq.gated_recurrence_grad(plan, ld, a[0], do, st, st), sq.gated_recurrence_grad(plan, bad[1], b[0], bad[2], st2, st2)
    for y, z in zip(ga[:2], gb[:2]):
        assert torch.equal(y[keep], z[keep])
    assert torch.equal(ga[2][[0, 2]], gb[2][[0, 2]])


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_a_number_goes_on_and_not_back(dtype, cuda):
    from f3m_b200 import sequence as sq
    n, c, at = 700, 24, 391
    plan = sq.SequencePlan([n])
    x, ld = inputs(15, n, c, dtype)
    do = inputs(16, n, c, dtype)[0]
    out, final = sq.gated_recurrence(plan, x, ld)
    for what in (x, ld):
        y = [z.clone() for z in (x, ld)]
        y[0 if what is x else 1][at, 5] = float("nan")
        o, f = sq.gated_recurrence(plan, *y)
        assert torch.equal(o[:at], out[:at]) and o[at:, 5].isnan().all() and f[0, 5].isnan()
        rest = [i for i in range(c) if i != 5]
        assert torch.equal(o[:, rest], out[:, rest]) and torch.equal(f[:, rest], final[:, rest])
    d = do.clone()
    d[at, 5] = float("nan")
    a, b = sq.gated_recurrence_grad(plan, ld, out, do), sq.gated_recurrence_grad(plan, ld, out, d)
    assert torch.equal(a[0][at + 1:], b[0][at + 1:]) and b[0][:at + 1, 5].isnan().all() and b[2][0, 5].isnan()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,channels", [(1, 8), (3, 72), (257, 1032)])
def test_step(n, channels, dtype, cuda):
    """As many steps as a prompt has tokens: the prompt's outputs and state."""
    from f3m_b200 import sequence as sq
    tokens = 3
    x, ld = inputs(17, n * tokens, channels, dtype)
    ld[0], ld[1, 0] = 0.25, float("-inf")
    st = states(18, n, channels)
    want = ref.recurrence(x, ld, [tokens] * n, st)
    for t in range(tokens):
        out = sq.gated_recurrence_step(x[t::tokens], ld[t::tokens], st)
        assert_within(out, tuple(y[t::tokens] for y in want["out"]), f"token {t}")
    assert_within(st, want["final"], "state")


def test_autograd(cuda):
    """Gradients of the formula, and against differences of the definition in 64 bits."""
    from f3m_b200 import sequence as sq
    lengths, c = [50, 1, 200], 16
    plan = sq.SequencePlan(lengths)
    x, ld = inputs(19, sum(lengths), c, torch.float32)
    st = states(20, 3, c)
    leaves = [t.clone().requires_grad_(True) for t in (x, ld, st)]
    out, final = sq.gated_recurrence(plan, *leaves)
    do, df = inputs(21, sum(lengths), c, torch.float32)[0], states(22, 3, c)
    ((out * do).sum() + (final * df).sum()).backward()
    want = ref.recurrence(x, ld, lengths, st, do, df)
    for name, t in zip(("dx", "dlog", "dstate"), leaves):
        assert_within(t.grad, want[name], name)

    def loss(x, ld, st):
        w = ref.recurrence(x, ld, lengths, st)
        return float((w["out"][0] * do).sum() + (w["final"][0] * df).sum())

    base = [x.double(), ld.double(), st.double()]
    for i, t in enumerate(leaves):
        along = torch.randn(t.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(23 + i), dtype=torch.float64)
        if i == 1:
            along *= ld.double()         # decays stay below 0
        step = 1e-5
        up, down = ([y + (s * step * along if j == i else 0) for j, y in enumerate(base)] for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / (2 * step)
        # the gradient's own bounds, and what a difference leaves: its third term, some 1e-10 of sums of a few thousand terms
        bound = float((along.abs() * want[("dx", "dlog", "dstate")[i]][1]).sum()) + 1e-5 * float((along * t.grad).abs().sum())
        assert abs(slope - float((along * t.grad).sum())) <= bound


def test_gradients_that_nobody_asked_for(cuda):
    """Only out, only the state is used; no state is given; part of the inputs need none."""
    from f3m_b200 import sequence as sq
    plan, c = sq.SequencePlan([40, 9]), 8
    x, ld = inputs(24, 49, c, torch.float32)
    for use in (0, 1):
        a, b = x.clone().requires_grad_(True), ld.clone().requires_grad_(True)
        sq.gated_recurrence(plan, a, b)[use].sum().backward()
        do, df = (torch.ones_like(x), None) if use == 0 else (torch.zeros_like(x), torch.ones(2, c, device="cuda"))
        want = ref.recurrence(x, ld, [40, 9], None, do, df)
        assert_within(a.grad, want["dx"])
        assert_within(b.grad, want["dlog"])
    b = ld.clone().requires_grad_(True)
    sq.gated_recurrence(plan, x, b)[0].sum().backward()
    assert_within(b.grad, ref.recurrence(x, ld, [40, 9], None, torch.ones_like(x))["dlog"])


@pytest.mark.parametrize("dtype", TYPES)
def test_calls_repeat_and_replay(dtype, cuda):
    """The same bits again, on another stream, and from a captured graph with other inputs in place; two graphs at once."""
    from f3m_b200 import sequence as sq
    lengths, c = [3000, 77, 1500], 264
    n = sum(lengths)
    plan = sq.SequencePlan(lengths)
    data = [(*inputs(30 + i, n, c, dtype), inputs(40 + i, n, c, dtype)[0], states(50 + i, 3, c)) for i in range(2)]

    def run(x, ld, do, st):
        out, final = sq.gated_recurrence(plan, x, ld, st)
        return (out, final) + sq.gated_recurrence_grad(plan, ld, out, do, st, st)

    first = [run(*d) for d in data]
    for _ in range(20):
        for a, b in zip(run(*data[0]), first[0]):
            assert torch.equal(a, b)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    held = [[t.clone() for t in data[0]] for _ in side]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for s, h in zip(side, held):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(run(*h))
        graphs.append(g)
    for h, d in zip(held, (data[1], data[0])):
        for a, b in zip(h, d):
            a.copy_(b)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, want in zip(outs, (first[1], first[0])):
        for a, b in zip(o, want):
            assert torch.equal(a, b)


def test_captured_autograd_is_refused(cuda):
    from f3m_b200 import sequence as sq
    plan = sq.SequencePlan([20])
    x, ld = inputs(60, 20, 8, torch.float32)
    x.requires_grad_(True)
    sq.gated_recurrence(plan, x, ld)[0].sum().backward()
    refused = []
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        try:
            sq.gated_recurrence(plan, x, ld)
        except RuntimeError as e:
            refused.append(str(e))
    assert refused and "captured" in refused[0]


def test_refusals(cuda):
    from f3m_b200 import sequence as sq
    plan = sq.SequencePlan([20])
    x, ld = inputs(61, 20, 16, torch.bfloat16)
    st = states(62, 1, 16)
    for call in (lambda: sq.gated_recurrence(plan, x[:19], ld[:19]), lambda: sq.gated_recurrence(plan, x[:, :12], ld[:, :12]), lambda: sq.gated_recurrence(plan, x[None], ld[None]),
                 lambda: sq.gated_recurrence(plan, x, ld[:19]), lambda: sq.gated_recurrence(plan, x, ld, st[:, :8]), lambda: sq.gated_recurrence_grad(plan, ld, x, x, dfinal=st[0]),
                 lambda: sq.gated_recurrence(plan, x, ld.cpu())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: sq.gated_recurrence(plan, x, ld.float()), lambda: sq.gated_recurrence(plan, x.double(), ld.double()), lambda: sq.gated_recurrence(plan, x, ld, st.double()),
                 lambda: sq.gated_recurrence_step(x[:1], ld[:1], st.half()), lambda: sq.gated_recurrence_step(x[:2], ld[:2], states(62, 2, 16).t().contiguous().t())):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError):
        sq.gated_recurrence_step(x[:1], ld[:1], st.clone().requires_grad_(True))


def test_arrays_behind_two_billion_elements(cuda):
    """The last sequence of arrays of more than 2^31 elements: the bits it has by itself."""
    from f3m_b200 import sequence as sq
    c, last = 8192, 200
    n = (1 << 31) // c + 300
    x, ld = torch.zeros(n, c, device="cuda", dtype=torch.bfloat16), torch.full((n, c), -1.0, device="cuda", dtype=torch.bfloat16)
    a, b = inputs(63, last, c, torch.bfloat16)
    x[-last:], ld[-last:] = a, b
    plan, alone = sq.SequencePlan([n - last, last]), sq.SequencePlan([last])
    out, final = sq.gated_recurrence(plan, x, ld)
    o, f = sq.gated_recurrence(alone, a, b)
    assert torch.equal(out[-last:], o) and torch.equal(final[1], f[0])
    del x
    dx, dl, ds = sq.gated_recurrence_grad(plan, ld, out, out)
    gx, gl, gs = sq.gated_recurrence_grad(alone, b, o, o)
    assert torch.equal(dx[-last:], gx) and torch.equal(dl[-last:], gl) and torch.equal(ds[1], gs[0])
