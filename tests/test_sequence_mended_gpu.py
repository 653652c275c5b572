"""Kernel products over sequences: repeated calls at uneven widths, batches of very uneven lengths, small gradients, values that are not numbers."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def normal(seed, *shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


@pytest.mark.parametrize("width_k,width_v", [(128, 64), (64, 128), (128, 128), (128, 8), (64, 64)])
def test_many_calls_of_attention_with_a_decay(width_k, width_v, cuda):
    """The weights of a tile may be ready before the products ask for those of the tile before, most easily where width_v is small and width_k
    is not: the same bits from call to call, and no wait runs out."""
    from f3m_b200 import sequence as sq
    lengths, h = [6000, 1, 2300, 130], 16
    n = sum(lengths)
    q, k = normal(1, n, h, width_k, dtype=torch.bfloat16), normal(2, n, h, width_k, dtype=torch.bfloat16)
    v, do = normal(3, n, h, width_v, dtype=torch.bfloat16), normal(4, n, h, width_v, dtype=torch.bfloat16)
    state, dfinal = (normal(5 + i, len(lengths), h, width_k, width_v, dtype=torch.float32) for i in range(2))
    ld = -torch.exp2(-torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / 2)
    plan = sq.SequencePlan(lengths)

    def calls():
        return sq.decay_attention(plan, q, k, v, ld, state) + sq.decay_attention_grad(plan, q, k, v, ld, do, state, dfinal)

    first = calls()
    for _ in range(100):
        assert all(torch.equal(x, y) for x, y in zip(calls(), first))
    want = ref.decay(q[:, :1], k[:, :1], v[:, :1], ld[:1].tolist(), lengths, state[:, :1], dout=do[:, :1], dfinal=dfinal[:, :1])
    for name, x in zip(("out", "final", "dq", "dk", "dv", "dstate"), first):
        ref.assert_within(x[:, :1], want[name], name)
