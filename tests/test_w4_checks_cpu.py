"""What the router and the 4-bit products accept and refuse on CPU tensors: the same as on the GPU."""

import pytest
import torch

from minisgl import ops


def _weight(shape, group=32, gated=False):
    gen = torch.Generator().manual_seed(sum(shape))
    q = torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,), generator=gen, dtype=torch.uint8)
    s = torch.rand(shape[:-1] + (shape[-1] // group,), generator=gen) * 0.02
    return ops.W4Weight.pack(q, s.to(torch.bfloat16), gated=gated)


def test_num_experts_is_an_estimate_only():
    w1, w2 = _weight((4, 64, 128), gated=True), _weight((4, 128, 32))
    x, wt = torch.randn(5, 128).to(torch.bfloat16), torch.rand(5, 2)
    ids = torch.randint(0, 16, (5, 2), dtype=torch.int32)
    want = ops.experts_w4(x, w1, w2, wt, ids, expert_offset=8)
    for n in (4, 16, 10 ** 6):
        assert torch.equal(ops.experts_w4(x, w1, w2, wt, ids, expert_offset=8, num_experts=n), want)
    with pytest.raises(ValueError, match="num_experts"):
        ops.experts_w4(x, w1, w2, wt, ids, num_experts=3)
