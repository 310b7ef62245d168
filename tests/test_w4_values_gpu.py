"""The 4-bit products and the router at values that a sum, a clamp or a bound on errors could lose."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from minisgl import ops  # noqa: E402
from test_w4_gpu import DEV, _codes, _cuda_only, _experts_case, _packed  # noqa: E402,F401


# 12 and 16 pairs of 4 experts: the streaming product; 300: the tensor core
@pytest.mark.parametrize("T", [6, 8, 150])
@pytest.mark.parametrize("activation", ["silu", "gelu", "swiglu_oai"])
def test_nan_stays_in_sight(T, activation):
    """A NaN among a token's inputs is in all of its row of the result, and in no other."""
    x, c1, c2, weights, ids = _experts_case(T, 4, 2, 256, 128, 64, 64, False)
    w1, w2 = _packed(c1, c2)
    clean = ops.experts_w4(x, w1, w2, weights, ids, activation=activation)
    x[1, 3] = float("nan")
    got = ops.experts_w4(x, w1, w2, weights, ids, activation=activation)
    assert bool(got[1].isnan().all())
    keep = [i for i in range(T) if i != 1]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("T", [6, 150])
@pytest.mark.parametrize("row", [5, 128 + 5])
@pytest.mark.parametrize("activation", ["silu", "gelu", "swiglu_oai"])
def test_nan_of_one_side(T, row, activation):
    """A NaN in the gate alone, and in the other factor alone (through a bias of one expert)."""
    x, c1, c2, weights, ids = _experts_case(T, 4, 2, 256, 128, 64, 64, False)
    b1 = torch.zeros(4, 256, device=DEV, dtype=torch.bfloat16)
    b1[2, row] = float("nan")
    got = ops.experts_w4(x, *_packed(c1, c2), weights, ids, activation=activation, w1_bias=b1)
    hit = (ids == 2).any(dim=1)
    assert bool(hit.any()) and not bool(hit.all())
    assert torch.equal(got.isnan(), hit[:, None].expand_as(got))


@pytest.mark.parametrize("T", [6, 150])
def test_infinite_factors_are_clamped(T):
    """+inf is 7 for the gate, both infinities are 7 of their sign for the other factor."""
    x, c1, c2, weights, ids = _experts_case(T, 4, 2, 256, 128, 64, 64, False)
    w1, w2 = _packed(c1, c2)
    b1 = torch.zeros(4, 256, device=DEV, dtype=torch.bfloat16)
    b1[:, 9], b1[:, 128 + 9], b1[:, 128 + 40] = float("inf"), float("inf"), -float("inf")
    far = b1.clamp(-1e30, 1e30)
    assert torch.equal(ops.experts_w4(x, w1, w2, weights, ids, activation="swiglu_oai", w1_bias=b1),
                       ops.experts_w4(x, w1, w2, weights, ids, activation="swiglu_oai", w1_bias=far))


def test_route_most_tokens():
    """As many tokens as a call takes: the last ones' numbers plus a grid's warps are beyond 31 bits."""
    T = 2 ** 31 - 1
    weights, ids = ops.route_experts(torch.ones(1, 1, device=DEV, dtype=torch.bfloat16).expand(T, 1), 1)
    assert ids.shape == (T, 1)
    assert not bool(ids.any()) and bool((weights == 1).all())
    with pytest.raises((RuntimeError, ValueError)):
        ops.route_experts(torch.ones(1, 1, device=DEV).expand(T + 1, 1), 1)
