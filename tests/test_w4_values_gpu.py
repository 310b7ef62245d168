"""The 4-bit products and the router at values that a sum, a clamp or a bound on errors could lose."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from minisgl import ops  # noqa: E402
from test_w4_gpu import (DEV, _check_experts, _check_linear, _check_route, _codes, _cuda_only,  # noqa: E402,F401
                         _experts_case, _experts_wide, _packed)


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


def _check_finite(got):
    assert bool(got.isfinite().all())


# With codes of up to 15 a group's sum before its scale passes the end of fp32 where the result does not
# come near it; at the other end a small unit of the codes must not lose a result that is still normal.
@pytest.mark.parametrize("M", [1, 7, 12, 16, 40, 200])
@pytest.mark.parametrize("power", [123, -110])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, False), (128, True)])
def test_linear_at_the_ends_of_the_range(M, power, group, zeros):
    q, s, z = _codes((160, 512), group, zeros)
    x = (torch.randn(M, 512, device=DEV) * 2.0 ** power).to(torch.bfloat16)
    got = ops.linear_w4(x, ops.W4Weight.pack(q, s, z))
    _check_finite(got)
    _check_linear(x, q, s, z, None, got)


def test_linear_largest_activations():
    """Every activation the largest bf16, every code 15 and its zero point 0; 2^-20 brings the result back."""
    big = torch.finfo(torch.bfloat16).max
    for M in (1, 9, 33):
        q = torch.full((48, 64), 255, device=DEV, dtype=torch.uint8)
        s = torch.full((48, 1), 2.0 ** -20, device=DEV, dtype=torch.bfloat16)
        got = ops.linear_w4(torch.full((M, 128), big, device=DEV, dtype=torch.bfloat16),
                            ops.W4Weight.pack(q, s, torch.zeros(48, 1, device=DEV, dtype=torch.uint8)))
        # bf16 has 8 bits: 128 * 15 * big * 2^-20 is (2 - 2^-7) * 15 * 2^114, rounded once
        assert bool((got == torch.tensor(128.0 * 15 * big * 2.0 ** -20, dtype=torch.float64).to(torch.bfloat16).item()).all())


@pytest.mark.parametrize("T", [3, 8, 60])
def test_experts_of_large_activations(T):
    """Activated values of about 2^122, results below 2^127."""
    x, c1, c2, weights, ids = _experts_case(T, 4, 2, 256, 256, 128, 128, False)
    x = (x.float() * 2.0 ** 60).to(torch.bfloat16)
    got = ops.experts_w4(x, *_packed(c1, c2), weights, ids)
    _check_finite(got)
    _check_experts(got, *_experts_wide(x, c1, c2, weights, ids))


@pytest.mark.parametrize("E,groups", [(32, 1), (96, 3), (256, 1), (256, 8), (512, 16), (300, 1)])
@pytest.mark.parametrize("values", [[-1e9], [-float("inf")], [float("nan"), -3e38], [1e9], [1e9, -1e9], [3e38, -3e38, -1e30]])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_biases_far_apart(E, groups, values, scoring):
    """Biases that mask experts or force them, for one expert, a few, most and all but three of them."""
    for many in (1, E // 8, E - E // 8, E - 3):
        bias = torch.randn(E, device=DEV) * 0.1
        at = torch.randperm(E, device=DEV)[:many]
        bias[at] = torch.tensor(values, device=DEV).repeat(many)[:many]
        logits = torch.randn(150, E, device=DEV) * 1.5
        for k in (1, 8):
            _check_route(logits, k, scoring=scoring, bias=bias)
            if groups > 1:
                for group_score in ("max", "top2"):
                    _check_route(logits, k, scoring=scoring, bias=bias, num_groups=groups, top_groups=max(1, groups // 2),
                                 group_score=group_score)


@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_route_whole_groups_masked(group_score):
    """Groups without an expert to choose are passed over, and chosen from when only they are left."""
    for mask in (-1e9, -float("inf")):
        bias = torch.randn(256, device=DEV) * 0.1
        bias[32:160] = mask
        for kept in (3, 4, 6):
            logits = torch.randn(200, 256, device=DEV)
            kw = dict(scoring="sigmoid", bias=bias, num_groups=8, top_groups=kept, group_score=group_score)
            _check_route(logits, 8, **kw)
            if kept <= 4:
                ids = ops.route_experts(logits, 8, **kw)[1]
                assert not bool(((ids >= 32) & (ids < 160)).any())
