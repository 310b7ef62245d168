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


def bad_calls(dev):
    """(name, call) of what both forms refuse, before anything is copied or launched"""
    logits = torch.randn(2, 512, device=dev)
    zeros = lambda *shape, dtype=torch.float32: torch.zeros(*shape, device=dev, dtype=dtype)  # noqa: E731
    w, w1, w2 = (t.to(dev) for t in (_weight((32, 128)), _weight((4, 64, 128), gated=True), _weight((4, 128, 32))))
    many1, many2 = _weight((1025, 64, 32), gated=True).to(dev), _weight((1025, 32, 32)).to(dev)
    x, wt, ids = zeros(4, 128, dtype=torch.bfloat16), zeros(4, 2), zeros(4, 2, dtype=torch.int32)
    long = zeros(2 ** 23, 2, dtype=torch.int32)
    route, linear, experts = ops.route_experts, ops.linear_w4, ops.experts_w4
    bf16 = torch.bfloat16
    return [
        ("513 experts", lambda: route(zeros(2, 513), 2)),
        ("no experts", lambda: route(zeros(2, 0), 1)),
        ("512 groups", lambda: route(logits, 2, num_groups=512, top_groups=2)),
        ("no groups", lambda: route(logits, 2, num_groups=0)),
        ("negative groups", lambda: route(logits, 2, num_groups=-2, top_groups=-2)),
        ("no group kept", lambda: route(logits, 2, num_groups=4, top_groups=0)),
        ("none chosen", lambda: route(logits, 0)),
        ("33 chosen", lambda: route(logits, 33)),
        ("a bias in 64 bits", lambda: route(logits, 2, bias=zeros(512, dtype=torch.float64))),
        ("a strided bias", lambda: route(logits, 2, bias=zeros(1024)[::2])),
        ("2^31 rows", lambda: route(zeros(1, 1).expand(2 ** 31, 1), 1)),
        ("x in 32 bits", lambda: linear(x.float(), w)),
        ("a linear bias in 32 bits", lambda: linear(x, w, zeros(32))),
        ("a short linear bias", lambda: linear(x, w, zeros(31, dtype=bf16))),
        ("a strided linear bias", lambda: linear(x, w, zeros(64, dtype=bf16)[::2])),
        ("2^30 tokens", lambda: linear(x[:1].expand(2 ** 30, 128), w)),
        ("experts' x in 32 bits", lambda: experts(x.float(), w1, w2, wt, ids)),
        ("experts' x of one row", lambda: experts(x[0], w1, w2, wt, ids)),
        ("weights in 64 bits", lambda: experts(x, w1, w2, wt.double(), ids)),
        ("ids in 64 bits", lambda: experts(x, w1, w2, wt, ids.long())),
        ("weights turned", lambda: experts(x, w1, w2, wt.t().contiguous().t(), ids)),
        ("no choices", lambda: experts(x, w1, w2, wt[:, :0], ids[:, :0])),
        ("a negative offset", lambda: experts(x, w1, w2, wt, ids, expert_offset=-1)),
        ("w1_bias in 32 bits", lambda: experts(x, w1, w2, wt, ids, w1_bias=zeros(4, 64))),
        ("a short w2_bias", lambda: experts(x, w1, w2, wt, ids, w2_bias=zeros(4, 32, dtype=bf16))),
        ("1025 experts here", lambda: experts(x[:, :32].contiguous(), many1, many2, wt, ids)),
        ("2^24 pairs", lambda: experts(x[:1].expand(2 ** 23, 128), w1, w2, long.float(), long)),
        ("fewer in all than here", lambda: experts(x, w1, w2, wt, ids, num_experts=3)),
    ]


@pytest.mark.parametrize("name,call", bad_calls("cpu"), ids=lambda v: v if isinstance(v, str) else "")
def test_refused(name, call):
    with pytest.raises(ValueError):
        call()


def test_at_the_limits():
    logits = torch.randn(2, 512)
    assert ops.route_experts(logits, 32, num_groups=256, top_groups=16, bias=torch.zeros(1, 512))[1].shape == (2, 32)
    w1, w2 = _weight((1024, 64, 32), gated=True), _weight((1024, 32, 32))
    ids = torch.tensor([[0, 1023]], dtype=torch.int32)
    y = ops.experts_w4(torch.ones(1, 32, dtype=torch.bfloat16), w1, w2, torch.ones(1, 2), ids,
                       w1_bias=torch.zeros(1024, 64, dtype=torch.bfloat16), w2_bias=torch.ones(1024, 32, dtype=torch.bfloat16))
    assert y.shape == (1, 32) and bool(y.isfinite().all())


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("scales", [torch.bfloat16, torch.float16])
def test_quantize_refuses_scales_that_are_not_finite(symmetric, scales):
    """An infinite scale would make every weight of its group an infinity or NaN."""
    w = torch.randn(4, 128, generator=torch.Generator().manual_seed(7))
    for bad in (float("inf"), -float("inf"), float("nan"), 1e7 if scales == torch.float16 else None):
        if bad is None:
            continue
        v = w.clone()
        v[2, 77] = bad
        with pytest.raises(ValueError, match="scale"):
            ops.quantize_w4(v, 64, symmetric, scales)
    q, s, z = ops.quantize_w4(w * 1e4, 64, symmetric, scales)
    assert bool(ops.W4Weight.pack(q, s, z).dequant().isfinite().all())
    with pytest.raises(ValueError):
        ops.quantize_w4(w, 64, symmetric, torch.float32)


def test_launch_counts_come_from_the_call():
    from types import SimpleNamespace

    from minisgl._native import _CountingModule
    from minisgl.engine.counters import COUNTERS

    mod = _CountingModule(SimpleNamespace(linear_w4=lambda m: ("y", m), experts_w4=lambda m: ("z", m + 2),
                                          route_experts=lambda: "r"))
    before = COUNTERS.launches
    assert mod.linear_w4(2) == "y" and COUNTERS.launches == before + 2
    assert mod.linear_w4(0) == "y" and COUNTERS.launches == before + 2
    assert mod.experts_w4(2) == "z" and COUNTERS.launches == before + 6
    assert mod.route_experts() == "r" and COUNTERS.launches == before + 7


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pack_refuses_scales_that_are_not_finite(dtype):
    q = torch.zeros(3, 64, dtype=torch.uint8)
    for bad in (float("inf"), -float("inf"), float("nan")):
        s = torch.ones(3, 4, dtype=dtype)
        s[1, 2] = bad
        with pytest.raises(ValueError, match="finite"):
            ops.W4Weight.pack(q, s)
