"""The router and the 4-bit products at their limits: offsets beyond 32 bits, rows that overlap, many tiles a
CTA, one and 1024 experts, and a first call that is being captured. Tolerances as in test_w4_gpu.py."""

import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

from minisgl import ops  # noqa: E402
from test_w4_gpu import (DEV, _check_experts, _check_linear, _check_route, _codes, _cuda_only,  # noqa: E402,F401
                               _experts_case, _experts_wide, _packed)


@pytest.mark.parametrize("M", [2, 12, 17, 40])
@pytest.mark.parametrize("step", [0, 8, 64])
def test_linear_rows_overlap(M, step):
    """One row for all, and windows that share inputs."""
    q, s, z = _codes((112, 256), 64, True)
    w = ops.W4Weight.pack(q, s, z)
    x = torch.randn(step * M + 256, device=DEV).to(torch.bfloat16).as_strided((M, 256), (step, 1))
    assert torch.equal(ops.linear_w4(x, w), ops.linear_w4(x.clone(memory_format=torch.contiguous_format), w))


@pytest.mark.parametrize("M,N,K", [(3001, 4000, 416), (700, 33, 256), (208, 2048, 1024), (224, 2048, 1024), (624, 34816, 256),
                                   (1021, 64, 1152)])
def test_linear_many_tiles(M, N, K):
    q, s, z = _codes((N, K), 32, False)
    x = torch.randn(M, K, device=DEV).to(torch.bfloat16)
    bias = torch.randn(N, device=DEV).to(torch.bfloat16)
    _check_linear(x, q, s, z, bias, ops.linear_w4(x, ops.W4Weight.pack(q, s, z), bias))


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (20, 1, 1), (3, 1024, 6), (1100, 1024, 8), (4000, 4, 3)])
def test_experts_few_and_many(T, E, k):
    """One expert, 1024 of them, many tiles a CTA."""
    H, inter = 128, 64
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    c1, c2 = _codes((E, 2 * inter, H), 64, False), _codes((E, H, inter), 32, False)
    ids = torch.randint(0, E, (T, k), device=DEV, dtype=torch.int32)
    weights = torch.rand(T, k, device=DEV)
    _check_experts(ops.experts_w4(x, *_packed(c1, c2), weights, ids), *_experts_wide(x, c1, c2, weights, ids))


@pytest.mark.parametrize("T", [1, 2, 4, 5])
@pytest.mark.parametrize("E", [5, 8, 20])
@pytest.mark.parametrize("chosen", [1, 2, 5])
def test_experts_around_a_warp_of_pairs(T, E, chosen):
    """8 to 40 pairs of a few experts: as many as a pass takes, and more."""
    x, c1, c2, _, _ = _experts_case(T, E, 1, 128, 64, 64, 32, False)
    ids = torch.randint(0, chosen, (T, 8), device=DEV, dtype=torch.int32) * 2 % E
    weights = torch.rand(T, 8, device=DEV)
    _check_experts(ops.experts_w4(x, *_packed(c1, c2), weights, ids), *_experts_wide(x, c1, c2, weights, ids))


@pytest.mark.parametrize("T", [2, 300])
def test_experts_all_elsewhere(T):
    x, c1, c2, weights, ids = _experts_case(T, 4, 2, 128, 64, 32, 32, False)
    assert not ops.experts_w4(x, *_packed(c1, c2), weights, ids, expert_offset=100).any()


@pytest.mark.parametrize("T", [6, 150])
def test_experts_tokens_are_apart(T):
    x, c1, c2, weights, ids = _experts_case(T, 4, 2, 256, 128, 64, 64, False)
    w1, w2 = _packed(c1, c2)
    clean = ops.experts_w4(x, w1, w2, weights, ids)
    x[1, 3], x[4, 200] = float("nan"), float("inf")
    got = ops.experts_w4(x, w1, w2, weights, ids)
    keep = [i for i in range(T) if i not in (1, 4)]
    assert torch.equal(got[keep], clean[keep]) and bool(got[1].isnan().all())


def test_offsets_beyond_32_bits():
    """Rows 2^31 and more elements behind the first one."""
    step = 2 ** 27 + 8
    big = torch.empty(20 * step, device=DEV, dtype=torch.bfloat16)
    x = big.as_strided((20, 256), (step, 1))
    x.normal_()
    q, s, z = _codes((112, 256), 64, True)
    w = ops.W4Weight.pack(q, s, z)
    for rows in (x, x[4:]):
        assert torch.equal(ops.linear_w4(rows, w), ops.linear_w4(rows.contiguous(), w))
    _check_route(x, 8)
    c1, c2 = _codes((3, 64, 256), 64, False), _codes((3, 128, 32), 32, False)
    w1, w2 = _packed(c1, c2)
    for rows in (x, x[8:]):  # 40 pairs of three experts, and 24
        weights, ids = ops.route_experts(torch.randn(rows.shape[0], 3, device=DEV), 2)
        assert torch.equal(ops.experts_w4(rows, w1, w2, weights, ids), ops.experts_w4(rows.contiguous(), w1, w2, weights, ids))


@pytest.mark.parametrize("T", [1, 1100])
def test_weights_beyond_4_gb(T):
    """The last of 1024 experts of 4 and 2 MB."""
    E, H, inter, k = 1024, 2048, 2048, 8
    c1, c2 = _codes((1, 2 * inter, H), 128, False), _codes((1, H, inter), 128, False)
    one = _packed(c1, c2)
    full = []
    for w in one:
        data = torch.zeros(E, *w.data.shape[1:], device=DEV, dtype=torch.uint8)
        data[E - 1] = w.data[0]
        full.append(ops.W4Weight(data, w.n, w.k, w.group, w.zeros, w.scale_dtype, w.gated, True))
    assert full[0].nbytes() > 2 ** 32
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    weights = torch.rand(T, k, device=DEV)
    ids = torch.full((T, k), E - 1, device=DEV, dtype=torch.int32)
    want = ops.experts_w4(x, *one, weights, torch.zeros_like(ids))
    assert bool(want.any())
    _check_experts(ops.experts_w4(x, *full, weights, ids), *_experts_wide(x, c1, c2, weights, torch.zeros_like(ids)))


_FIRST = """
import torch
from minisgl import ops
def weight(shape, gated=False):
    q = torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,), dtype=torch.uint8, device="cuda")
    return ops.W4Weight.pack(q, torch.rand(shape[:-1] + (shape[-1] // 64,), device="cuda").bfloat16(), gated=gated)
w, w1, w2 = weight((320, 512)), weight((4, 256, 512), True), weight((4, 512, 128))
x, logits = torch.randn(64, 512, device="cuda").bfloat16(), torch.randn(64, 4, device="cuda")
def run():
    out = []
    for t in (4, 12, 64):
        weights, ids = ops.route_experts(logits[:t], 2)
        out += [weights, ops.linear_w4(x[:t], w), ops.experts_w4(x[:t], w1, w2, weights, ids)]
    return out
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
print("as captured")
"""


def test_first_call_captured():
    done = subprocess.run([sys.executable, "-c", _FIRST], capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and "as captured" in done.stdout, done.stderr[-2000:]
