"""4-bit weights and the expert router on CPU tensors: layout, plain forms and refusals."""

import pytest
import torch

from minisgl import ops


def _codes(gen, shape, group, zeros, dtype=torch.bfloat16):
    q = torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,), generator=gen, dtype=torch.uint8)
    side = shape[:-1] + (shape[-1] // group,)
    s = (torch.rand(side, generator=gen) * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 16, side, generator=gen, dtype=torch.uint8) if zeros else None
    return q, s, z


def _plain(q, s, z):
    """(code - zero) * scale, one value at a time along the inputs."""
    k = 2 * q.shape[-1]
    group = k // s.shape[-1]
    cols = []
    for i in range(k):
        code = (q[..., i // 2] >> (4 * (i % 2))) & 15
        zero = 8 if z is None else z[..., i // group].double()
        cols.append((code.double() - zero) * s[..., i // group].double())
    return torch.stack(cols, dim=-1)


@pytest.mark.parametrize("shape", [(16, 64), (1, 32), (37, 96), (48, 256), (3, 20, 128), (2, 6, 160)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_pack_keeps_the_weights(shape, zeros, gated):
    gen = torch.Generator().manual_seed(1)
    for group in (32, 64, 128):
        if shape[-1] % group or (gated and shape[-2] % 2):
            continue
        q, s, z = _codes(gen, shape, group, zeros)
        w = ops.W4Weight.pack(q, s, z, gated=gated)
        assert tuple(w.shape) == shape and w.group == group
        got = w.codes()
        assert torch.equal(got[0], q) and torch.equal(got[1], s)
        assert (z is None and got[2] is None) or torch.equal(got[2], z)
        # a product of a 4-bit integer and a 16-bit scale is exact in 32 bits
        assert torch.equal(w.dequant().double(), _plain(q, s, z))


def test_pack_layout():
    """The documented place of one code: tile, block, lane, word and nibble."""
    q = torch.zeros(64, 128, dtype=torch.uint8)
    row, k = 59, 239  # tile 1, half 1, row 11 = g 3 of its upper 8; record 1, block 1, word 2, t 3, last code
    q[row, k // 2] = 0xD0
    s = torch.zeros(64, 8, dtype=torch.bfloat16)
    s[row, k // 32] = 1.0
    z = torch.zeros(64, 8, dtype=torch.uint8)
    z[row, k // 32] = 5
    w = ops.W4Weight.pack(q, s, z)
    assert w.data.shape == (1, 2, 2, 2048 + 4 * 96) and w.data.count_nonzero() == 4  # 0xD, 1.0 = 0x3F80, 5
    rec = w.data[0, 1, 1]
    words = rec[:2048].view(torch.int32).view(2, 2, 32, 4)
    g, t, word, nibble = 3, 3, 2, 7
    assert (int(words[1, 1, 4 * g + t, word]) >> (4 * nibble)) & 15 == 0xD
    assert rec[2048:2304].view(torch.bfloat16).view(4, 8, 2, 2)[3, g, 1, 1] == 1.0
    assert rec[2304:].view(4, 8, 2, 2)[3, g, 1, 1] == 5


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize(symmetric):
    gen = torch.Generator().manual_seed(2)
    w = torch.randn(24, 256, generator=gen)
    w[3, :64] = 0.0
    q, s, z = ops.quantize_w4(w, 64, symmetric)
    assert (z is None) == symmetric
    back = ops.W4Weight.pack(q, s, z).dequant()
    # half a step, plus what rounding the scale moves the ends of the range by (15 steps x 2^-8 at most),
    # plus, with zero points, half a step more for the rounded zero point
    step = s.float().repeat_interleave(64, dim=1)
    bound = (0.5 if symmetric else 1.0) * step + 15 * 2.0 ** -8 * step + 1e-6
    assert bool(((back - w).abs() <= bound).all())
    assert bool((back[3, :64] == 0).all())


def test_linear_and_experts_plain_forms():
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(5, 96, generator=gen).to(torch.bfloat16)
    q, s, z = _codes(gen, (21, 96), 32, True, torch.float16)
    b = torch.randn(21, generator=gen).to(torch.bfloat16)
    y = ops.linear_w4(x, ops.W4Weight.pack(q, s, z), b)
    want = x.double() @ _plain(q, s, z).t() + b.double()
    torch.testing.assert_close(y.double(), want, atol=1e-4, rtol=2.0 ** -8)

    E, inter, H, T = 3, 32, 64, 7
    q1, s1, z1 = _codes(gen, (E, 2 * inter, H), 32, False)
    q2, s2, z2 = _codes(gen, (E, H, inter), 32, True)
    x = torch.randn(T, H, generator=gen).to(torch.bfloat16)
    weights, ids = ops.route_experts(torch.randn(T, 4, generator=gen), 2)
    y = ops.experts_w4(x, ops.W4Weight.pack(q1, s1, z1, gated=True), ops.W4Weight.pack(q2, s2, z2), weights, ids,
                       expert_offset=1)
    m1, m2 = _plain(q1, s1, z1), _plain(q2, s2, z2)
    want = torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for w, e in zip(weights[t].tolist(), ids[t].tolist()):
            if not 1 <= e <= E:
                continue
            h = m1[e - 1] @ x[t].double()
            a = torch.nn.functional.silu(h[:inter]) * h[inter:]
            want[t] += w * (m2[e - 1] @ a)
    torch.testing.assert_close(y.double(), want, atol=1e-4, rtol=2.0 ** -8)


def test_route_plain_form_by_hand():
    logits = torch.tensor([[0.0, 2.0, 2.0, -1.0, 5.0, 0.0]])
    w, ids = ops.route_experts(logits, 3, renormalize=False)
    assert ids.tolist() == [[4, 1, 2]]  # equal logits: the lower id first
    torch.testing.assert_close(w, torch.softmax(logits, -1)[:, [4, 1, 2]])
    # groups {0, 1}, {2, 3}, {4, 5}: the bias of expert 4 takes its group out
    bias = torch.tensor([0.0, 0.0, 0.0, 0.0, -3.0, 0.0])
    w, ids = ops.route_experts(logits, 2, scoring="sigmoid", bias=bias, num_groups=3, top_groups=2, group_score="top2",
                               scale=2.0)
    assert ids.tolist() == [[1, 2]]
    torch.testing.assert_close(w, torch.tensor([[1.0, 1.0]]))


def test_route_rows_without_anything_finite():
    inf = float("inf")
    logits = torch.tensor([[-inf] * 4, [float("nan")] * 4, [inf, inf, 0.0, -inf], [torch.finfo(torch.float32).min] * 4])
    w, ids = ops.route_experts(logits, 2)
    assert ids.tolist() == [[0, 1]] * 4
    assert w[:2].tolist() == [[0.0, 0.0]] * 2
    torch.testing.assert_close(w[2:], torch.full((2, 2), 0.5))


def test_refusals():
    q, s, _ = _codes(torch.Generator().manual_seed(4), (16, 64), 64, False)
    pack = ops.W4Weight.pack
    for bad in (
        lambda: pack(q.int(), s),                                  # codes' type
        lambda: pack(q, s.float()),                                # scales' type
        lambda: pack(q, s[:8]),                                    # rows differ
        lambda: pack(q[:, :24], s),                                # a group of 48
        lambda: pack(q[:, :8], s),                                 # a group of 16
        lambda: pack(q, s, torch.zeros(16, 2, dtype=torch.uint8)),  # zero points' shape
        lambda: pack(q, s, torch.full((16, 1), 16, dtype=torch.uint8)),
        lambda: pack(q[:15], s[:15], gated=True),                  # an odd number of gate and up rows
        lambda: pack(q[:0], s[:0]),
        lambda: ops.quantize_w4(torch.zeros(4, 96), 64),
        lambda: ops.linear_w4(torch.zeros(1, 64, dtype=torch.bfloat16), pack(q[None], s[None])),
        lambda: ops.experts_w4(torch.zeros(1, 64, dtype=torch.bfloat16), pack(q[None], s[None]), pack(q[None], s[None]),
                               torch.zeros(1, 1), torch.zeros(1, 1, dtype=torch.int32)),
        lambda: ops.route_experts(torch.zeros(2, 8), 9),
        lambda: ops.route_experts(torch.zeros(2, 8), 2, num_groups=3),
        lambda: ops.route_experts(torch.zeros(2, 8), 5, num_groups=2, top_groups=1),
        lambda: ops.route_experts(torch.zeros(2, 8), 1, num_groups=8, top_groups=2, group_score="top2"),
        lambda: ops.route_experts(torch.zeros(2, 8), 2, scoring="tanh"),
        lambda: ops.route_experts(torch.zeros(2, 8), 2, group_score="mean"),
    ):
        with pytest.raises(ValueError):
            bad()


def test_refusals_of_sizes():
    gen = torch.Generator().manual_seed(3)
    w = ops.W4Weight.pack(*_codes(gen, (32, 128), 64, False))
    w1 = ops.W4Weight.pack(*_codes(gen, (4, 64, 128), 64, False), gated=True)
    w2 = ops.W4Weight.pack(*_codes(gen, (4, 128, 32), 32, False))
    x, wt, ids = torch.randn(4, 128), torch.rand(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    logits = torch.randn(4, 8)
    for bad in (
        lambda: ops.linear_w4(x[:, :64], w),
        lambda: ops.linear_w4(x[0], w),
        lambda: ops.linear_w4(x, w, torch.zeros(1)),
        lambda: ops.experts_w4(x, w1, w2, wt[:3], ids),
        lambda: ops.experts_w4(x, w1, w2, wt, ids[:, :1]),
        lambda: ops.experts_w4(x[:, :64], w1, w2, wt, ids),
        lambda: ops.experts_w4(x, w1, ops.W4Weight.pack(*_codes(gen, (3, 128, 32), 32, False)), wt, ids),
        lambda: ops.route_experts(logits[0], 2),
        lambda: ops.route_experts(logits.double(), 2),
        lambda: ops.route_experts(logits, 2, bias=torch.zeros(1)),
    ):
        with pytest.raises(ValueError):
            bad()
