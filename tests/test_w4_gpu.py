"""The expert router, the 4-bit linear product and the 4-bit experts on the GPU against 64-bit forms.

Tolerances. One rounding to bf16 is off by at most 2^-8 of the value. Sums are held in fp32: a chain of
n additions is off by at most n 2^-23 of the sum of magnitudes (2^-23 rather than 2^-24, since a tensor
core may truncate), and the chains here are at most K / 16 + 64 additions long. Products that run
with the weights rounded to bf16 (many tokens) are off by another 2^-8 of the sum of magnitudes at
most, and by far less in the 2-norm: there one rounding is 2^-8 / sqrt(3) at most.
"""

from dataclasses import replace

import pytest
import torch

pytestmark = pytest.mark.gpu

from minisgl import ops  # noqa: E402

DEV = "cuda"
R = 2.0 ** -8  # half a step of bf16
A = 2.0 ** -23


@pytest.fixture(autouse=True)
def _cuda_only():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(0)
    yield
    torch.cuda.synchronize()
    from minisgl._native import cuda

    assert cuda().get_error()[0] == 0


def _codes(shape, group, zeros, dtype=torch.bfloat16):
    q = torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,), dtype=torch.uint8, device=DEV)
    side = shape[:-1] + (shape[-1] // group,)
    s = (torch.rand(side, device=DEV) * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 16, side, dtype=torch.uint8, device=DEV) if zeros else None
    return q, s, z


def _wide(q, s, z):
    """The weights in 64 bits, straight from the codes."""
    v = torch.stack([q & 15, q >> 4], dim=-1).flatten(-2).double().unflatten(-1, (s.shape[-1], -1))
    zero = 8.0 if z is None else z.double().unsqueeze(-1)
    return ((v - zero) * s.double().unsqueeze(-1)).flatten(-2)


def _near(got, want, bound):
    if got.numel() == 0:
        return
    off = (got.double() - want).abs()
    worst = (off - bound).argmax()
    inside = bool((off <= bound).all())
    assert inside, f"off by {off.flatten()[worst]:.3g}, bound {bound.flatten()[worst]:.3g}"


def _near_norm(got, want, rel):
    d = (got.double() - want).norm() / want.norm().clamp(min=1e-30)
    assert d <= rel, f"2-norm off by {d:.3g}"


def _check_linear(x, q, s, z, bias, got):
    m, xd = _wide(q, s, z), x.double()
    want, size = xd @ m.t(), xd.abs() @ m.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    assert got.shape == want.shape and got.dtype == torch.bfloat16
    k = x.shape[1]
    if x.shape[0] <= 16:  # scales on the fp32 sums; above, every weight is rounded: R of its magnitude each
        _near(got, want, R * want.abs() + (k / 16 + 64) * A * size)
    else:
        _near(got, want, R * want.abs() + (R + (k / 16 + 64) * A) * size)
    if got.numel() >= 256:
        _near_norm(got, want, 2 * R / 3 ** 0.5)


# ------------------------------------------------------------------------------------------ linear
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 24, 32, 33, 64, 100, 130, 257])
@pytest.mark.parametrize("N,K,group", [(16, 64, 64), (1001, 2880, 32), (2048, 1024, 128), (640, 8320, 64)])
def test_linear(M, N, K, group):
    zeros = (M + N) % 2 == 0
    q, s, z = _codes((N, K), group, zeros, torch.float16 if M % 3 == 0 else torch.bfloat16)
    x = torch.randn(M, K, device=DEV).to(torch.bfloat16)
    bias = torch.randn(N, device=DEV).to(torch.bfloat16) if M % 2 else None
    _check_linear(x, q, s, z, bias, ops.linear_w4(x, ops.W4Weight.pack(q, s, z), bias))


@pytest.mark.parametrize("M", [1, 16, 48])
@pytest.mark.parametrize("N", [1, 5, 15, 17, 129, 2384])
@pytest.mark.parametrize("K,group", [(32, 32), (96, 32), (160, 32), (192, 64), (128, 128), (896, 128)])
def test_linear_ragged(M, N, K, group):
    q, s, z = _codes((N, K), group, N % 2 == 0)
    x = torch.randn(M, K, device=DEV).to(torch.bfloat16)
    _check_linear(x, q, s, z, None, ops.linear_w4(x, ops.W4Weight.pack(q, s, z)))


@pytest.mark.parametrize("M,N,K", [(1, 34816, 5120), (12, 5120, 17408), (32, 256, 20480), (16, 64, 33024), (3, 151936, 1024)])
def test_linear_large(M, N, K):
    q, s, z = _codes((N, K), 128, M == 12)
    x = torch.randn(M, K, device=DEV).to(torch.bfloat16)
    _check_linear(x, q, s, z, None, ops.linear_w4(x, ops.W4Weight.pack(q, s, z)))


def test_linear_no_tokens():
    q, s, z = _codes((48, 128), 64, False)
    y = ops.linear_w4(torch.empty(0, 128, device=DEV, dtype=torch.bfloat16), ops.W4Weight.pack(q, s, z))
    assert y.shape == (0, 48)


@pytest.mark.parametrize("M", [6, 40])
def test_linear_strides(M):
    """Rows inside a wider tensor, rows off the 16-byte grid, columns apart: all as the dense copy."""
    q, s, z = _codes((112, 256), 64, True)
    w = ops.W4Weight.pack(q, s, z)
    wide = torch.randn(M, 1024, device=DEV).to(torch.bfloat16)
    for x in (wide[:, 256:512], wide[:, 3:259], wide[:, ::4], wide[:1, 5:261].expand(M, 256)):
        assert torch.equal(ops.linear_w4(x, w), ops.linear_w4(x.contiguous().clone(), w))


@pytest.mark.parametrize("M", [4, 20, 60])
def test_linear_rows_are_apart(M):
    """What one token holds (an infinity, NaN) stays in its own row, and infinities keep their sign."""
    q, s, z = _codes((80, 128), 128, False)
    q[0] = 0xFF  # row 0: every weight is 7 scales
    q[1] = 0x11  # row 1: -7
    w = ops.W4Weight.pack(q, s, z)
    x = torch.randn(M, 128, device=DEV).to(torch.bfloat16)
    clean = ops.linear_w4(x, w)
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    got = ops.linear_w4(x, w)
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(got[keep], clean[keep])
    assert bool(got[1].isnan().all())
    assert got[2, 0] == float("inf") and got[2, 1] == float("-inf")


# ----------------------------------------------------------------------------------------- experts
def _act(h, inter, activation):
    g, u = h[:, :inter], h[:, inter:]
    if activation == "silu":
        return g * torch.sigmoid(g) * u
    if activation == "gelu":
        return torch.nn.functional.gelu(g, approximate="tanh") * u
    g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
    return g * torch.sigmoid(1.702 * g) * (u + 1)


def _experts_wide(x, c1, c2, weights, ids, activation="silu", offset=0, b1=None, b2=None):
    """(result, what one rounding of every activated value and of the sums can move it by)"""
    E, H, inter = c1[0].shape[0], c2[0].shape[1], c1[0].shape[1] // 2
    out = torch.zeros(x.shape[0], H, dtype=torch.float64, device=x.device)
    size = torch.zeros_like(out)
    for e in range(E):
        tok, slot = torch.nonzero(ids == e + offset, as_tuple=True)
        if len(tok) == 0:
            continue
        m1, m2 = (_wide(*(None if t is None else t[e] for t in c)) for c in (c1, c2))
        h = x[tok].double() @ m1.t() + (0 if b1 is None else b1[e].double())
        a = _act(h, inter, activation)
        w = weights[tok, slot, None].double()
        out.index_add_(0, tok, w * (a @ m2.t() + (0 if b2 is None else b2[e].double())))
        size.index_add_(0, tok, w.abs() * (a.abs() @ m2.abs().t() + (0 if b2 is None else b2[e].double().abs())))
    return out, size


def _check_experts(got, want, size):
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    # roundings: the activated values, with many tokens the weights of both products too (those of the
    # first move an activated value by a few roundings of it), and the result
    _near(got, want, R * want.abs() + 6 * R * size)
    if want.norm() > 0 and got.numel() >= 256:
        _near_norm(got, want, 3 * R / 3 ** 0.5)


def _experts_case(T, E, k, H, inter, g1, g2, zeros, dtype=torch.bfloat16):
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    c1, c2 = _codes((E, 2 * inter, H), g1, zeros, dtype), _codes((E, H, inter), g2, zeros, dtype)
    c1[1].mul_(0.3)
    weights, ids = ops.route_experts(torch.randn(T, E, device=DEV), k)
    return x, c1, c2, weights, ids


def _packed(c1, c2):
    return ops.W4Weight.pack(*c1, gated=True), ops.W4Weight.pack(*c2)


@pytest.mark.parametrize("T", [1, 2, 5, 16, 33, 80, 300])
@pytest.mark.parametrize("E,k,H,inter,g1,g2", [(8, 2, 256, 128, 64, 32), (128, 8, 512, 192, 128, 64), (4, 4, 96, 32, 32, 32),
                                              (3, 1, 2880, 160, 64, 32), (32, 6, 384, 256, 32, 128)])
def test_experts(T, E, k, H, inter, g1, g2):
    x, c1, c2, weights, ids = _experts_case(T, E, k, H, inter, g1, g2, T % 2 == 1, torch.float16 if T == 5 else torch.bfloat16)
    got = ops.experts_w4(x, *_packed(c1, c2), weights, ids)
    _check_experts(got, *_experts_wide(x, c1, c2, weights, ids))


@pytest.mark.parametrize("T", [3, 200])
@pytest.mark.parametrize("activation", ["silu", "gelu", "swiglu_oai"])
def test_experts_activations_and_biases(T, activation):
    E, H, inter = 6, 192, 96
    x, c1, c2, weights, ids = _experts_case(T, E, 3, H, inter, 64, 32, True)
    b1 = torch.randn(E, 2 * inter, device=DEV).to(torch.bfloat16)
    b2 = torch.randn(E, H, device=DEV).to(torch.bfloat16)
    got = ops.experts_w4(x, *_packed(c1, c2), weights, ids, activation=activation, w1_bias=b1, w2_bias=b2)
    _check_experts(got, *_experts_wide(x, c1, c2, weights, ids, activation, 0, b1, b2))


@pytest.mark.parametrize("T", [1, 4, 40, 200])
def test_experts_of_a_share(T):
    """Ids of experts that are elsewhere add nothing, whatever their weight; a token may have none here."""
    E, H, inter = 4, 128, 64
    x, c1, c2, _, _ = _experts_case(T, E, 1, H, inter, 64, 64, False)
    ids = torch.randint(-3, 12, (T, 3), device=DEV, dtype=torch.int32)
    ids[0] = torch.tensor([-1, 2 ** 31 - 1, -2 ** 31], device=DEV, dtype=torch.int64).to(torch.int32)
    weights = torch.rand(T, 3, device=DEV)
    weights[0] = float("nan")
    got = ops.experts_w4(x, *_packed(c1, c2), weights, ids, expert_offset=5)
    assert bool((got[0] == 0).all())
    _check_experts(got[1:], *_experts_wide(x[1:], c1, c2, weights[1:], ids[1:], offset=5))


@pytest.mark.parametrize("T", [1, 7, 90])
def test_experts_chosen_twice_and_alone(T):
    """The same expert twice in a row of ids counts twice; every token at one expert."""
    x, c1, c2, _, _ = _experts_case(T, 5, 1, 128, 96, 32, 32, True)
    ids = torch.full((T, 2), 3, device=DEV, dtype=torch.int32)
    weights = torch.rand(T, 2, device=DEV)
    got = ops.experts_w4(x, *_packed(c1, c2), weights, ids)
    _check_experts(got, *_experts_wide(x, c1, c2, weights, ids))


def test_experts_no_tokens():
    x, c1, c2, _, _ = _experts_case(1, 5, 1, 128, 96, 32, 32, True)
    got = ops.experts_w4(x[:0], *_packed(c1, c2), torch.empty(0, 2, device=DEV),
                         torch.empty(0, 2, device=DEV, dtype=torch.int32))
    assert got.shape == (0, 128)


@pytest.mark.parametrize("T", [5, 70])
def test_experts_are_the_same_every_time(T):
    x, c1, c2, weights, ids = _experts_case(T, 16, 4, 256, 128, 64, 64, False)
    w1, w2 = _packed(c1, c2)
    first = ops.experts_w4(x, w1, w2, weights, ids)
    for _ in range(5):
        assert torch.equal(first, ops.experts_w4(x, w1, w2, weights, ids))


# ------------------------------------------------------------------------------------------ router
def _check_route(logits, k, **kw):
    w, ids = ops.route_experts(logits, k, **kw)
    cpu = {n: v.cpu() if torch.is_tensor(v) else v for n, v in kw.items()}
    want_w, want_ids = ops.route_experts(logits.cpu(), k, **cpu)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu(), want_ids)
    # exponentials of fp32 (a few roundings of 2^-24), of arguments whose own rounding counts |x| <= 32 times
    torch.testing.assert_close(w.cpu(), want_w, rtol=64 * 2.0 ** -24, atol=1e-30)


@pytest.mark.parametrize("T", [1, 3, 64, 1000])
@pytest.mark.parametrize("E,k", [(1, 1), (8, 2), (96, 6), (128, 8), (160, 5), (256, 8), (511, 10), (512, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route(T, E, k, scoring):
    logits = torch.randn(T, E, device=DEV) * 2
    _check_route(logits, k, scoring=scoring)
    _check_route(logits.to(torch.bfloat16), k, scoring=scoring, renormalize=False, scale=1.5)
    _check_route(logits, k, scoring=scoring, bias=torch.randn(E, device=DEV) * 0.2)


@pytest.mark.parametrize("E,groups,kept,k", [(256, 8, 4, 8), (96, 3, 2, 6), (64, 32, 5, 7), (512, 2, 1, 9), (40, 20, 1, 2),
                                             (512, 256, 256, 8), (12, 4, 4, 12)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_groups(E, groups, kept, k, group_score, scoring):
    logits = torch.randn(333, E, device=DEV) * 1.5
    kw = dict(scoring=scoring, num_groups=groups, top_groups=kept, group_score=group_score)
    _check_route(logits, k, **kw)
    _check_route(logits.to(torch.bfloat16), k, bias=torch.randn(E, device=DEV) * 0.1, renormalize=False, **kw)


@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_route_ties(group_score):
    """Few different logits and biases: almost everything is a tie, decided by the lower id."""
    logits = torch.randint(0, 3, (500, 64), device=DEV).float()
    kw = dict(num_groups=8, top_groups=3, group_score=group_score)
    for bias in (None, torch.zeros(64, device=DEV), torch.randint(0, 2, (64,), device=DEV).float() * 0.25):
        for scoring in ("softmax", "sigmoid"):
            _check_route(logits, 8, scoring=scoring, bias=bias, **kw)
            _check_route(logits, 8, scoring=scoring, bias=bias)


def test_route_near_ties():
    """Scores plus bias that differ by less than fp32 resolves near 1, but not equal: 64-bit order."""
    x = torch.linspace(-1e-6, 1e-6, 128, device=DEV)[torch.randperm(128, device=DEV)]
    logits = x.repeat(50, 1) * torch.rand(50, 1, device=DEV)
    for scoring in ("softmax", "sigmoid"):
        _check_route(logits, 8, scoring=scoring, bias=torch.full((128,), 0.5, device=DEV))
        _check_route(logits, 8, scoring=scoring, bias=torch.full((128,), 0.5, device=DEV), num_groups=4, top_groups=2,
                     group_score="top2")
        _check_route(logits, 8, scoring=scoring, num_groups=4, top_groups=2, group_score="top2")


def test_route_extremes():
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    rows = torch.randn(8, 16, device=DEV)
    rows[0] = -inf
    rows[1] = nan
    rows[2, ::2] = nan
    rows[3, :5] = inf
    rows[4] = low
    rows[5, 3:] = -inf
    rows[6, :4] = low
    rows[7] *= 300
    bias = torch.randn(16, device=DEV)
    odd = bias.clone()
    odd[0], odd[3], odd[7], odd[9] = nan, inf, -inf, -inf
    for scoring in ("softmax", "sigmoid"):
        for b in (None, bias, odd):
            for kw in ({}, dict(num_groups=4, top_groups=2), dict(num_groups=4, top_groups=2, group_score="top2")):
                _check_route(rows, 6, scoring=scoring, bias=b, **kw)


def test_route_strides():
    wide = torch.randn(40, 300, device=DEV)
    for x in (wide[:, 7:135], wide[::2, :128], wide[:, ::2][:, :128], wide[:1, :128].expand(40, 128)):
        _check_route(x, 8)
    assert ops.route_experts(wide[:0], 4)[1].shape == (0, 4)


# -------------------------------------------------------------------------------- together and apart
def _layer(x, router, w1, w2, wo):
    logits = ops.linear_f32(x, router)
    weights, ids = ops.route_experts(logits, 4, scoring="sigmoid", num_groups=4, top_groups=2, group_score="top2", scale=1.5)
    return ops.linear_w4(ops.experts_w4(x, w1, w2, weights, ids), wo), ids, weights


@pytest.mark.parametrize("T", [1, 9, 64, 150])
def test_layer_eager_and_captured(T):
    """Router -> experts -> projection as a model runs them, eagerly and replayed on new tokens."""
    E, H, inter = 16, 256, 128
    x, c1, c2, _, _ = _experts_case(T, E, 1, H, inter, 64, 64, False)
    w1, w2 = _packed(c1, c2)
    co = _codes((192, H), 128, True)
    wo = ops.W4Weight.pack(*co)
    router = (torch.randn(E, H, device=DEV) * 0.1).to(torch.bfloat16)
    y, ids, weights = _layer(x, router, w1, w2, wo)
    mid, size = _experts_wide(x, c1, c2, weights, ids)
    m = _wide(*co)
    # the experts' result goes on in bf16: its bound of 7 roundings, through the projection, and one more
    _near(y, mid @ m.t(), 7 * R * (size @ m.abs().t()) + 2 * R * (mid.abs() @ m.abs().t()) + R * (mid @ m.t()).abs())

    static = x.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            _layer(static, router, w1, w2, wo)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        captured = _layer(static, router, w1, w2, wo)
    for seed in range(3):
        torch.manual_seed(seed)
        static.copy_(torch.randn(T, H, device=DEV))
        g.replay()
        again = [t.clone() for t in captured]
        for a, b in zip(again, _layer(static, router, w1, w2, wo)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [2, 100])
def test_two_streams_at_once(T):
    """Calls on two streams share nothing."""
    x, c1, c2, weights, ids = _experts_case(T, 8, 2, 512, 256, 64, 64, False)
    w1, w2 = _packed(c1, c2)
    co = _codes((1024, 512), 64, False)
    wo = ops.W4Weight.pack(*co)
    other = torch.randn_like(x)
    want = [(ops.experts_w4(v, w1, w2, weights, ids), ops.linear_w4(v, wo)) for v in (x, other)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for i, v in enumerate((x, other)):
            with torch.cuda.stream(streams[i]):
                got[i].append((ops.experts_w4(v, w1, w2, weights, ids), ops.linear_w4(v, wo)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


def test_refusals():
    q, s, z = _codes((32, 128), 64, True)
    w = ops.W4Weight.pack(q, s, z)
    x = torch.randn(4, 128, device=DEV).to(torch.bfloat16)
    c1, c2 = _codes((4, 64, 128), 64, False), _codes((4, 128, 32), 32, False)
    w1, w2 = _packed(c1, c2)
    wt, ids = torch.rand(4, 2, device=DEV), torch.zeros(4, 2, device=DEV, dtype=torch.int32)
    logits = torch.randn(4, 8, device=DEV)
    short = replace(w, n=500)
    wrong_group = replace(w, group=16)
    for bad in (
        lambda: ops.linear_w4(x.float(), w),
        lambda: ops.linear_w4(x[:, :64], w),
        lambda: ops.linear_w4(x[0], w),
        lambda: ops.linear_w4(x, w.to("cpu")),
        lambda: ops.linear_w4(x, w, torch.zeros(31, device=DEV, dtype=torch.bfloat16)),
        lambda: ops.linear_w4(x, w, torch.zeros(32, device=DEV)),
        lambda: ops.linear_w4(x, short),
        lambda: ops.linear_w4(x, wrong_group),
        lambda: ops.experts_w4(x, w1, w2, wt[:3], ids),
        lambda: ops.experts_w4(x, w1, w2, wt, ids.long()),
        lambda: ops.experts_w4(x, w1, w2, wt.half(), ids),
        lambda: ops.experts_w4(x[:, :64], w1, w2, wt, ids),
        lambda: ops.experts_w4(x, w1, ops.W4Weight.pack(*_codes((4, 128, 64), 32, False)), wt, ids),
        lambda: ops.experts_w4(x, w1, ops.W4Weight.pack(*_codes((3, 128, 32), 32, False)), wt, ids),
        lambda: ops.experts_w4(x, w1, w2, wt, ids, w1_bias=torch.zeros(4, 32, device=DEV, dtype=torch.bfloat16)),
        lambda: ops.route_experts(logits.double(), 2),
        lambda: ops.route_experts(logits[0], 2),
        lambda: ops.route_experts(logits, 9),
        lambda: ops.route_experts(logits, 5, num_groups=2),
        lambda: ops.route_experts(logits, 2, num_groups=3),
        lambda: ops.route_experts(logits, 2, num_groups=2, top_groups=3),
        lambda: ops.route_experts(logits, 1, num_groups=8, top_groups=2, group_score="top2"),
        lambda: ops.route_experts(logits, 2, bias=torch.zeros(7, device=DEV)),
        lambda: ops.route_experts(logits, 2, bias=torch.zeros(8)),
        lambda: ops.route_experts(torch.zeros(2, 513, device=DEV), 2),
    ):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
