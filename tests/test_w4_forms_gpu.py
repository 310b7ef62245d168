"""Every form of the 4-bit products for many tokens, against 64-bit sums with their roundings made.

Above 16 tokens a weight of the linear product is (code - zero) * scale rounded to bf16. That rounding is part of the
form, so the oracle makes it too, and what is left is narrow: the sums' chains of at most K / 16 + 64 additions in
fp32, 2^-23 of the sum of magnitudes each, and one rounding of the result, 2^-8. The experts' weights are exact (two
parts of them added one after the other: K / 8 additions); their activated values are two bf16 for few tokens and
rounded to one for many.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

from minisgl import ops  # noqa: E402
from test_w4_checks_cpu import bad_calls  # noqa: E402
from test_w4_gpu import A, DEV, R, _codes, _cuda_only, _experts_wide, _near, _packed, _wide  # noqa: E402,F401


def _check_tiles(x, q, s, z, bias, got):
    m, xd = _wide(q, s, z).to(torch.bfloat16).double(), x.double()
    want, size = xd @ m.t(), xd.abs() @ m.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    assert got.shape == want.shape and got.dtype == torch.bfloat16
    _near(got, want, R * want.abs() + (x.shape[1] / 16 + 64) * A * size)


@pytest.mark.parametrize("M", [1, 5, 16, 20])
def test_linear_of_very_wide_rows(M):
    """Not even one row fits beside the streaming product's rings: the form for many tokens, whatever their number."""
    q, s, z = _codes((33, 460800), 128, False)
    x = torch.randn(M, 460800, device=DEV).to(torch.bfloat16)
    _check_tiles(x, q, s, z, None, ops.linear_w4(x, ops.W4Weight.pack(q, s, z)))


def _experts_bounded(x, c1, c2, weights, ids, offset=0, few=False):
    """(result, bound) of silu experts. ``few``: an activated value is two bf16, off by 2^-16 of it. Else it is rounded to
    one; the fp32 sums before it move it a little, and where that reaches the middle between two bf16 values it may
    become the other one. What an activated value is off by goes through the second product.
    An fp16 scale of 11 bits is its first four, whose product with a code is exact, and seven more, an eighth of it at
    most, whose product is rounded to bf16: off by 2^-9 2^-3."""
    E, H, inter = c1[0].shape[0], c2[0].shape[1], c1[0].shape[1] // 2
    w1_off, w2_off = (2.0 ** -12 if c[1].dtype == torch.float16 else 0.0 for c in (c1, c2))
    out = torch.zeros(x.shape[0], H, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    for e in range(E):
        tok, slot = torch.nonzero(ids == e + offset, as_tuple=True)
        if len(tok) == 0:
            continue
        m1, m2 = (_wide(*(None if t is None else t[e] for t in c)) for c in (c1, c2))
        xd = x[tok].double()
        h, dh = xd @ m1.t(), ((x.shape[1] / 8 + 64) * A + w1_off) * (xd.abs() @ m1.abs().t())
        g, u, dg, du = h[:, :inter], h[:, inter:], dh[:, :inter], dh[:, inter:]
        silu = g * torch.sigmoid(g)
        a = silu * u
        # silu's slope is at most 1.1; the fast exponential is off by 2 + 1.2 |g| steps of fp32 and the quotient by 2
        # (and is zero where it would be below 2^-126)
        off = 1.1 * dg * (u.abs() + du) + silu.abs() * du + (8 + 2 * g.abs()) * A * a.abs() + 1e-35
        if few:
            off = off + 2.0 ** -16 * a.abs()
        else:
            exact, a = a, a.to(torch.bfloat16).double()
            exponent = torch.frexp((exact.abs() - off).clamp(min=2.0 ** -120))[1]
            half = torch.ldexp(torch.ones_like(a), exponent - 9)  # of a step of bf16
            off = torch.where((exact - a).abs() + off >= half, off + 2 * R * (exact.abs() + off), torch.zeros_like(a))
        w = weights[tok, slot, None].double()
        out.index_add_(0, tok, w * (a @ m2.t()))
        bound.index_add_(0, tok, w.abs() * (off @ m2.abs().t()
                                            + ((inter / 8 + 64 + ids.shape[1]) * A + w2_off) * ((a.abs() + off) @ m2.abs().t())))
    return out, R * (out.abs() + bound) + bound


@pytest.mark.parametrize("T,E,H,inter", [(1, 2, 65536, 32), (4, 2, 65536, 32), (3, 2, 64, 65536), (16, 2, 64, 65536)])
def test_experts_of_very_wide_rows(T, E, H, inter):
    c1, c2 = _codes((E, 2 * inter, H), 32, False), _codes((E, H, inter), 32, True)
    c1[1].mul_(0.02)
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    ids = torch.arange(T, device=DEV, dtype=torch.int32)[:, None] % E
    weights = torch.rand(T, 1, device=DEV)
    want, bound = _experts_bounded(x, c1, c2, weights, ids)
    _near(ops.experts_w4(x, *_packed(c1, c2), weights, ids), want, bound)


MOST = 12  # pairs an expert up to which the form for few tokens runs


@pytest.mark.parametrize("T", [9, 17, 64, 8 * MOST, 8 * MOST + 1])
@pytest.mark.parametrize("spread", ["all ranks", "one expert", "elsewhere", "here"])
def test_experts_of_a_share_choose_by_all(T, spread):
    """4 experts of 64, 8 a token: up to 96 tokens an expert has 12 pairs if they spread over all ranks, and the form
    for few tokens runs whatever they do (three kernels; for many tokens there are four)."""
    from minisgl.engine.counters import COUNTERS

    E, total, k, H, inter, offset = 4, 64, 8, 256, 128, 20
    c1, c2 = _codes((E, 2 * inter, H), 64, True), _codes((E, H, inter), 128, False)
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    lo, hi = {"all ranks": (0, total), "one expert": (22, 23), "elsewhere": (24, total), "here": (20, 24)}[spread]
    ids = torch.randint(lo, hi, (T, k), device=DEV, dtype=torch.int32)
    weights = torch.rand(T, k, device=DEV)
    w1, w2 = _packed(c1, c2)
    want = {few: _experts_bounded(x, c1, c2, weights, ids, offset, few) for few in (False, True)}
    before = COUNTERS.launches
    got = ops.experts_w4(x, w1, w2, weights, ids, expert_offset=offset, num_experts=total)
    few = T <= MOST * 8
    assert COUNTERS.launches - before == (3 if few else 4)
    _near(got, *want[few])
    if spread == "elsewhere":
        assert not got.any()
    for n in (E, total + 1000):  # whatever the estimate, the same experts' results
        before = COUNTERS.launches
        other = ops.experts_w4(x, w1, w2, weights, ids, expert_offset=offset, num_experts=n)
        few = T * k <= min(MOST * n, 4096)
        assert COUNTERS.launches - before == (3 if few else 4)
        _near(other, *want[few])


def test_refused_as_on_the_cpu():
    before = torch.cuda.memory_allocated()
    for name, call in bad_calls(DEV):
        torch.cuda.reset_peak_memory_stats()
        with pytest.raises((RuntimeError, ValueError)) as what:
            call()
        assert not isinstance(what.value, torch.OutOfMemoryError), name
    assert torch.cuda.max_memory_allocated() - before < 2 ** 30


def test_kernels_are_counted():
    """One kernel a linear call, two where 16 rows of 33024 inputs run in halves; three for few tokens of experts,
    four for many (a plan before them)."""
    from minisgl.engine.counters import COUNTERS

    def launched(call):
        before = COUNTERS.launches
        call()
        return COUNTERS.launches - before

    w = ops.W4Weight.pack(*_codes((64, 33024), 128, False))
    x = torch.randn(40, 33024, device=DEV).to(torch.bfloat16)
    assert [launched(lambda: ops.linear_w4(x[:m], w)) for m in (0, 1, 16, 40)] == [0, 1, 2, 1]
    w1, w2 = _packed(_codes((4, 64, 128), 64, False), _codes((4, 128, 32), 32, False))
    x = torch.randn(25, 128, device=DEV).to(torch.bfloat16)
    ids, wt = torch.zeros(25, 2, device=DEV, dtype=torch.int32), torch.rand(25, 2, device=DEV)
    assert [launched(lambda: ops.experts_w4(x[:t], w1, w2, wt[:t], ids[:t])) for t in (0, 1, 24, 25)] == [0, 3, 3, 4]


# -------------------------------------------------------------------------- every form of the many-token product
def _side(M, form):
    """Scale types, zero points and inputs that end inside a record, another combination for each size and form."""
    i = M + 3 * form[0] + 5 * form[1]
    return (32, 64, 128)[i % 3], i % 2 == 0, (torch.bfloat16, torch.float16)[i // 2 % 2]


def _forced(form, x, q, s, z, bias):
    from minisgl._native import cuda

    cuda().w4_force_form(*form)
    try:
        return ops.linear_w4(x, ops.W4Weight.pack(q, s, z), bias)
    finally:
        cuda().w4_force_form(0, 0)


FORMS = [(1, 1), (1, 2), (1, 5), (1, 8), (2, 1), (2, 2), (2, 3), (2, 8)]


# up to 192 tokens a tile: whole steps in a stage; 193 to 208: half steps with 256-row tiles; 300: two tiles of tokens
@pytest.mark.parametrize("M", [17, 64, 96, 97, 130, 192, 193, 200, 208, 209, 300])
@pytest.mark.parametrize("form", FORMS)
def test_linear_every_form(M, form):
    for shift in range(3):
        group, zeros, dtype = _side(M + shift, form)
        N, K = 530 + 13 * shift, {32: 1184, 64: 1088, 128: 1152}[group]  # 37 x 32, 17 x 64, 9 x 128
        q, s, z = _codes((N, K), group, zeros, dtype)
        x = torch.randn(M, K, device=DEV).to(torch.bfloat16)
        bias = torch.randn(N, device=DEV).to(torch.bfloat16) if shift else None
        _check_tiles(x, q, s, z, bias, _forced(form, x, q, s, z, bias))


@pytest.mark.parametrize("M", [64, 130, 192, 200, 700])
@pytest.mark.parametrize("form", [(1, 1), (2, 1)])
@pytest.mark.parametrize("group,zeros,dtype", [(32, True, torch.float16), (64, False, torch.float16), (128, False, torch.bfloat16),
                                               (128, True, torch.bfloat16)])
def test_linear_many_tiles_a_block(M, form, group, zeros, dtype):
    """More tiles than SMs: blocks go on to further tiles with their rings and phases where they are."""
    q, s, z = _codes((39700, 640), group, zeros, dtype)
    x = torch.randn(M, 640, device=DEV).to(torch.bfloat16)
    _check_tiles(x, q, s, z, None, _forced(form, x, q, s, z, None))


@pytest.mark.parametrize("form", [(2, 1), (2, 3), (1, 4)])
@pytest.mark.parametrize("group,zeros,dtype", [(32, True, torch.float16), (128, False, torch.bfloat16)])
def test_linear_long_inputs(form, group, zeros, dtype):
    """Some hundred steps a tile: the rings turn many times."""
    for M in (40, 200):
        q, s, z = _codes((1000, 17408), group, zeros, dtype)
        x = torch.randn(M, 17408, device=DEV).to(torch.bfloat16)
        _check_tiles(x, q, s, z, None, _forced(form, x, q, s, z, None))


def test_linear_form_that_does_not_fit():
    q, s, z = _codes((64, 256), 64, False)
    x = torch.randn(20, 256, device=DEV).to(torch.bfloat16)
    with pytest.raises(RuntimeError, match="not supported"):
        _forced((2, 3), x, q, s, z, None)  # two records of inputs cannot be cut in three


@pytest.mark.parametrize("M,N,K", [(17, 34816, 1024), (64, 34500, 640), (130, 10240, 5120), (192, 5120, 17408), (64, 5120, 17408),
                                   (200, 34816, 1024), (256, 10240, 1024), (16384, 640, 512), (16385, 1001, 96)])
def test_linear_of_real_sizes(M, N, K):
    """Projections as models have them, at decode batches and prompts up to a whole chunk."""
    q, s, z = _codes((N, K), 32 if K % 128 else 128, M % 2 == 0, torch.float16 if M in (64, 192) else torch.bfloat16)
    x = torch.randn(M, K, device=DEV).to(torch.bfloat16)
    _check_tiles(x, q, s, z, None, ops.linear_w4(x, ops.W4Weight.pack(q, s, z)))


# ------------------------------------------------------------------------------------ the experts, element by element
@pytest.mark.parametrize("T,E,k,H,inter,g1,g2", [(4, 8, 2, 256, 128, 64, 32), (16, 128, 8, 512, 192, 128, 64), (33, 4, 4, 96, 32, 32, 32),
                                                (80, 3, 1, 2880, 160, 64, 32), (300, 32, 6, 384, 256, 32, 128),
                                                (777, 5, 2, 160, 416, 32, 32), (100, 1, 1, 128, 64, 128, 64)])
@pytest.mark.parametrize("zeros,dtype", [(False, torch.bfloat16), (True, torch.float16)])
def test_experts_element_by_element(T, E, k, H, inter, g1, g2, zeros, dtype):
    c1, c2 = _codes((E, 2 * inter, H), g1, zeros, dtype), _codes((E, H, inter), g2, zeros, dtype)
    c1[1].mul_(0.3)
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    weights, ids = ops.route_experts(torch.randn(T, E, device=DEV), k)
    want, bound = _experts_bounded(x, c1, c2, weights, ids, few=T * k <= MOST * E)
    _near(ops.experts_w4(x, *_packed(c1, c2), weights, ids), want, bound)


@pytest.mark.parametrize("E,k,offset,all_experts", [(32, 8, 0, None), (16, 8, 48, 128)])
def test_experts_of_a_whole_chunk(E, k, offset, all_experts):
    """16384 tokens, uneven shares: an expert without any, one that a quarter of the pairs goes to."""
    T, H, inter = 16384, 256, 128
    c1, c2 = _codes((E, 2 * inter, H), 64, False), _codes((E, H, inter), 128, True)
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    p = torch.randn(T, all_experts or E, device=DEV)
    p[:, offset + 3] = -100.0
    p[:, offset + 5] += 2.0
    weights, ids = ops.route_experts(p, k)
    got = ops.experts_w4(x, *_packed(c1, c2), weights, ids, expert_offset=offset, num_experts=all_experts)
    _near(got, *_experts_bounded(x, c1, c2, weights, ids, offset))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k", [(1, 64, 8), (3, 8, 2), (40, 64, 2), (90, 8, 2), (300, 8, 2), (700, 5, 3), (4000, 8, 2)])
def test_experts_lose_no_bits(T, E, k, dtype):
    """In the 2-norm: the result's rounding to bf16, for many tokens the activated values' too, and nothing else. A
    rounding is even over half a step to either side, 2^-8 / sqrt(3) at most for values just above a power of two; a
    hundredth more for fp32 sums and chance."""
    c1, c2 = _codes((E, 512, 512), 64, True, dtype), _codes((E, 512, 256), 32, False, dtype)
    x = torch.randn(T, 512, device=DEV).to(torch.bfloat16)
    weights, ids = ops.route_experts(torch.randn(T, E, device=DEV), k)
    want, _ = _experts_wide(x, c1, c2, weights, ids)
    got = ops.experts_w4(x, *_packed(c1, c2), weights, ids)
    roundings = 1 if T * k <= MOST * E else 2
    assert (got.double() - want).norm() / want.norm() <= 1.01 * R * (roundings / 3) ** 0.5
