"""The 8-bit key/value cache on the GPU: rows against the format's definition, attention against 64 bits."""

import math

import pytest
import torch

from kv8_cases import FMTS, RAGGED, Case, bad_calls, nearest, values
from minisgl import ops

pytestmark = pytest.mark.gpu


def error_word():
    from minisgl._native import cuda

    return cuda().get_error()


@pytest.fixture(autouse=True)
def clean_error_word():
    error_word()
    yield
    assert error_word()[0] == 0


# ------------------------------------------------------------------------------------ rows
def rows_of(gen, *shape):
    x = torch.randn(*shape, generator=gen) * torch.randn(*shape[:-1], 1, generator=gen).mul(2).exp()
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("T,nkv,hd", [(1, 1, 64), (3, 2, 128), (77, 8, 128), (130, 5, 64)])
def test_store_is_exact(dtype, T, nkv, hd):
    gen = torch.Generator().manual_seed(T)
    cache = ops.KV8Cache.alloc(256, nkv, hd, dtype)
    k, v = rows_of(gen, T, nkv, hd), rows_of(gen, T, nkv, hd)
    k[0, 0] = torch.linspace(-1, 1, hd).to(torch.bfloat16)
    v[0, 0, ::2] = v[0, 0].abs().max() / 2  # on a tie of int8
    loc = torch.randperm(256, generator=gen)[:T].to(torch.int32)
    ops.store_kv8(k.cuda(), v.cuda(), cache, loc.cuda())
    rest = torch.ones(256, dtype=torch.bool)
    rest[loc.long()] = False
    for x, codes, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        want, s = nearest(x, dtype)
        got = values(codes[:, loc.long().cuda()], torch.ones(nkv, T)).transpose(0, 1)
        assert torch.equal(got, want)
        top = x.float().abs().amax(-1)
        assert torch.equal(scale[:, loc.long().cuda()].t().cpu(), top / (127.0 if dtype == torch.int8 else 448.0))
        assert (codes.view(torch.uint8)[:, rest.cuda()] == 0).all() and (scale[:, rest.cuda()] == 0).all()
    got_k, got_v = ops.load_kv8(cache, loc.cuda())
    for x, got in ((k, got_k), (v, got_v)):
        want, s = nearest(x, dtype)
        want = want * s
        # half a bf16 step, and two fp32 roundings (the scale's, the product's)
        assert ((got.cpu().double() - want).abs() <= want.abs() * (2.0**-8 + 2.0**-22)).all()


@pytest.mark.parametrize("dtype", FMTS)
def test_store_of_every_pair_of_magnitudes(dtype):
    """Every bf16 mantissa against every other one as the row's largest, in three distances: ties and borders."""
    a = torch.arange(128, 256, dtype=torch.float32)
    x = torch.cat([a.mul(by).expand(128, 1, 128) for by in (1.0, 0.5, 0.0078125)])
    x[:, 0, 0] = 2 * a.repeat(3)
    x = x.to(torch.bfloat16).cuda()
    cache = ops.KV8Cache.alloc(384, 1, 128, dtype)
    loc = torch.arange(384, dtype=torch.int32, device="cuda")
    ops.store_kv8(x, -x, cache, loc)
    want, _ = nearest(x, dtype)
    assert torch.equal(values(cache.k, torch.ones(1, 384)).transpose(0, 1), want)
    assert torch.equal(values(cache.v, torch.ones(1, 384)).transpose(0, 1), -want)


@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e30, 1e38])
def test_store_of_extreme_rows(dtype, size):
    gen = torch.Generator().manual_seed(3)
    x = (torch.rand(4, 2, 64, generator=gen) * 2 - 1).mul(size).to(torch.bfloat16)
    cache = ops.KV8Cache.alloc(16, 2, 64, dtype)
    ops.store_kv8(x.cuda(), x.cuda(), cache, torch.arange(4, dtype=torch.int32, device="cuda"))
    want, _ = nearest(x, dtype)
    assert torch.equal(values(cache.k[:, :4], torch.ones(2, 4)).transpose(0, 1), want)


@pytest.mark.parametrize("dtype", FMTS)
def test_store_skips_and_odd_rows(dtype):
    cache = ops.KV8Cache.alloc(32, 2, 64, dtype)
    x = torch.ones(5, 2, 64, dtype=torch.bfloat16, device="cuda")
    x[1, 0, 3], x[2, 1, 60], x[3] = math.inf, math.nan, 0
    ops.store_kv8(x, x, cache, torch.tensor([0, 1, 2, 3, -1], dtype=torch.int32, device="cuda"))
    assert cache.k_scale[0, 1].isnan() and cache.v_scale[1, 2].isnan() and (cache.k_scale[:, 3:] == 0).all()
    assert (cache.k[0, 1].float() == 0).all() and cache.k_scale[1, 1].isfinite()
    k, v = ops.load_kv8(cache, torch.tensor([1, -5, 3, 0], dtype=torch.int32, device="cuda"))
    assert k[0, 0].isnan().all() and (v[1:3] == 0).all() and torch.equal(k[3], x[0])
    # strided rows and heads: views of a merged projection, every other head, an odd offset
    gen = torch.Generator().manual_seed(5)
    big = rows_of(gen, 5, 9 * 64 + 1).cuda()
    loc = torch.arange(5, dtype=torch.int32, device="cuda")
    for kv in (big[:, 64:192].unflatten(1, (2, 64)), big[:, : 4 * 64].unflatten(1, (4, 64))[:, ::2], big[:, 1:129].unflatten(1, (2, 64)),
               big[:1, :128].unflatten(1, (2, 64)).expand(5, 2, 64)):
        want = ops.KV8Cache.alloc(32, 2, 64, dtype)
        ops.store_kv8(kv, kv, cache, loc)
        ops.store_kv8(kv.contiguous(), kv.contiguous(), want, loc)
        assert torch.equal(cache.k[:, :5].view(torch.uint8), want.k[:, :5].view(torch.uint8))
        assert torch.equal(cache.v_scale[:, :5], want.v_scale[:, :5])


def test_slots_beyond_the_cache_are_recorded():
    cache = ops.KV8Cache.alloc(32, 2, 64)
    whole = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda") + 1
    ops.store_kv8(whole, whole, cache, torch.tensor([32, 2**31 - 1], dtype=torch.int32, device="cuda"))
    assert error_word()[0] == 3 and (cache.k_scale == 0).all()
    k, _ = ops.load_kv8(cache, torch.tensor([40], dtype=torch.int32, device="cuda"))
    assert (k == 0).all() and error_word()[0] == 3


def test_nothing_to_do():
    cache = ops.KV8Cache.alloc(16, 2, 64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    x = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    ops.store_kv8(x, x, cache, none)
    assert ops.load_kv8(cache, none)[0].shape == (0, 2, 64)
    table = torch.zeros(1, 16, dtype=torch.int32, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert ops.attention_kv8(x, cache, table, none, zero, none, page_size=16).shape == (0, 2, 64)
    got = ops.attention_kv8(torch.ones(3, 2, 64, dtype=torch.bfloat16, device="cuda"), cache, table, none, zero, none, page_size=16)
    assert (got == 0).all()
    got = ops.attention_kv8(torch.ones(3, 2, 64, dtype=torch.bfloat16, device="cuda"), cache, table[:0, :0], none, zero, none, page_size=16)
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("n,nkv,hd", [(20001, 2, 128), (13001, 7, 64), (5001, 16, 128)])
def test_many_rows(dtype, n, nkv, hd):
    """Enough rows that a lane takes two: the same as the plain forms, whose steps round as the kernels' do."""
    gen = torch.Generator().manual_seed(n)
    k, v = (rows_of(gen, n, nkv, hd) for _ in range(2))
    size = n // 16 * 16 + 16
    cache, want = (ops.KV8Cache.alloc(size, nkv, hd, dtype, device) for device in ("cuda", "cpu"))
    loc = torch.randperm(size, generator=gen)[:n].to(torch.int32)
    loc[5] = -1
    ops.store_kv8(k, v, want, loc)
    loc = loc.cuda()
    ops.store_kv8(k.cuda(), v.cuda(), cache, loc)
    assert all(torch.equal(a.view(torch.uint8).cpu(), b.view(torch.uint8))
               for a, b in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), (want.k, want.v, want.k_scale, want.v_scale)))
    for got, codes, scale in zip(ops.load_kv8(cache, loc), (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        x = codes[:, loc.long().clamp(min=0)].float() * scale[:, loc.long().clamp(min=0), None]
        x[:, 5] = 0
        assert torch.equal(got, x.transpose(0, 1).to(torch.bfloat16))


def heads_case(T, nq, nkv, hd, norm, seed=0):
    gen = torch.Generator().manual_seed(seed)
    qkv = rows_of(gen, T, nq + 2 * nkv, hd).flatten(1).cuda()
    pos = torch.randint(0, 500, (T,), generator=gen).to(torch.int32).cuda()
    cs = ops.ref.rope_cos_sin(500, hd, ops.ref.default_inv_freq(hd, 1e4)).cuda()
    w = [torch.randn(hd, generator=gen).to(torch.bfloat16).cuda() for _ in range(2)] if norm else [None, None]
    return qkv, pos, cs, *w


def same_cache(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8))
               for x, y in zip((a.k, a.v, a.k_scale, a.v_scale), (b.k, b.v, b.k_scale, b.v_scale)))


@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("T,nq,nkv,hd", [(1, 1, 1, 64), (5, 16, 8, 128), (130, 14, 2, 64), (33, 5, 5, 128)])
def test_heads_to_cache(dtype, norm, T, nq, nkv, hd):
    """The same queries and codes as storing bf16 rows first."""
    qkv, pos, cs, qn, kn = heads_case(T, nq, nkv, hd, norm)
    loc = torch.randperm(160)[:T].to(torch.int32).cuda()
    loc[T // 2] = -1 if T > 1 else 3
    cache, want = (ops.KV8Cache.alloc(160, nkv, hd, dtype) for _ in range(2))
    q = ops.qk_norm_rope_store_kv8(qkv, pos, cs, qn, kn, 1e-6, cache, loc, nq)
    k, v = torch.zeros(2, T, nkv, hd, dtype=torch.bfloat16, device="cuda")
    at = torch.arange(T, dtype=torch.int32, device="cuda")
    assert torch.equal(q, ops.qk_norm_rope_store(qkv, pos, cs, qn, kn, 1e-6, k, v, at, nq, nkv, hd))
    ops.store_kv8(k, v, want, loc)
    assert same_cache(cache, want)


def test_heads_to_cache_without_tokens_and_beyond_tables():
    qkv, pos, cs, qn, kn = heads_case(3, 4, 2, 64, True)
    cache, want = (ops.KV8Cache.alloc(32, 2, 64, torch.int8) for _ in range(2))
    loc = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    q = ops.qk_norm_rope_store_kv8(qkv[:0], pos[:0], cs, qn, kn, 1e-6, cache, loc[:0], 4)
    assert q.shape == (0, 4, 64) and same_cache(cache, want)
    good = ops.qk_norm_rope_store_kv8(qkv, pos, cs, qn, kn, 1e-6, want, loc, 4)
    assert error_word()[0] == 0
    q = ops.qk_norm_rope_store_kv8(qkv, pos, cs, qn, kn, 1e-6, cache, torch.tensor([1, 32, 3], dtype=torch.int32, device="cuda"), 4)
    assert error_word()[0] == 3 and torch.equal(q, good)
    for t in (want.k, want.v, want.k_scale, want.v_scale):
        t[:, 2] = 0
    assert same_cache(cache, want)
    bad = pos.clone()
    bad[1] = 500
    q = ops.qk_norm_rope_store_kv8(qkv, bad, cs, qn, kn, 1e-6, cache, loc, 4)
    assert error_word()[0] == 3 and torch.equal(q[::2], good[::2])
    assert torch.equal(cache.k.view(torch.uint8), want.k.view(torch.uint8))  # (the bad token's key is not stored)


def test_heads_to_cache_captured():
    qkv, pos, cs, qn, kn = heads_case(4, 4, 2, 128, True)
    cache, want = (ops.KV8Cache.alloc(32, 2, 128, torch.float8_e4m3fn) for _ in range(2))
    loc = torch.tensor([1, 2, 3, 9], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    ops.qk_norm_rope_store_kv8(qkv, pos, cs, qn, kn, 1e-6, cache, loc, 4)
    with torch.cuda.graph(graph):
        q = ops.qk_norm_rope_store_kv8(qkv, pos, cs, qn, kn, 1e-6, cache, loc, 4)
    new = heads_case(4, 4, 2, 128, True, seed=1)
    qkv.copy_(new[0]), pos.copy_(new[1]), loc.add_(10)
    graph.replay()
    for at in (torch.tensor([1, 2, 3, 9], device="cuda"), loc):
        old = heads_case(4, 4, 2, 128, True) if at is not loc else (qkv, pos, cs, qn, kn)
        good = ops.qk_norm_rope_store_kv8(old[0], old[1], cs, qn, kn, 1e-6, want, at.to(torch.int32), 4)
    assert torch.equal(q, good) and same_cache(cache, want)


# ------------------------------------------------------------------------------- attention
# the form is chosen by max_q_len: both hold for every batch
HINTS = [1, 6, 1000]


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("nq,nkv,hd,page,window,sinks", [
    (4, 2, 128, 16, -1, False), (5, 1, 128, 32, -1, True), (8, 8, 64, 64, 20, False), (14, 2, 128, 48, 1, True),
    (16, 1, 64, 16, 64, True), (40, 8, 128, 64, -1, False), (17, 1, 128, 128, -1, False), (64, 8, 64, 32, 128, True),
])
def test_attention(hint, dtype, nq, nkv, hd, page, window, sinks):
    c = Case(RAGGED, nq, nkv, hd, dtype, page, window, sinks, tail=2).to("cuda")
    got = c.call(max_q_len=hint)
    c.check(got)
    assert (got[-2:] == 0).all()
    out = torch.full_like(c.q, 3.0)
    assert c.call(max_q_len=hint, out=out) is out
    assert torch.equal(out[:-2], got[:-2]) and (out[-2:] == 3).all()


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("reqs,nq,nkv", [
    ([(1, 5000)], 8, 1), ([(3, 4099)], 10, 2), ([(1, 64 * n + n % 3) for n in range(1, 34)], 6, 3), ([(40, 700), (1, 2000)], 5, 1),
    ([(130, 130)], 2, 1), ([(129, 1000)], 4, 2), ([(33, 33), (64, 100), (1, 1), (100, 613)], 7, 1), ([(2, 900), (2, 0), (9, 4)], 100, 1),
])
def test_long_and_many(hint, dtype, hd, reqs, nq, nkv):
    c = Case(reqs, nq, nkv, hd, dtype, 16 if hd == 64 else 64, seed=7).to("cuda")
    c.check(c.call(max_q_len=hint))


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("B,longest,tokens,nkv,window", [
    (300, 300, 1, 2, -1), (700, 200, 2, 3, -1), (150, 320, 9, 4, -1), (90, 510, 130, 4, -1), (60, 900, 200, 3, 100), (513, 64, 1, 8, 20),
])
def test_many_short_requests(hint, B, longest, tokens, nkv, window):
    """More requests than a CTA has threads, more segments than there are CTAs."""
    gen = torch.Generator().manual_seed(B)
    lens = torch.randint(1, longest + 1, (B,), generator=gen).tolist()
    reqs = [(min(1 + (7 * i) % tokens, n), n) for i, n in enumerate(lens)]
    reqs[3], reqs[B // 2] = (0, 10), (1, 0)
    c = Case(reqs, 4 * nkv, nkv, 64, torch.int8, 16, window, seed=B).to("cuda")
    got = c.call(max_q_len=hint)
    c.check(got)
    assert torch.equal(c.call(max_q_len=hint), got)


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("nq,nkv", [(128, 1), (130, 2), (96, 2), (64, 64)])
def test_groups_of_any_size(hint, nq, nkv):
    c = Case([(1, 100), (5, 77), (0, 9), (3, 2), (2, 500)], nq, nkv, 64, torch.int8, 16, sinks=True, seed=nq).to("cuda")
    c.check(c.call(max_q_len=hint))


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("window", [1, 63, 64, 65, 200, 10**6])
def test_windows(hint, dtype, window):
    c = Case([(1, 500), (70, 300), (3, 129), (1, 64)], 4, 2, 64, dtype, 32, window, sinks=True, seed=window).to("cuda")
    c.check(c.call(max_q_len=hint))


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("q_scale,k_size,v_size,scale", [
    (1e4, 1e-4, 1e20, None), (1e-30, 1e30, 1e-30, None), (1e30, 1e-30, 1.0, None), (1.5, 1.0, 1.0, -0.1), (1.5, 1.0, 1.0, 0.0), (0.0, 1.0, 1.0, None),
])
def test_extreme_sizes(hint, dtype, q_scale, k_size, v_size, scale):
    c = Case([(1, 200), (5, 70), (2, 2)], 4, 2, 128, dtype, 16, q_scale=q_scale, k_size=k_size, v_size=v_size, scale=scale).to("cuda")
    c.check(c.call(max_q_len=hint))


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("dtype", FMTS)
def test_values_of_very_different_sizes(hint, dtype):
    """The first token takes most of the softmax and has a value row of almost nothing; one value row is huge."""
    c = Case([(1, 600), (4, 90)], 8, 2, 64, dtype, 16, seed=11).to("cuda")
    for b in range(2):
        table = c.table[int(c.rows[b])]
        c.cache.k_scale[:, int(table[0])] *= 6
        c.cache.v_scale[:, int(table[0])] *= 1e-12
        c.cache.v_scale[:, int(table[70])] *= 1e6
        c.cache.v_scale[:, int(table[71])] = 0
    c.check(c.call(max_q_len=hint))


@pytest.mark.parametrize("hint", HINTS)
def test_a_seen_row_without_a_scale(hint):
    c = Case([(3, 40)], 4, 2, 64, torch.int8, window=4).to("cuda")
    slot = int(c.table[int(c.rows[0]), 35])
    c.cache.v_scale[1, slot] = math.nan
    got = c.call(max_q_len=hint)
    assert got[:2, 2:].isnan().all() and got[2].isfinite().all() and got[:, :2].isfinite().all()
    c.cache.v_scale[1, slot] = 1
    c.cache.k_scale[0, slot] = math.nan
    got = c.call(max_q_len=hint)
    assert got[:2, :2].isnan().all() and got[2].isfinite().all() and got[:, 2:].isfinite().all()


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("hd", [64, 128])
def test_strided_queries(hint, hd):
    c = Case([(2, 30), (1, 70)], 4, 2, hd, torch.int8).to("cuda")
    want = c.call(max_q_len=hint)
    merged = torch.randn(3, 8 * hd + 8, dtype=torch.bfloat16, device="cuda")
    merged[:, : 4 * hd] = c.q.flatten(1)
    q = c.q
    c.q = merged[:, : 4 * hd].unflatten(1, (4, hd))
    assert torch.equal(c.call(max_q_len=hint), want)
    c.q = torch.stack([q, q], 2)[:, :, 1]
    assert torch.equal(c.call(max_q_len=hint), want)
    c.q = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(c.call(max_q_len=hint), want)
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    c.q = odd
    assert torch.equal(c.call(max_q_len=hint), want)
    wide = torch.full((c.table.shape[0], 200), -9, dtype=torch.int32, device="cuda")
    wide[:, 3 : 3 + c.table.shape[1]] = c.table
    c.q, c.table = q, wide[:, 3:]
    assert torch.equal(c.call(max_q_len=hint), want)


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("dtype", FMTS)
def test_equal_calls_give_equal_results(hint, dtype):
    c = Case([(1, 3000)] * 3 + [(20, 900)], 8, 2, 128, dtype, 64).to("cuda")
    first = c.call(max_q_len=hint)
    for _ in range(5):
        assert torch.equal(c.call(max_q_len=hint), first)


@pytest.mark.parametrize("hint", HINTS)
def test_entries_outside_their_tables_are_recorded(hint):
    def fresh():
        return Case([(2, 20), (1, 40), (2, 70)], 4, 2, 64, torch.int8).to("cuda")

    c = fresh()
    want = c.call(max_q_len=hint)
    sound = [slice(2, None), slice(0, 2)]
    for name, at, value, keep in (("rows", 0, 99, sound[0]), ("rows", 0, -1, sound[0]), ("kv_lens", 0, 10**6, sound[0]),
                                  ("kv_lens", 0, -4, sound[0]), ("cu_q", 3, 9, slice(0, 3)), ("cu_q", 0, -2, sound[0]),
                                  ("cu_q", 0, 1, sound[0])):
        c = fresh()
        getattr(c, name)[at] = value
        got = c.call(max_q_len=hint)
        assert torch.equal(got[keep], want[keep])
        assert error_word()[0] == 3, name
    for slot in (-1, 8, c.cache.num_slots, c.cache.num_slots - 8, 2**31 - 16, -(2**31)):
        c = fresh()
        c.table[c.rows[0].long(), 0] = slot
        got = c.call(max_q_len=hint)
        assert got[:2].isfinite().all() and torch.equal(got[2:], want[2:])
        assert error_word()[0] == 3, slot


@pytest.mark.parametrize("hint", HINTS)
def test_graph_replays_with_new_lengths(hint):
    a = Case([(1, 900), (1, 30), (1, 1)], 8, 2, 128, torch.int8, 16, seed=1, width=1024).to("cuda")
    b = Case([(1, 40), (1, 1000), (1, 0)], 8, 2, 128, torch.int8, 16, seed=2, width=1024).to("cuda")
    size = max(a.cache.num_slots, b.cache.num_slots)
    live = ops.KV8Cache.alloc(size, 2, 128)
    c = Case([(1, 16)] * 3, 8, 2, 128, torch.int8, 16, width=1024).to("cuda")
    c.cache = live
    torch.cuda.synchronize()

    def call():
        ops.store_kv8(new, new, live, loc)
        return c.call(max_q_len=hint)

    def load(x):
        # (its scales, where it has slots: the rest holds no position)
        for dst, src in ((live.k, x.cache.k), (live.v, x.cache.v), (live.k_scale, x.cache.k_scale), (live.v_scale, x.cache.v_scale)):
            dst[:, : src.shape[1]].copy_(src)
        for n in ("table", "rows", "kv_lens", "q"):
            getattr(c, n).copy_(getattr(x, n))

    new = torch.randn(1, 2, 128, device="cuda").to(torch.bfloat16)
    loc = torch.tensor([-1], dtype=torch.int32, device="cuda")
    load(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for x in (b, a, b):
        load(x)
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            x.check(out)


def test_calls_on_several_streams():
    cases = [Case([(1, 1500)] * 4 + [(30, 400)], 8, 2, 64, dtype, 16, seed=i).to("cuda") for i, dtype in enumerate(FMTS * 2)]
    want = [[c.call(max_q_len=h) for h in HINTS] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append([c.call(max_q_len=h) for h in HINTS])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.parametrize("hint", HINTS)
def test_cache_beyond_32_bits(hint):
    """4.6 GB of codes each: the last pages give what the same rows give in a small cache."""
    nq, nkv, hd, n, slots = 32, 16, 128, 300, 2_240_000
    gen = torch.Generator().manual_seed(5)
    k, v = (rows_of(gen, n, nkv, hd).cuda() for _ in range(2))
    q = torch.randn(2, nq, hd, generator=gen).to(torch.bfloat16).cuda()
    rows, ends, lens = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0], [0, 2], [n]))
    got = []
    for size in (512, slots):
        cache = ops.KV8Cache.alloc(size, nkv, hd, torch.int8)
        at = torch.arange(size - 512, size, dtype=torch.int32, device="cuda").view(-1, 64)[torch.arange(7, -1, -1, device="cuda")].flatten()
        ops.store_kv8(k, v, cache, at[:n].contiguous())
        back = ops.load_kv8(cache, at[:n].contiguous())
        got.append((ops.attention_kv8(q, cache, at[None], rows, ends, lens, page_size=64, max_q_len=hint), *back))
        assert not cache.k[0, : size - 512].any()
        del cache
    assert got[0][0].isfinite().all() and got[0][0].any()
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_as_a_model_uses_them():
    """A prompt in two chunks, then single tokens: every step's rows are stored, then attended to."""
    torch.manual_seed(0)
    nq, nkv, hd, page, n = 10, 2, 128, 16, 150
    for dtype in FMTS:
        cache = ops.KV8Cache.alloc(320, nkv, hd, dtype)
        table = torch.arange(320, dtype=torch.int32).view(20, 16)[torch.randperm(20)].flatten()[None].cuda()
        q, k, v = (torch.randn(n, h, hd).to(torch.bfloat16).cuda() for h in (nq, nkv, nkv))
        near = []
        for x in (k, v):
            code, s = nearest(x, dtype)
            near.append(code * s)
        at = 0
        row = torch.zeros(1, dtype=torch.int32, device="cuda")
        for step in [100, 37] + [1] * 13:
            loc = table[0, at : at + step].contiguous()
            ops.store_kv8(k[at : at + step], v[at : at + step], cache, loc)
            ends, lens = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, step], [at + step]))
            got = ops.attention_kv8(q[at : at + step], cache, table, row, ends, lens, page_size=page, max_q_len=step).cpu().double()
            for i in range(step):
                kx, vx = (t[: at + i + 1].repeat_interleave(nq // nkv, 1).transpose(0, 1) for t in near)
                x = (q[at + i].cpu().double().unsqueeze(1) * kx).sum(-1) / math.sqrt(hd)
                p = torch.softmax(x, -1).unsqueeze(-1)
                want, A = (p * vx).sum(1), (p * vx.abs()).sum(1)
                # as Case.exact counts, with logits of at most 2^7 in all their terms, and a scale rounded to fp32
                assert ((got[i] - want).abs() <= want.abs() * 2.0**-8 + A * (2.0**-11 + 2.0**-7)).all()
            at += step


@pytest.mark.parametrize("name,call", [(n, i) for i, (n, _) in enumerate(bad_calls("cpu"))],
                         ids=lambda v: v.replace(" ", "_") if isinstance(v, str) else "")
def test_refusals(name, call):
    with pytest.raises((ValueError, RuntimeError)):
        bad_calls("cuda")[call][1]()


def test_tensors_of_two_devices():
    c = Case([(1, 5)], 4, 2, 64, torch.int8).to("cuda")
    for n in ("q", "table", "rows", "cu_q", "kv_lens"):
        keep = getattr(c, n)
        setattr(c, n, keep.cpu())
        with pytest.raises((ValueError, RuntimeError), match="device"):
            c.call()
        setattr(c, n, keep)
    with pytest.raises((ValueError, RuntimeError), match="device"):
        ops.load_kv8(c.cache, torch.zeros(1, dtype=torch.int32))
