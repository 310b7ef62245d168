"""The 8-bit key/value cache on CPU tensors: the plain form against 64 bits, and what is refused."""

import math

import pytest
import torch

from kv8_cases import FMTS, RAGGED, Case, bad_calls, nearest, values
from minisgl import ops


@pytest.mark.parametrize("dtype", FMTS)
def test_rows_are_rounded_to_the_nearest_code(dtype):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(50, 2, 64, generator=gen) * torch.randn(50, 2, 1, generator=gen).mul(3).exp()
    x[0] = 0
    x[1, 0] = torch.linspace(-1, 1, 64)  # the largest on both sides, and halves of it
    x[1, 1, ::2] = 0.5
    x = x.to(torch.bfloat16)
    codes, scale = ops.ref.quantise_kv8(x, dtype)
    want, s = nearest(x, dtype)
    assert torch.equal(values(codes.transpose(0, 1), torch.ones(2, 50)), want.transpose(0, 1))
    assert torch.equal(scale, (s.squeeze(-1) * 1.0).float()) or ((scale - s.squeeze(-1)).abs() <= s.squeeze(-1) * 2.0**-24).all()
    assert (scale[0] == 0).all() and (codes[0].float() == 0).all()


@pytest.mark.parametrize("dtype", FMTS)
def test_rows_without_finite_values_have_no_scale(dtype):
    x = torch.ones(3, 1, 64, dtype=torch.bfloat16)
    x[0, 0, 5], x[1, 0, 6] = math.inf, math.nan
    codes, scale = ops.ref.quantise_kv8(x, dtype)
    assert scale[:2].isnan().all() and scale[2].isfinite().all() and (codes[:2].float() == 0).all()


@pytest.mark.parametrize("dtype", FMTS)
def test_store_and_load(dtype):
    gen = torch.Generator().manual_seed(2)
    cache = ops.KV8Cache.alloc(32, 2, 64, dtype, "cpu")
    k, v = (torch.randn(4, 2, 64, generator=gen).to(torch.bfloat16) for _ in range(2))
    loc = torch.tensor([5, -1, 31, 0], dtype=torch.int32)
    ops.store_kv8(k, v, cache, loc)
    got_k, got_v = ops.load_kv8(cache, torch.tensor([31, 0, -3, 5, 1, 5], dtype=torch.int32))
    for x, got in ((k, got_k), (v, got_v)):
        near, s = nearest(x, dtype)
        rows = near * s
        want = torch.stack([rows[2], rows[3], torch.zeros(2, 64), rows[0], torch.zeros(2, 64), rows[0]])
        assert ((got.double() - want).abs() <= want.abs() * (2.0**-8 + 2.0**-22)).all()
    with pytest.raises(ValueError, match="slot 32"):
        ops.store_kv8(k, v, cache, torch.tensor([0, 32, 1, 2], dtype=torch.int32))
    with pytest.raises(ValueError, match="slot 40"):
        ops.load_kv8(cache, torch.tensor([40], dtype=torch.int32))
    assert cache.nbytes() == 2 * 2 * 32 * 68


@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("nq,nkv,hd,page,window,sinks", [(4, 2, 64, 16, -1, False), (5, 1, 128, 32, -1, True), (8, 8, 64, 64, 20, False),
                                                         (14, 2, 64, 48, 1, True)])
def test_attention_against_64_bits(dtype, nq, nkv, hd, page, window, sinks):
    c = Case(RAGGED, nq, nkv, hd, dtype, page, window, sinks, tail=2)
    got = c.call()
    c.check(got)
    assert (got[-2:] == 0).all()
    out = torch.full_like(c.q, 3.0)
    assert c.call(out=out) is out and torch.equal(out[:-2], got[:-2]) and (out[-2:] == 3).all()


def test_a_seen_row_without_a_scale_makes_its_queries_no_numbers():
    c = Case([(3, 40)], 4, 2, 64, torch.int8, window=4)
    slot = int(c.table[int(c.rows[0]), 35])  # seen by the first two queries (34..37, 35..38), not by the last
    c.cache.v_scale[1, slot] = math.nan
    got = c.call()
    assert got[:2, 2:].isnan().all() and got[2].isfinite().all() and got[:, :2].isfinite().all()


def test_tables_that_do_not_hold():
    c = Case([(2, 20)], 4, 2, 64, torch.int8)
    for name, bad in (("rows", torch.tensor([9])), ("kv_lens", torch.tensor([33])), ("cu_q", torch.tensor([0, 3])),
                      ("cu_q", torch.tensor([1, 2]))):
        keep = getattr(c, name)
        setattr(c, name, bad.to(torch.int32))
        with pytest.raises(ValueError, match="attention_kv8"):
            c.call()
        setattr(c, name, keep)
    for slot in (-1, 8, 16 * 5):
        c.table[c.rows.long(), 16] = slot
        with pytest.raises(ValueError, match="page"):
            c.call()


@pytest.mark.parametrize("name,call", bad_calls("cpu"), ids=lambda v: v.replace(" ", "_") if isinstance(v, str) else "")
def test_refusals(name, call):
    with pytest.raises(ValueError):
        call()


# --------------------------------------------------------------------------------- fused store
@pytest.mark.parametrize("dtype", FMTS)
@pytest.mark.parametrize("norm", [True, False])
def test_heads_to_cache(dtype, norm):
    gen = torch.Generator().manual_seed(3)
    T, nq, nkv, hd = 5, 6, 2, 64
    qkv = torch.randn(T, (nq + 2 * nkv) * hd, generator=gen).to(torch.bfloat16)
    pos = torch.tensor([3, 0, 9, 9, 1], dtype=torch.int32)
    cs = ops.ref.rope_cos_sin(10, hd, ops.ref.default_inv_freq(hd, 1e4))
    qn, kn = (torch.randn(2, hd, generator=gen).to(torch.bfloat16)) if norm else (None, None)
    loc = torch.tensor([4, 17, -1, 30, 0], dtype=torch.int32)
    cache, want = (ops.KV8Cache.alloc(32, nkv, hd, dtype, "cpu") for _ in range(2))
    q = ops.qk_norm_rope_store_kv8(qkv, pos, cs, qn, kn, 1e-6, cache, loc, nq)
    heads = qkv.view(T, -1, hd)
    hq, hk = heads[:, :nq], heads[:, nq:nq + nkv]
    if norm:
        hq, hk = ops.ref.rmsnorm(hq, qn, 1e-6), ops.ref.rmsnorm(hk, kn, 1e-6)
    assert torch.equal(q, ops.ref.rope(hq, pos, cs))
    ops.store_kv8(ops.ref.rope(hk, pos, cs), heads[:, nq + nkv:], want, loc)
    for a, b in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), (want.k, want.v, want.k_scale, want.v_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    with pytest.raises(ValueError):
        ops.qk_norm_rope_store_kv8(qkv, pos + 1, cs, qn, kn, 1e-6, cache, loc, nq)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_store_kv8(qkv, pos, cs, qn, kn, 1e-6, cache, loc + 2, nq)
