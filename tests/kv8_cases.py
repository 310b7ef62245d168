"""Cases of the 8-bit key/value cache and their results in 64 bits, shared by its CPU and GPU tests."""

import math
import random

import torch

from minisgl import ops

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FMTS = [torch.int8, torch.float8_e4m3fn]


def e4m3_values():
    """The value of each of the 256 codes, from the format's definition."""
    out = []
    for b in range(256):
        s, e, m = b >> 7, (b >> 3) & 15, b & 7
        v = m * 2.0**-9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(math.nan if (e, m) == (15, 7) else -v if s else v)
    return torch.tensor(out, dtype=torch.float64)


def values(codes, scale):
    """What codes [h, n, hd] and scales [h, n] stand for, in 64 bits, on the CPU."""
    codes = codes.cpu()
    if codes.dtype == torch.int8:
        v = codes.double()
    else:
        v = e4m3_values()[codes.view(torch.uint8).long()]
    return v * scale.cpu().double().unsqueeze(-1)


def nearest(x, dtype):
    """(codes' values, scale) of rows x, in 64 bits: the nearest of the format's values, ties to the even code."""
    x = x.cpu().double()
    top = x.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, x * LARGEST[dtype] / top, 0.0)
    if dtype == torch.int8:
        return q.round(), top / 127.0
    grid = e4m3_values()[:127]  # rising
    hi = torch.searchsorted(grid, q.abs()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - q.abs(), q.abs() - grid[lo]
    take = torch.where(up < down, hi, torch.where(up > down, lo, torch.where(hi % 2 == 0, hi, lo)))
    return grid[take] * q.sign(), top / 448.0


class Case:
    """A batch of requests over a paged cache with shuffled pages; slots that hold no position are unfit for use."""

    def __init__(self, reqs, nq, nkv, hd, dtype, page=16, window=-1, sinks=False, seed=0, width=None, tail=0, q_scale=1.5,
                 k_size=1.0, v_size=1.0, scale=None):
        self.reqs, self.page, self.window, self.dtype, self.scale = reqs, page, window, dtype, scale
        gen = torch.Generator().manual_seed(seed)
        pages = [-(-L // page) for _, L in reqs]
        total = sum(pages) + 3
        slots = total * page
        rows = torch.randn(2, nkv, slots, hd, generator=gen) * torch.randn(hd, generator=gen).mul(0.5).exp()
        rows *= torch.randn(2, nkv, slots, 1, generator=gen).mul(0.4).exp()
        rows[0] *= k_size
        rows[1] *= v_size
        codes, scales = ops.ref.quantise_kv8(rows.to(torch.bfloat16), dtype)
        order = list(range(total))
        random.Random(seed).shuffle(order)
        B = len(reqs)
        width = max([1] + [n * page for n in pages]) if width is None else width
        table = torch.full((B + 2, width), -7, dtype=torch.int32)  # what is not a position's slot is no slot at all
        back = torch.randperm(B + 2, generator=gen)[:B]
        used = torch.zeros(slots, dtype=torch.bool)
        at = 0
        for b, (n, (_, L)) in enumerate(zip(pages, reqs)):
            s = (torch.tensor(order[at : at + n], dtype=torch.int32)[:, None] * page + torch.arange(page, dtype=torch.int32)).flatten()[:L]
            table[back[b], :L] = s
            used[s.long()] = True
            at += n
        # unused slots: no numbers
        scales[:, :, ~used] = math.nan
        if dtype == torch.float8_e4m3fn:
            codes.view(torch.uint8)[:, :, ~used] = 0x7F
        self.codes, self.scales = codes, scales
        self.cache = ops.KV8Cache(codes[0].clone(), codes[1].clone(), scales[0].clone(), scales[1].clone())
        self.table, self.rows = table, back.to(torch.int32)
        self.cu_q = torch.tensor([0] + [n for n, _ in reqs]).cumsum(0).to(torch.int32)
        self.kv_lens = torch.tensor([L for _, L in reqs], dtype=torch.int32)
        self.q = (torch.randn(int(self.cu_q[-1]) + tail, nq, hd, generator=gen) * q_scale).to(torch.bfloat16)
        self.sinks = torch.randn(nq, generator=gen) * 2 if sinks else None

    def to(self, dev):
        c = self.cache
        self.cache = ops.KV8Cache(*(t.to(dev) for t in (c.k, c.v, c.k_scale, c.v_scale)))
        for n in ("table", "rows", "cu_q", "kv_lens", "q", "sinks"):
            t = getattr(self, n)
            setattr(self, n, None if t is None else t.to(dev))
        return self

    def call(self, **kw):
        kw = dict(dict(page_size=self.page, window=self.window, sinks=self.sinks, scale=self.scale), **kw)
        return ops.attention_kv8(self.q, self.cache, self.table, self.rows, self.cu_q, self.kv_lens, **kw)

    def exact(self):
        """(result, bound of the error) in 64 bits. With A = sum_j p_j |v_j| the kernels' result differs by at most
        half a bf16 step of the value; half an fp16 step (2^-11) of A, for the weights p_j s^v_j; 2 d A for logits that are
        off by at most d, in the weights and in their sum: an fp32 product sum of hd terms, each addition off by at
        most 2^-23 of the terms' total, and the rounding of its scale, of the maximum taken off it and of the power of 2;
        and 2 (L / 8 + 16) 2^-23 A for the sums over L keys, added 8 at a time at least.

        Half an fp16 step of a weight is 2^-11 of it where fp16 is normal, but not less than half of the smallest step,
        2^-25. Weights p_j s^v_j are scaled so that the largest one, M, comes to 2^6 at least (the streaming form's to 2^14;
        for a warp that has not seen the largest yet the step is a smaller part of M): each of them can be off by
        2^-25 / 2^6 M, together by 2^-31 M sum_j |c_j|. That is what is left of a head dim in which the keys that count
        have codes of 0."""
        q, sinks = self.q.cpu().double(), None if self.sinks is None else self.sinks.cpu().double()
        T, nq, hd = q.shape
        c = self.cache
        kx, vx = values(c.k, c.k_scale), values(c.v, c.v_scale)
        cx, sx = values(c.v, torch.ones_like(c.v_scale)).abs(), c.v_scale.cpu().double()
        g = nq // kx.shape[0]
        out, tol = torch.zeros_like(q), torch.zeros_like(q)
        scale = hd**-0.5 if self.scale is None else self.scale
        at = 0
        for b, (n, L) in enumerate(self.reqs):
            slots = self.table[int(self.rows[b]), :L].cpu().long()
            for i in range(n):
                pos = L - n + i
                first = max(0, pos - self.window + 1) if self.window > 0 else 0
                if pos < 0:
                    continue
                s = slots[first : pos + 1]
                k, v = kx[:, s].repeat_interleave(g, 0), vx[:, s].repeat_interleave(g, 0)  # [nq, m, hd]
                x = (q[at + i].unsqueeze(1) * k).sum(-1) * scale
                big = (q[at + i].unsqueeze(1) * k).abs().sum(-1).amax(-1) * abs(scale) + x.abs().amax(-1)
                if sinks is not None:
                    x = torch.cat([x, sinks[:, None]], 1)
                p = torch.softmax(x, -1)[:, : len(s)].unsqueeze(-1)
                out[at + i] = (p * v).sum(1)
                d = ((hd + 16) * big + 16) * 2.0**-23
                A = (p * v.abs()).sum(1)
                M = (p.squeeze(-1) * sx[:, s].repeat_interleave(g, 0)).amax(-1, keepdim=True)
                least = 2.0**-31 * M * cx[:, s].repeat_interleave(g, 0).sum(1)
                tol[at + i] = out[at + i].abs() * 2.0**-8 + A * (2.0**-11 + 2 * d.unsqueeze(-1) + 2 * (len(s) / 8 + 16) * 2.0**-23) + least + 1e-37
            at += n
        return out, tol

    def check(self, got):
        want, tol = self.exact()
        n = int(self.cu_q[-1])
        got = got.cpu().double()
        assert torch.isfinite(got[:n]).all()
        bad = (got[:n] - want[:n]).abs() > tol[:n]
        assert not bad.any(), (bad.nonzero()[:5].tolist(), float(((got[:n] - want[:n]).abs() / tol[:n]).max()))


# what the calls have to get right: (queries, keys) of the requests
RAGGED = [(1, 1), (1, 16), (3, 17), (1, 0), (2, 64), (0, 40), (5, 65), (1, 127), (7, 7), (4, 129), (1, 300), (2, 1)]


def bad_calls(dev):
    """(name, call) of what is refused before anything is copied or launched"""
    c = Case([(2, 20), (1, 5)], 4, 2, 64, torch.int8).to(dev)
    bf16, i32 = torch.bfloat16, torch.int32
    zeros = lambda *shape, dtype=torch.float32: torch.zeros(*shape, device=dev, dtype=dtype)  # noqa: E731
    kv = zeros(3, 2, 64, dtype=bf16)
    loc = zeros(3, dtype=i32)
    k = c.cache

    def attend(q=c.q, table=c.table, rows=c.rows, cu_q=c.cu_q, kv_lens=c.kv_lens, page_size=16, cache=k, **kw):
        return ops.attention_kv8(q, cache, table, rows, cu_q, kv_lens, page_size=page_size, **kw)

    def cache(**kw):
        t = dict(dict(k=k.k, v=k.v, k_scale=k.k_scale, v_scale=k.v_scale), **kw)
        return ops.KV8Cache(t["k"], t["v"], t["k_scale"], t["v_scale"])

    heads = zeros(3, 8 * 64, dtype=bf16)

    def fused(qkv=heads, pos=loc, cs=zeros(4, 64), qn=None, kn=None, at=loc, nq=4):
        return ops.qk_norm_rope_store_kv8(qkv, pos, cs, qn, kn, 1e-6, k, at, nq)

    long = zeros(3, 16, 64, dtype=torch.int8)
    odd = zeros(2, 24, 64, dtype=torch.int8)
    wide = zeros(2, 16, 96, dtype=torch.int8)
    return [
        ("codes in uint8", lambda: cache(k=k.k.view(torch.uint8))),
        ("codes of two types", lambda: cache(v=k.v.view(torch.float8_e4m3fn))),
        ("codes of one row", lambda: cache(k=k.k[0])),
        ("values of another length", lambda: cache(v=k.v[:, :16].contiguous())),
        ("scales in bf16", lambda: cache(k_scale=k.k_scale.to(bf16))),
        ("short scales", lambda: cache(v_scale=k.v_scale[:, :16].contiguous())),
        ("strided codes", lambda: cache(k=k.k.transpose(0, 1).contiguous().transpose(0, 1))),
        ("one tensor for both codes", lambda: cache(v=k.k)),
        ("one tensor for both scales", lambda: cache(v_scale=k.k_scale)),
        ("codes that overlap", lambda: ops.KV8Cache(long[:2], long[1:], k.k_scale[:, :16].contiguous(), k.v_scale[:, :16].contiguous())),
        ("24 slots", lambda: ops.KV8Cache(odd, odd, zeros(2, 24), zeros(2, 24))),
        ("head dim 96", lambda: ops.KV8Cache(wide, wide, zeros(2, 16), zeros(2, 16))),
        ("a cache in bf16", lambda: ops.KV8Cache.alloc(16, 2, 64, bf16, dev)),
        ("k in 32 bits", lambda: ops.store_kv8(kv.float(), kv, k, loc)),
        ("v of three heads", lambda: ops.store_kv8(kv, zeros(3, 3, 64, dtype=bf16), k, loc)),
        ("k of wide heads", lambda: ops.store_kv8(zeros(3, 2, 128, dtype=bf16), kv, k, loc)),
        ("fewer values", lambda: ops.store_kv8(kv, kv[:2], k, loc)),
        ("flat rows", lambda: ops.store_kv8(kv.flatten(1), kv.flatten(1), k, loc)),
        ("slots in 64 bits", lambda: ops.store_kv8(kv, kv, k, loc.long())),
        ("too few slots", lambda: ops.store_kv8(kv, kv, k, loc[:2])),
        ("strided slots", lambda: ops.store_kv8(kv, kv, k, zeros(6, dtype=i32)[::2])),
        ("heads of 32 bits", lambda: fused(qkv=heads.float())),
        ("heads of a cache with more", lambda: fused(nq=2)),
        ("no query heads", lambda: fused(nq=0)),
        ("strided heads", lambda: fused(qkv=zeros(3, 2 * 8 * 64, dtype=bf16)[:, ::2])),
        ("positions in 64 bits", lambda: fused(pos=loc.long())),
        ("fewer positions", lambda: fused(pos=loc[:2])),
        ("angles in bf16", lambda: fused(cs=zeros(4, 64, dtype=bf16))),
        ("angles of wide heads", lambda: fused(cs=zeros(4, 128))),
        ("a norm of queries alone", lambda: fused(qn=zeros(64, dtype=bf16))),
        ("norms in 32 bits", lambda: fused(qn=zeros(64), kn=zeros(64))),
        ("norms of wide heads", lambda: fused(qn=zeros(128, dtype=bf16), kn=zeros(128, dtype=bf16))),
        ("too few slots for the heads", lambda: fused(at=loc[:2])),
        ("read at 64-bit slots", lambda: ops.load_kv8(k, loc.long())),
        ("read at a table of slots", lambda: ops.load_kv8(k, loc[None])),
        ("q in 32 bits", lambda: attend(q=c.q.float())),
        ("q of one row", lambda: attend(q=c.q[0])),
        ("q of wide heads", lambda: attend(q=zeros(3, 4, 128, dtype=bf16))),
        ("three heads over two", lambda: attend(q=zeros(3, 3, 64, dtype=bf16))),
        ("no heads", lambda: attend(q=zeros(3, 0, 64, dtype=bf16))),
        ("258 heads over two", lambda: attend(q=zeros(3, 258, 64, dtype=bf16))),
        ("a table in 64 bits", lambda: attend(table=c.table.long())),
        ("a table of one row", lambda: attend(table=c.table[0])),
        ("a turned table", lambda: attend(table=c.table.t().contiguous().t())),
        ("too few ends", lambda: attend(cu_q=c.cu_q[:-1])),
        ("too many lengths", lambda: attend(kv_lens=zeros(3, dtype=i32))),
        ("lengths in 64 bits", lambda: attend(kv_lens=c.kv_lens.long())),
        ("pages of 8", lambda: attend(page_size=8)),
        ("pages of 24", lambda: attend(page_size=24)),
        ("no page", lambda: attend(page_size=0)),
        ("a negative max_q_len", lambda: attend(max_q_len=-2)),
        ("a window of 0", lambda: attend(window=0)),
        ("a window of -2", lambda: attend(window=-2)),
        ("an infinite scale", lambda: attend(scale=math.inf)),
        ("a scale that is no number", lambda: attend(scale=math.nan)),
        ("sinks in bf16", lambda: attend(sinks=zeros(4, dtype=bf16))),
        ("sinks of three heads", lambda: attend(sinks=zeros(3))),
        ("strided sinks", lambda: attend(sinks=zeros(8)[::2])),
        ("out in 32 bits", lambda: attend(out=zeros(3, 4, 64))),
        ("a short out", lambda: attend(out=zeros(2, 4, 64, dtype=bf16))),
        ("a strided out", lambda: attend(out=zeros(3, 8, 64, dtype=bf16)[:, ::2])),
        ("out over q", lambda: attend(out=c.q)),
    ]


# ------------------------------------------------------------------------------------ engines
# Logits of an engine with an 8-bit cache against an fp32 engine whose cache rows are rounded to the same codes. Without
# codes a bf16 engine is within 0.06 of fp32 on the tiny models. A row that bf16 arithmetic moves by d (about 2^-9 of it)
# changes codes where it crosses a tie: on average by sqrt(d * step), with a step of 2^-7 of the row's largest value
# (int8), up to 2^-3 of the value itself (e4m3): 2 and 8 times a bf16 rounding of the row. A layer has some 20
# bf16 roundings, 2 of them of cached rows; in squares (20 + 2 * 2^2) / 20 = 1.1^2 and (20 + 2 * 8^2) / 20 = 2.7^2.
ENGINE_TOL = {"int8": 1.1 * 0.06, "fp8_e4m3": 2.7 * 0.06}


def round_cache_rows(monkeypatch, name):
    """Engines on the CPU store the values of 8-bit codes instead of the rows."""
    dtype = {"int8": torch.int8, "fp8_e4m3": torch.float8_e4m3fn}[name]

    def store_kv(k, v, k_cache, v_cache, out_loc):
        for x, cache in ((k, k_cache), (v, v_cache)):
            codes, scale = nearest(x.to(torch.bfloat16), dtype)
            cache.view(cache.shape[0], -1)[out_loc.long()] = (codes * scale).flatten(1).to(cache.dtype)

    monkeypatch.setattr(ops.ref, "store_kv", store_kv)
