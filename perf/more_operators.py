"""Measured cases of the 8-bit key/value cache: quantising it as it is written, reading it back, and
attention of new tokens over it.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes a case's
inputs on the GPU from a seed, and ``run()`` is one pass: the framework's operators where ``own`` is
true, elementary torch operations otherwise. ``exact()`` is the same result in 64 bits, written
apart from both, and ``work()`` the bytes and operations that a pass cannot do without.

The cache holds, per kv head and slot (one token), the codes of a key and of a value row and one fp32
scale each: ``codes [kv heads, slots, head dim]`` in int8 or e4m3, ``scales [kv heads, slots]``. A row's
scale is its largest magnitude over 127 (int8) or 448 (e4m3), its codes are the nearest ones to
``value / scale`` (ties to even), and it stands for ``code * scale``. ``page_table[row, position]`` is the
slot of a position of the request in that row; pages are runs of consecutive slots. The queries of
request b are the last ones of its ``kv_lens[b]`` positions, and a query sees the keys up to its own
position (with a window, the last ``window`` of them). A sink is a logit that takes its share of the
softmax and adds no value. A query that sees no key gives zeros.
"""

import math
import random

import torch

own = False

DEV = "cuda"
LARGEST = {"int8": 127.0, "e4m3": 448.0}
DTYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


# ---------------------------------------------------------------------------------------- cases
def _attend(name, B, new, cached, heads, hd, page, fmt, window=-1, sinks=False, padded=0):
    return dict(name=name, op="attend", B=B, new_lo=new[0], new_hi=new[1], cached_lo=cached[0], cached_hi=cached[1],
                nq=heads[0], nkv=heads[1], hd=hd, page=page, fmt=fmt, window=window, sinks=sinks, padded=padded)


def listed():
    return [
        # one decoded token's keys and values go into one layer's cache: latency
        dict(name="write and read 1x8x128 int8", op="write", T=1, nkv=8, hd=128, fmt="int8"),
        # a prompt's chunk at once: bytes
        dict(name="write and read 16384x8x128 e4m3", op="write", T=16384, nkv=8, hd=128, fmt="e4m3"),
        # an odd batch of a tensor-parallel rank with two kv heads
        dict(name="write and read 777x2x64 int8", op="write", T=777, nkv=2, hd=64, fmt="int8"),
        # a long cached prefix is read back, page after page
        dict(name="read 120000x8x128 int8", op="read", T=120000, nkv=8, hd=128, fmt="int8"),
        # a few tokens are looked at
        dict(name="read 33x8x64 e4m3", op="read", T=33, nkv=8, hd=64, fmt="e4m3"),
        # one decoded token after a thousand: latency
        _attend("decode 1 at 1000 int8", 1, (1, 1), (999, 999), (40, 8), 128, 16, "int8"),
        # a decode batch of mixed lengths with a padded request: the cache's bytes
        _attend("decode 128 at 100 to 2048 e4m3", 128, (1, 1), (99, 2047), (40, 8), 128, 64, "e4m3", padded=1),
        # long contexts, few requests: one request's keys are spread over many processors
        _attend("decode 4 at 100000 int8", 4, (1, 1), (99000, 101000), (64, 8), 128, 32, "int8"),
        # a few drafted tokens of every request are verified at once
        _attend("verify 5 of 16 at 6000 e4m3", 16, (4, 5), (3000, 9000), (40, 8), 128, 16, "e4m3"),
        # a chunk of a long prompt, most of it cached already
        _attend("chunk 2048 after 30000 int8", 1, (2048, 2048), (30000, 30000), (40, 8), 128, 64, "int8"),
        # a batch of whole prompts
        _attend("prompts 28 of 100 to 1024 e4m3", 28, (100, 1024), (0, 0), (40, 8), 128, 16, "e4m3"),
        # narrow heads, a sliding window and sinks; odd chunks of three requests
        _attend("chunk 777 window 128 sinks int8", 3, (333, 777), (0, 5000), (64, 8), 64, 32, "int8", window=128, sinks=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend"])
    hd, fmt = rng.choice([64, 128]), rng.choice(["int8", "e4m3"])
    if op != "attend":
        nkv = rng.choice([1, 2, 4, 8])
        return dict(op=op, T=_log_int(rng, 1, 16384 if op == "write" else 120000), nkv=nkv, hd=hd, fmt=fmt)
    nkv = rng.choice([1, 2, 4, 8])
    c = dict(op=op, nq=nkv * rng.choice([1, 2, 4, 5, 7, 8]), nkv=nkv, hd=hd, page=rng.choice([16, 32, 64]), fmt=fmt,
             window=rng.choice([-1, -1, -1, 128, 1000]), sinks=rng.random() < 0.3, padded=rng.choice([0, 0, 1, 3]))
    kind = rng.choice(["decode", "verify", "chunk"])
    if kind == "chunk":
        n = _log_int(rng, 17, 2048)
        B = rng.randint(1, max(1, min(28, 16384 // n)))
        most = max(1, min(30000, 2048 * 30000 // (B * n)))
        hi = rng.choice([0, _log_int(rng, 1, most)])
    else:
        n = 1 if kind == "decode" else rng.randint(2, 16)
        B = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, 400000 // B)
    lo = rng.choice([hi, hi // 2, hi // 8])
    return dict(c, B=B, new_lo=rng.choice([n, max(1, n // 2)]), new_hi=n, cached_lo=lo, cached_hi=hi)


def _spread(i, lo, hi):
    return lo + int((hi - lo + 1) * ((0.5 + i * 0.6180339887498949) % 1.0))


def _lengths(c):
    """(new tokens, all tokens) of every request; a padded one has a query and no key."""
    new = [_spread(i, c["new_lo"], c["new_hi"]) for i in range(c["B"])]
    total = [n + _spread(i + 7, c["cached_lo"], c["cached_hi"]) for i, n in enumerate(new)]
    return new + [1] * c["padded"], total + [0] * c["padded"]


# --------------------------------------------------------------------------------------- inputs
def _rows(gen, *shape):
    """Key or value rows: a few channels are larger than the rest, and tokens differ in size."""
    x = torch.randn(*shape, generator=gen, device=DEV)
    x *= torch.randn(shape[-1], generator=gen, device=DEV).mul_(0.5).exp_()
    x *= torch.randn(*shape[:-1], 1, generator=gen, device=DEV).mul_(0.3).exp_()
    return x.to(torch.bfloat16)


def _quantise(x, fmt):
    """(codes, scales) of rows, from the definition: the quotients in 64 bits, for those next to a border."""
    top = x.float().abs().amax(-1, keepdim=True)
    scale = top / LARGEST[fmt]
    q = torch.where(top > 0, x.double() * LARGEST[fmt] / top.double(), 0.0)
    codes = q.round().to(torch.int8) if fmt == "int8" else q.float().to(torch.float8_e4m3fn)
    return codes, scale.squeeze(-1)


def _cache(gen, c, slots):
    kv = []
    for _ in range(2):
        codes = torch.empty(c["nkv"], slots, c["hd"], dtype=DTYPE[c["fmt"]], device=DEV)
        scale = torch.empty(c["nkv"], slots, device=DEV)
        for h in range(c["nkv"]):
            codes[h], scale[h] = _quantise(_rows(gen, slots, c["hd"]), c["fmt"])
        kv.append((codes, scale))
    (k, ks), (v, vs) = kv
    c.update(k=k, v=v, ks=ks, vs=vs)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    c = dict(case)
    if c["op"] == "attend":
        new, total = _lengths(c)
        page, B = c["page"], len(new)
        pages = [-(-t // page) for t in total]
        spare = 5
        c["new_tokens"], c["total_tokens"] = new, total
        _cache(gen, c, (sum(pages) + spare) * page)
        order = list(range(sum(pages) + spare))
        random.Random(seed).shuffle(order)
        table = torch.zeros(B, max(1, max(pages)) * page, dtype=torch.int32)
        at = 0
        for b, n in enumerate(pages):
            first = torch.tensor(order[at : at + n], dtype=torch.int32) * page
            table[b, : n * page] = (first[:, None] + torch.arange(page, dtype=torch.int32)).flatten()
            at += n
        back = torch.randperm(B, generator=torch.Generator().manual_seed(seed))  # which row holds request b
        rows = torch.empty(B, dtype=torch.int64)
        rows[back] = torch.arange(B)
        c["row_of"] = rows.tolist()
        c["page_table"] = table[back].to(DEV)
        c["rows"] = rows.to(torch.int32).to(DEV)
        ends = torch.tensor([0] + new, dtype=torch.int32).cumsum(0)
        c["cu_q"] = ends.to(torch.int32).to(DEV)
        c["kv_lens"] = torch.tensor(total, dtype=torch.int32, device=DEV)
        q = torch.randn(sum(new), c["nq"], c["hd"], generator=gen, device=DEV) * 1.5
        c["q"] = q.to(torch.bfloat16)
        c["sink"] = torch.randn(c["nq"], generator=gen, device=DEV) + 1.0 if c["sinks"] else None
    else:
        T = c["T"]
        slots = -(-T // 64) * 64 + 192
        first = torch.randperm(slots // 64, generator=gen, device=DEV) * 64
        c["slots"] = (first[:, None] + torch.arange(64, device=DEV)).flatten()[:T].to(torch.int32)
        _cache(gen, c, slots)
        if c["op"] == "write":
            c["new_k"], c["new_v"] = _rows(gen, T, c["nkv"], c["hd"]), _rows(gen, T, c["nkv"], c["hd"])
    if own:
        from minisgl import ops

        c["cache"] = ops.KV8Cache(c["k"], c["v"], c["ks"], c["vs"])
    return c


# --------------------------------------------------------------------------------------- a pass
def _read_plain(c):
    at = c["slots"].long()
    return tuple((codes[:, at].float() * scale[:, at, None]).to(torch.bfloat16).transpose(0, 1).contiguous()
                 for codes, scale in ((c["k"], c["ks"]), (c["v"], c["vs"])))


def _write_plain(c):
    at = c["slots"].long()
    for x, codes, scale in ((c["new_k"], c["k"], c["ks"]), (c["new_v"], c["v"], c["vs"])):
        q, s = _quantise(x, c["fmt"])
        codes.view(torch.uint8)[:, at] = q.transpose(0, 1).view(torch.uint8)
        scale[:, at] = s.transpose(0, 1)
    return _read_plain(c)


def _attend_plain(c):
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    out = torch.zeros(c["q"].shape, dtype=torch.bfloat16, device=DEV)
    start = 0
    for b, (n, L) in enumerate(zip(c["new_tokens"], c["total_tokens"])):
        q = c["q"][start : start + n].float().view(n, nkv, nq // nkv, hd)
        o = out[start : start + n].view(n, nkv, nq // nkv, hd)
        start += n
        if L == 0:
            continue
        at = c["page_table"][c["row_of"][b], :L].long()
        far = torch.arange(L - n, L, device=DEV)[:, None] - torch.arange(L, device=DEV)[None]
        seen = far >= 0 if c["window"] < 0 else (far >= 0) & (far < c["window"])
        for h in range(nkv):
            k = c["k"][h, at].float() * c["ks"][h, at, None]
            v = c["v"][h, at].float() * c["vs"][h, at, None]
            s = (q[:, h].transpose(0, 1) @ k.t()) * hd**-0.5  # [heads of the group, n, L]
            s = torch.where(seen, s, -math.inf)
            top = s.amax(-1, keepdim=True)
            if c["sink"] is not None:
                sink = c["sink"].view(nkv, -1, 1, 1)[h]
                top = torch.maximum(top, sink)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            if c["sink"] is not None:
                total = total + torch.exp(sink - top)
            o[:, h] = ((p @ v) / total).transpose(0, 1).to(torch.bfloat16)
    return out


def run(state):
    c = state
    if own:
        from minisgl import ops

        if c["op"] == "attend":
            return ops.attention_kv8(c["q"], c["cache"], c["page_table"], c["rows"], c["cu_q"], c["kv_lens"],
                                     page_size=c["page"], max_q_len=c["new_hi"], window=c["window"], sinks=c["sink"])
        if c["op"] == "write":
            ops.store_kv8(c["new_k"], c["new_v"], c["cache"], c["slots"])
        return ops.load_kv8(c["cache"], c["slots"])
    return {"attend": _attend_plain, "write": _write_plain, "read": _read_plain}[c["op"]](c)


# ----------------------------------------------------------------------------------------- work
def _pairs(n, L, window):
    """Pairs of a query and a key that it sees, and the keys that any of them sees."""
    pairs = 0
    for pos in range(L - n, L):
        seen = max(0, pos + 1)
        pairs += seen if window < 0 else min(seen, window)
    return pairs, L if window < 0 else min(L, window + n - 1)


def work(case):
    c = case
    row = c["nkv"] * (c["hd"] + 4)  # one token's codes and scales, of keys or of values
    if c["op"] == "read":
        return {"bytes": c["T"] * (2 * row + 4 * c["nkv"] * c["hd"] + 4), "flops": 2.0 * c["T"] * c["nkv"] * c["hd"]}
    if c["op"] == "write":  # the new rows in, codes and scales out, and back into 16 bits
        return {"bytes": c["T"] * (4 * row + 8 * c["nkv"] * c["hd"] + 8), "flops": 8.0 * c["T"] * c["nkv"] * c["hd"]}
    new, total = _lengths(c)
    seen = [_pairs(n, L, c["window"]) for n, L in zip(new, total)]
    return {"bytes": 2 * row * sum(k for _, k in seen) + 4 * sum(new) * c["nq"] * c["hd"],
            "flops": 4.0 * c["hd"] * c["nq"] * sum(p for p, _ in seen)}


# ---------------------------------------------------------------------------------------- exact
def _exact_values(codes, scale):
    return codes.float().double() * scale.double().unsqueeze(-1)


def _exact_write(x, fmt):
    """What quantised rows stand for: the nearest of the type's values to each quotient."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    q = x * LARGEST[fmt] / torch.where(top > 0, top, 1.0)
    if fmt == "int8":
        near = torch.round(q)
    else:
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0**-6))) - 3)
        near = torch.round(q / step) * step
    return near * (top / LARGEST[fmt])


def _exact_attend(c):
    q = c["q"].double()
    group = c["nq"] // c["nkv"]
    out = torch.zeros_like(q)
    end = c["cu_q"].tolist()
    for b, L in enumerate(c["kv_lens"].tolist()):
        where = c["page_table"][int(c["rows"][b])][:L].long()
        if L == 0:
            continue
        pos = torch.arange(L, device=DEV)
        mine = torch.arange(L - (end[b + 1] - end[b]), L, device=DEV)
        hidden = pos[None, :] > mine[:, None]
        if c["window"] > 0:
            hidden |= pos[None, :] <= mine[:, None] - c["window"]
        for head in range(c["nq"]):
            kv = head // group
            keys = _exact_values(c["k"][kv][where], c["ks"][kv][where])
            logits = torch.einsum("nd,ld->nl", q[end[b] : end[b + 1], head], keys) / math.sqrt(c["hd"])
            logits.masked_fill_(hidden, -math.inf)
            norm = torch.logsumexp(logits, dim=-1, keepdim=True)
            if c["sink"] is not None:
                norm = torch.logaddexp(norm, c["sink"][head].double().expand_as(norm))
            weight = torch.exp(logits - norm)
            out[end[b] : end[b + 1], head] = torch.einsum("nl,ld->nd", weight, _exact_values(c["v"][kv][where], c["vs"][kv][where]))
    return out


def exact(case, seed):
    c = prepare(case, seed)
    if c["op"] == "attend":
        return _exact_attend(c)
    if c["op"] == "write":
        return _exact_write(c["new_k"], c["fmt"]), _exact_write(c["new_v"], c["fmt"])
    at = c["slots"].long()
    return tuple(_exact_values(t[:, at], s[:, at]).transpose(0, 1) for t, s in ((c["k"], c["ks"]), (c["v"], c["vs"])))
