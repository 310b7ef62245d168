"""Measured cases of the expert router, the 4-bit linear product and the 4-bit experts.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes a case's
inputs on the GPU from a seed, and ``run()`` is one pass: the framework's operators where ``own`` is
true, elementary torch operations otherwise. ``exact()`` is the same result in 64 bits, written
apart from both, and ``work()`` the bytes and operations that a pass cannot do without.

4-bit weights are in the form in which checkpoints hold them: two codes 0..15 per byte along the
input dimension (low nibble first), one 16-bit scale per row and group of inputs, and either a zero
point per row and group or none, which means 8. The weight is (code - zero point) * scale.
"""

import math

import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the router of one decoded token: softmax over 128 experts, top 8, weights renormalised
        dict(name="route 1x128 softmax", op="route", T=1, E=128, k=8, score="softmax", bias=False, groups=1, kept=1,
             group_score="max", renorm=True, scale=1.0, dtype="float32"),
        # a decode batch with sigmoid scores, a balancing bias and groups of experts
        dict(name="route 64x256 sigmoid groups", op="route", T=64, E=256, k=8, score="sigmoid", bias=True, groups=8, kept=4,
             group_score="top2", renorm=True, scale=2.5, dtype="float32"),
        # a long prefill with the same router: here the logits' bytes count
        dict(name="route 16384x256 sigmoid groups", op="route", T=16384, E=256, k=8, score="sigmoid", bias=True, groups=8,
             kept=4, group_score="top2", renorm=True, scale=2.5, dtype="float32"),
        # odd sizes, 16-bit logits with many ties, groups ranked by their best expert, no renormalising
        dict(name="route 4099x96 softmax groups", op="route", T=4099, E=96, k=6, score="softmax", bias=False, groups=3, kept=2,
             group_score="max", renorm=False, scale=16.0, dtype="bfloat16"),
        # one decoded token through an attention output projection: latency
        dict(name="linear 1x5120x5120", op="linear", M=1, N=5120, K=5120, group=128, zeros=False, bias=False, scales="bfloat16"),
        # one decoded token through the widest projection of an MLP (gate and up): weight bytes
        dict(name="linear 1x34816x5120", op="linear", M=1, N=34816, K=5120, group=128, zeros=False, bias=False,
             scales="bfloat16"),
        # a small decode batch through the down projection, zero points, groups of 64
        dict(name="linear 16x5120x17408 zeros", op="linear", M=16, N=5120, K=17408, group=64, zeros=True, bias=False,
             scales="float16"),
        # odd row count (an uneven share of a vocabulary), short groups, a bias
        dict(name="linear 5x1001x2880", op="linear", M=5, N=1001, K=2880, group=32, zeros=False, bias=True, scales="bfloat16"),
        # a large decode batch or a short prompt: the products' operations count
        dict(name="linear 200x34816x5120", op="linear", M=200, N=34816, K=5120, group=128, zeros=False, bias=False,
             scales="bfloat16"),
        # one decoded token through its experts
        dict(name="experts 1 of 128", op="experts", T=1, E=128, k=8, H=2048, I=768, group=128, zeros=False,
             scales="bfloat16"),
        # a decode batch over wide experts of odd blocks, short groups and zero points
        dict(name="experts 32 of 32 wide", op="experts", T=32, E=32, k=4, H=2880, I=2880, group=32, zeros=True,
             scales="bfloat16"),
        # a prompt's chunk: every expert gets some tens of tokens
        dict(name="experts 512 of 128", op="experts", T=512, E=128, k=8, H=2048, I=768, group=128, zeros=False,
             scales="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "linear", "experts"])
    scales = rng.choice(["bfloat16", "float16"])
    if op == "route":
        T = _log_int(rng, 1, 16384)
        groups = rng.choice([1, 1, 2, 4, 8])
        per = rng.randint(max(3, 8 // groups), 256 // groups)
        kept = 1 if groups == 1 else rng.randint(1, groups)
        return dict(op=op, T=T, E=groups * per, k=rng.randint(1, min(10, kept * per)), score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, groups=groups, kept=kept, group_score=rng.choice(["max", "top2"]),
                    renorm=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["float32", "bfloat16"]))
    group = rng.choice([32, 64, 128])
    if op == "linear":
        M, N = _log_int(rng, 1, 200), _log_int(rng, 96, 34816)
        K = group * max(1, _log_int(rng, 256, 5120 * 34816 // max(N, 10240)) // group)
        return dict(op=op, M=M, N=N, K=K, group=group, zeros=rng.random() < 0.4, bias=rng.random() < 0.4, scales=scales)
    E = _log_int(rng, 4, 128)
    T = _log_int(rng, 1, 512)
    most = 128 * 2048 * 768
    H = group * max(1, _log_int(rng, 256, 2880) // group)
    inter = min(2880, most // (E * H), 512 * 8 * 2048 * 768 // (T * 8 * H))
    inter = group * max(1, _log_int(rng, 128, max(128, inter)) // group)
    return dict(op=op, T=T, E=E, k=rng.randint(1, min(8, E)), H=H, I=inter, group=group, zeros=rng.random() < 0.4, scales=scales)


# --------------------------------------------------------------------------------------- inputs
def _dtype(name):
    return getattr(torch, name)


def _four_bit(gen, shape, group, zeros, scales):
    """Codes, scales and zero points as quantising a normally distributed weight gives them."""
    n, k = shape[-2:]
    codes = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(0.0, 2.7, generator=gen)
    codes = codes.add_(8).round_().clamp_(0, 15).to(torch.uint8)
    q = codes[..., 0::2] | (codes[..., 1::2] << 4)
    side = tuple(shape[:-1]) + (k // group,)
    s = torch.rand(side, generator=gen, device=DEV).mul_(0.006).add_(0.004) * (4.0 / math.sqrt(k / 128))
    z = torch.randint(5, 11, side, generator=gen, device=DEV, dtype=torch.uint8) if zeros else None
    return dict(q=q.contiguous(), s=s.to(_dtype(scales)), z=z, group=group)


def _activations(gen, rows, cols):
    """Hidden states: a few channels are much larger than the rest."""
    ch = torch.randn(cols, generator=gen, device=DEV).mul_(0.5).exp_()
    return (torch.randn(rows, cols, generator=gen, device=DEV) * ch).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    c = dict(case)
    if c["op"] == "route":
        logits = torch.randn(c["T"], c["E"], generator=gen, device=DEV) * 1.5 - 0.5
        c["logits"] = logits.to(_dtype(c["dtype"]))
        c["b"] = torch.randn(c["E"], generator=gen, device=DEV) * 0.1 if c["bias"] else None
        return c
    if c["op"] == "linear":
        c["x"] = _activations(gen, c["M"], c["K"])
        c["w"] = _four_bit(gen, (c["N"], c["K"]), c["group"], c["zeros"], c["scales"])
        c["b"] = torch.randn(c["N"], generator=gen, device=DEV).to(torch.bfloat16) if c["bias"] else None
        if own:
            from minisgl import ops

            c["weight"] = ops.W4Weight.pack(c["w"]["q"], c["w"]["s"], c["w"]["z"])
        return c
    T, E, H, inter, k = c["T"], c["E"], c["H"], c["I"], c["k"]
    c["x"] = _activations(gen, T, H)
    c["w1"] = _four_bit(gen, (E, 2 * inter, H), c["group"], c["zeros"], c["scales"])
    c["w2"] = _four_bit(gen, (E, H, inter), c["group"], c["zeros"], c["scales"])
    # some experts are chosen more often than others
    p = torch.randn(T, E, generator=gen, device=DEV) + 0.5 * torch.randn(E, generator=gen, device=DEV)
    top, ids = torch.topk(p, k, dim=-1)
    c["weights"], c["ids"] = torch.softmax(top, dim=-1), ids.to(torch.int32)
    if own:
        from minisgl import ops

        c["weight1"] = ops.W4Weight.pack(c["w1"]["q"], c["w1"]["s"], c["w1"]["z"], gated=True)
        c["weight2"] = ops.W4Weight.pack(c["w2"]["q"], c["w2"]["s"], c["w2"]["z"])
    return c


# --------------------------------------------------------------------------------------- a pass
def _route_plain(c):
    """Scores in 64 bits: the order of two experts can hang on their last digits."""
    x = c["logits"].double()
    if c["score"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        scores = e / e.sum(-1, keepdim=True)
    else:
        scores = 1.0 / (1.0 + torch.exp(-x))
    choice = scores if c["b"] is None else scores + c["b"].double()
    T, E = x.shape
    if c["groups"] > 1:
        per = choice.view(T, c["groups"], E // c["groups"])
        rank = per.amax(-1) if c["group_score"] == "max" else per.topk(2, dim=-1).values.sum(-1)
        order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, : c["kept"]]
        keep = torch.zeros(T, c["groups"], dtype=torch.bool, device=x.device).scatter_(1, order, True)
        choice = torch.where(keep.repeat_interleave(E // c["groups"], dim=1), choice, -math.inf)
    ids = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, : c["k"]]
    w = scores.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return (w * c["scale"]).float(), ids.to(torch.int32)


def _dequant(w):
    """The weights that the codes stand for, in 32 bits."""
    codes = torch.stack([w["q"] & 15, w["q"] >> 4], dim=-1).flatten(-2).float()
    codes = codes.unflatten(-1, (-1, w["group"]))
    zero = 8.0 if w["z"] is None else w["z"].float().unsqueeze(-1)
    return ((codes - zero) * w["s"].float().unsqueeze(-1)).flatten(-2)


def _linear_plain(c):
    y = c["x"].float() @ _dequant(c["w"]).t()
    if c["b"] is not None:
        y = y + c["b"].float()
    return y.to(torch.bfloat16)


def _experts_plain(c):
    """Every expert on every token, weighted by the share that the router gave it."""
    h = torch.matmul(c["x"].float(), _dequant(c["w1"]).transpose(1, 2))  # [E, T, 2I]
    gate, up = h.chunk(2, dim=-1)
    a = gate / (1.0 + torch.exp(-gate)) * up
    z = torch.matmul(a, _dequant(c["w2"]).transpose(1, 2))  # [E, T, H]
    share = torch.zeros(c["T"], c["E"], device=z.device).scatter_add_(1, c["ids"].long(), c["weights"])
    return (z * share.t().unsqueeze(-1)).sum(0).to(torch.bfloat16)


def run(state):
    c = state
    if own:
        from minisgl import ops

        if c["op"] == "route":
            return ops.route_experts(c["logits"], c["k"], scoring=c["score"], bias=c["b"], num_groups=c["groups"],
                                     top_groups=c["kept"], group_score=c["group_score"], renormalize=c["renorm"],
                                     scale=c["scale"])
        if c["op"] == "linear":
            return ops.linear_w4(c["x"], c["weight"], c["b"])
        return ops.experts_w4(c["x"], c["weight1"], c["weight2"], c["weights"], c["ids"])
    return {"route": _route_plain, "linear": _linear_plain, "experts": _experts_plain}[c["op"]](c)


# ----------------------------------------------------------------------------------------- work
def _weight_bytes(n, k, group, zeros):
    return n * k / 2 + n * (k // group) * (3 if zeros else 2)


def work(case):
    c = case
    if c["op"] == "route":
        size = 4 if c["dtype"] == "float32" else 2
        return {"bytes": c["T"] * c["E"] * size + (4 * c["E"] if c["bias"] else 0) + c["T"] * c["k"] * 8,
                "flops": 8.0 * c["T"] * c["E"]}
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": _weight_bytes(N, K, c["group"], c["zeros"]) + 2 * M * (K + N) + (2 * N if c["bias"] else 0),
                "flops": 2.0 * M * N * K}
    T, E, H, inter, k = c["T"], c["E"], c["H"], c["I"], c["k"]
    hit = E * (1.0 - (1.0 - k / E) ** T)  # experts that at least one token goes to, if all are alike
    per = _weight_bytes(2 * inter, H, c["group"], c["zeros"]) + _weight_bytes(H, inter, c["group"], c["zeros"])
    return {"bytes": hit * per + 4 * T * H + 8 * T * k, "flops": 6.0 * T * k * H * inter}


# ---------------------------------------------------------------------------------------- exact
def _exact_route(c):
    import numpy as np

    x = c["logits"].double().cpu().numpy()
    T, E = x.shape
    if c["score"] == "softmax":
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = 1.0 / (1.0 + np.exp(-x))
    v = p.copy() if c["b"] is None else p + c["b"].double().cpu().numpy()[None]
    if c["groups"] > 1:
        size = E // c["groups"]
        tops = -np.sort(-v.reshape(T, c["groups"], size), axis=2)
        rank = tops[:, :, 0] if c["group_score"] == "max" else tops[:, :, 0] + tops[:, :, 1]
        place = np.argsort(np.argsort(-rank, axis=1, kind="stable"), axis=1, kind="stable")
        v[np.repeat(place >= c["kept"], size, axis=1)] = -np.inf
    ids = np.argsort(-v, axis=1, kind="stable")[:, : c["k"]]
    w = np.take_along_axis(p, ids, 1)
    if c["renorm"]:
        w = w / w.sum(1, keepdims=True)
    return torch.from_numpy(w * c["scale"]), torch.from_numpy(ids.astype(np.int32))


def _exact_weight(w, e=None):
    """One matrix in 64 bits, from its bytes: the even inputs' codes, then the odd ones'."""
    q, s, z = (t if t is None or e is None else t[e] for t in (w["q"], w["s"], w["z"]))
    out = torch.empty(q.shape[0], 2 * q.shape[1], dtype=torch.float64, device=q.device)
    out[:, 0::2] = (q % 16).double()
    out[:, 1::2] = (q // 16).double()
    every = torch.arange(out.shape[1], device=q.device) // w["group"]
    out -= 8.0 if z is None else z.double()[:, every]
    return out.mul_(s.double()[:, every])


def exact(case, seed):
    c = prepare(case, seed)
    if c["op"] == "route":
        return _exact_route(c)
    x = c["x"].double()
    if c["op"] == "linear":
        y = torch.einsum("nk,mk->mn", _exact_weight(c["w"]), x)
        return y if c["b"] is None else y.add_(c["b"].double())
    out = torch.zeros(c["T"], c["H"], dtype=torch.float64, device=DEV)
    for e in range(c["E"]):
        tok, slot = torch.nonzero(c["ids"] == e, as_tuple=True)
        if len(tok) == 0:
            continue
        h = torch.einsum("nk,mk->mn", _exact_weight(c["w1"], e), x[tok])
        g, u = h[:, : c["I"]], h[:, c["I"]:]
        a = g * torch.sigmoid(g) * u
        out.index_add_(0, tok, torch.einsum("nk,mk->mn", _exact_weight(c["w2"], e), a) * c["weights"][tok, slot, None].double())
    return out
