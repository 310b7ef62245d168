"""Routed-expert forward on the GPU (graph-capturable, no host synchronization):

route (softmax top-k) -> align (counting sort into per-expert segments padded to ``bn`` rows,
device work list) -> gather permuted activations -> grouped tcgen05 GEMM (gate|up, activation in
its epilogue when the weights are gate/up interleaved) -> grouped GEMM (down) -> weighted top-k
combine. Expert weights are bf16 ``[E, N, K]`` tensors or MXFP4 ``Mxfp4Experts`` (fp4 in HBM,
converted to bf16 tile by tile inside the grouped GEMM).

Behaviour matches ``moe/grouped.py:moe_reference`` (and the reference's fused MoE,
python/minisgl/moe/fused.py:127-227).
"""

from __future__ import annotations

import torch

from minisgl._native import cuda as _cuda

from . import reference as ref

_ACT = {"silu": 0, "gelu": 1, "swiglu_oai": 2}
_GATED_EPI = {"silu": 1, "gelu": 2, "swiglu_oai": 4}  # grouped-GEMM epilogue applying the activation


def interleave_experts(w1: torch.Tensor, w2: torch.Tensor, b1: torch.Tensor | None = None):
    """Expert weights for the gated grouped GEMM: ``w1 [E, 2I, H]`` as [gate; up] halves -> gate / up
    rows interleaved in blocks of GATE_UP_BLOCK (one 256-row weight tile then holds 128 gate rows and
    their 128 up rows, and the epilogue applies the activation). I is padded up to a whole block with
    zero rows (and ``w2 [E, H, I]`` with zero columns, ``b1`` with zeros): act(0, 0) * ... = 0 for
    SiLU, GELU and the clamped SwiGLU alike, so padding contributes nothing. Returns (w1, w2, b1)."""
    from .reference import GATE_UP_BLOCK

    E, two_i, H = w1.shape
    inter = two_i // 2
    ip = -(-inter // GATE_UP_BLOCK) * GATE_UP_BLOCK
    nb = ip // GATE_UP_BLOCK
    w1n = torch.zeros(E, 2 * ip, H, dtype=w1.dtype, device=w1.device)
    v = w1n.view(E, nb, 2, GATE_UP_BLOCK, H)  # [expert, block, gate/up, row, H]
    for half in range(2):
        src = torch.zeros(E, ip, H, dtype=w1.dtype, device=w1.device) if ip != inter else None
        part = w1[:, half * inter : (half + 1) * inter]
        if src is not None:
            src[:, :inter] = part
            part = src
        v[:, :, half] = part.reshape(E, nb, GATE_UP_BLOCK, H)
    w2n = w2
    if ip != inter:
        w2n = torch.zeros(E, w2.shape[1], ip, dtype=w2.dtype, device=w2.device)
        w2n[:, :, :inter] = w2
    b1n = None
    if b1 is not None:
        b1n = torch.zeros(E, 2 * ip, dtype=b1.dtype, device=b1.device)
        vb = b1n.view(E, nb, 2, GATE_UP_BLOCK)
        for half in range(2):
            part = torch.zeros(E, ip, dtype=b1.dtype, device=b1.device)
            part[:, :inter] = b1[:, half * inter : (half + 1) * inter]
            vb[:, :, half] = part.view(E, nb, GATE_UP_BLOCK)
    return w1n, w2n, b1n


def route_experts(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", bias: torch.Tensor | None = None,
                  num_groups: int = 1, top_groups: int = 1, group_score: str = "max", renormalize: bool = True,
                  scale: float = 1.0):
    """Experts of every token: (weights fp32 ``[T, top_k]``, ids int32 ``[T, top_k]``, best first).

    ``logits`` (fp32 or bf16 ``[T, E]``, E <= 512, may be strided) become scores by ``scoring``,
    ``softmax`` or ``sigmoid``. Up to 32 experts are chosen by score + ``bias`` (fp32 ``[E]``, a balancing bias
    that moves the choice but not the weights), without a bias by their logit; equal ones go to the
    lowest id, and the order is that of 64-bit arithmetic. With ``num_groups`` > 1 (at most 256) the experts form that
    many groups of consecutive ids, and only those of the ``top_groups`` best are chosen from: a
    group counts by its best expert (``group_score="max"``) or by the sum of the two best scores
    (plus bias) in it (``"top2"``). The weights are the chosen scores, divided by their sum with
    ``renormalize``, times ``scale``, in fp32 (on the GPU off by at most 2^-18 of
    the value, for scores down to e^-32 of the largest).

    A NaN logit counts as -inf and +inf as the largest fp32 value; a row without a finite logit has
    softmax scores of zero, and weights whose sum is zero stay zero. NaN biases count as the lowest fp32
    value, infinite ones as the largest or lowest."""
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"scoring must be softmax or sigmoid, got {scoring!r}")
    if group_score not in ("max", "top2"):
        raise ValueError(f"group_score must be max or top2, got {group_score!r}")
    if not logits.is_cuda:  # (the kernel's binding checks the same)
        if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"logits must be fp32 or bf16 [tokens, experts], got {logits.dtype} {tuple(logits.shape)}")
        T, E = logits.shape
        if not 1 <= E <= 512 or T >= 2**31:
            raise ValueError(f"route_experts: 1 to 512 experts and less than 2^31 tokens, got {tuple(logits.shape)}")
        if bias is not None:
            if bias.dtype != torch.float32 or bias.numel() != E or bias.is_cuda or not bias.is_contiguous():
                raise ValueError(f"bias must be contiguous fp32 [{E}] on the logits' device, got {bias.dtype} "
                                 f"{tuple(bias.shape)} on {bias.device}")
            bias = bias.view(E)
        if not 1 <= num_groups <= 256 or E % num_groups:
            raise ValueError(f"{E} experts do not split into {num_groups} groups (at most 256)")
        if not 1 <= top_groups <= num_groups or not 1 <= top_k <= min(32, top_groups * (E // num_groups)):
            raise ValueError(f"cannot choose {top_k} of {E} experts in {top_groups} of {num_groups} groups (at most 32)")
        if group_score == "top2" and num_groups > 1 and E // num_groups < 2:
            raise ValueError("group_score 'top2' needs two experts per group")
        return ref.route_experts(logits, top_k, scoring, bias, num_groups, top_groups, group_score, renormalize, scale)
    return _cuda().route_experts(logits, top_k, scoring == "sigmoid", bias, num_groups, top_groups,
                                 group_score == "top2", renormalize, scale)


def pick_bn(pairs: int, experts: int) -> int:
    avg = pairs / max(experts, 1)
    for bn in (16, 32, 64):
        if avg <= bn:
            return bn
    return 128


def _grouped(out, xs, w, bias, count, work, bn, epi):
    """Grouped GEMM over bf16 experts ``[E, N, K]`` or MXFP4 experts kept in fp4 (``Mxfp4Experts``)."""
    from minisgl.moe.mxfp4 import Mxfp4Experts

    if isinstance(w, Mxfp4Experts):
        _cuda().gemm_grouped_fp4(out, xs, w.q, w.s, w.n, bias, count, work, bn, epi)
    else:
        _cuda().gemm_grouped(out, xs, w, bias, count, work, bn, epi)


def moe_forward(x, w1, w2, gating, topk, renormalize, activation, w1_bias=None, w2_bias=None,
                softmax_after_topk=False, expert_offset: int = 0, w1_interleaved: bool = False):
    """``w1``/``w2`` hold experts [expert_offset, expert_offset + E) of the ``gating`` columns
    (expert parallelism); assignments to other experts contribute nothing here. With
    ``w1_interleaved`` (``interleave_experts`` layout) the first grouped GEMM's epilogue applies the
    activation; otherwise a separate kernel does."""
    c = _cuda()
    T, H = x.shape
    E, two_i, _ = w1.shape
    inter = two_i // 2
    dev = x.device
    logits = gating if gating.dtype == torch.float32 else gating.float()
    weights = torch.empty(T, topk, dtype=torch.float32, device=dev)
    ids = torch.empty(T, topk, dtype=torch.int32, device=dev)
    c.moe_route(logits.contiguous(), topk, bool(renormalize), bool(softmax_after_topk), weights, ids)
    pairs = T * topk
    bn = pick_bn(pairs, E)
    max_tiles = (pairs + bn - 1) // bn + E
    rows = max_tiles * bn
    perm = torch.empty(rows, dtype=torch.int32, device=dev)
    inv = torch.empty(pairs, dtype=torch.int32, device=dev)
    work = torch.empty(max_tiles, 2, dtype=torch.int32, device=dev)
    count = torch.empty(1, dtype=torch.int32, device=dev)
    c.moe_align(ids, E, bn, perm, inv, work, count, expert_offset)
    xs = torch.empty(rows, H, dtype=x.dtype, device=dev)
    c.moe_gather(xs, x.contiguous(), perm, topk)
    a = torch.empty(rows, inter, dtype=x.dtype, device=dev)
    if w1_interleaved:
        _grouped(a, xs, w1, w1_bias, count, work, bn, _GATED_EPI[activation])
    else:
        y1 = torch.empty(rows, two_i, dtype=x.dtype, device=dev)
        _grouped(y1, xs, w1, w1_bias, count, work, bn, 0)
        c.moe_act(a, y1, _ACT[activation], perm)
    y2 = torch.empty(rows, H, dtype=x.dtype, device=dev)
    _grouped(y2, a, w2, w2_bias, count, work, bn, 0)
    out = torch.empty(T, H, dtype=x.dtype, device=dev)
    c.moe_combine(out, y2, weights, inv, topk)
    return out
