"""4-bit weights with group scales: a linear product and the routed experts of an MoE layer.

``W4Weight`` holds one weight matrix ``[N, K]``, or the matrices ``[E, N, K]`` of a layer's experts,
whose values are ``(code - zero) * scale``: a code 0..15 per value, and per row and group of 32, 64 or
128 inputs one bf16 or fp16 scale and optionally a zero point 0..15 (without them every zero point is
8). ``W4Weight.pack`` takes two codes a byte along the inputs, as many checkpoints hold them (other orders
are the caller's to turn into this one), and lays them out once in the order in which the kernels read
them (``csrc/kernels/w4.cuh``); ``quantize_w4`` makes them from bf16 weights.

    w = ops.W4Weight.pack(q, scales, zeros)               # q [N, K/2] uint8, scales / zeros [N, K/group]
    y = ops.linear_w4(x, w, bias)                         # [M, K] bf16 -> [M, N] bf16

    w1 = ops.W4Weight.pack(q1, s1, gated=True)            # [E, 2I, H]: gate rows, then up rows
    w2 = ops.W4Weight.pack(q2, s2)                        # [E, H, I]
    weights, ids = ops.route_experts(router_logits, top_k)
    y = ops.experts_w4(x, w1, w2, weights, ids)

CUDA tensors run the sm_100a kernels, CPU tensors the plain form in ``ops.reference``. Calls may be
captured in CUDA graphs; they keep no state of their own, so calls on several streams are independent.

What is rounded on the GPU: the linear product holds weights exactly for up to 16 tokens (their scale
multiplies the fp32 sum of its group); for more tokens, and for rows too wide for that form's shared
memory, every weight is rounded once to bf16, as in a bf16 copy of the weights. A token's result so moves
a little, within what one rounding of the weights does, when a batch passes from the one to the other.
The experts' products hold weights exactly for any number of tokens (for many tokens and fp16 scales: to
2^-12), the activated values between them in 16 bits for few tokens (up to 12 pairs of a token and an
expert per expert) and in bf16 for more. Equal calls give equal results.
"""

from __future__ import annotations

import math
from dataclasses import dataclass, replace

import torch
import torch.nn.functional as F

from minisgl._native import cuda as _cuda

from . import reference as ref

GROUP_SIZES = (32, 64, 128)
_ACT = {"silu": 0, "gelu": 1, "swiglu_oai": 2}


@dataclass
class W4Weight:
    data: torch.Tensor         # uint8 [E, Nt, KC, bytes]: records of 32 rows x 128 inputs
    n: int                     # rows
    k: int                     # inputs
    group: int                 # inputs per scale
    zeros: bool                # zero points are stored (else 8)
    scale_dtype: torch.dtype   # bf16 / fp16
    gated: bool                # tiles of 16 gate rows and the up rows of the same outputs
    experts: bool              # [E, N, K] rather than one [N, K]

    @property
    def shape(self):
        return (self.data.shape[0], self.n, self.k) if self.experts else (self.n, self.k)

    @property
    def is_cuda(self) -> bool:
        return self.data.is_cuda

    @property
    def device(self) -> torch.device:
        return self.data.device

    def nbytes(self) -> int:
        return self.data.numel()

    def to(self, device) -> "W4Weight":
        return replace(self, data=self.data.to(device))

    @classmethod
    def pack(cls, q: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
             gated: bool = False) -> "W4Weight":
        """``q`` uint8 ``[(E,) N, K/2]``, two codes a byte along the inputs, the low nibble first;
        ``scales`` bf16 / fp16, finite, and ``zeros`` uint8 (0..15) ``[(E,) N, K/group]``. ``gated``: the rows
        are ``[gate; up]`` halves, as in the first matrix of a gated MLP."""
        if q.dtype != torch.uint8 or q.dim() not in (2, 3):
            raise ValueError(f"4-bit codes must be uint8 [N, K/2] or [E, N, K/2], got {q.dtype} {tuple(q.shape)}")
        experts = q.dim() == 3
        if scales.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"4-bit scales must be bf16 or fp16, got {scales.dtype}")
        if scales.dim() != q.dim() or scales.shape[:-1] != q.shape[:-1] or scales.shape[-1] == 0 or q.numel() == 0:
            raise ValueError(f"4-bit codes {tuple(q.shape)} / scales {tuple(scales.shape)} mismatch")
        k = 2 * q.shape[-1]
        group = k // scales.shape[-1]
        if group not in GROUP_SIZES or group * scales.shape[-1] != k:
            raise ValueError(f"{k} inputs over {scales.shape[-1]} scales a row: groups must be 32, 64 or 128 inputs")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
            raise ValueError(f"4-bit zero points must be uint8 {tuple(scales.shape)}, got {zeros.dtype} {tuple(zeros.shape)}")
        n = q.shape[-2]
        if gated and n % 2:
            raise ValueError(f"a gated weight has as many gate as up rows, got {n} rows")
        if zeros is not None and zeros.numel() and int(zeros.max()) > 15:
            raise ValueError("4-bit zero points must be 0..15")
        if any(t is not None and t.device != q.device for t in (scales, zeros)):
            raise ValueError("4-bit codes, scales and zero points must be on one device")
        if not bool(scales.isfinite().all()):
            raise ValueError("4-bit scales must be finite")
        if not experts:
            q, scales, zeros = q[None], scales[None], None if zeros is None else zeros[None]
        E = q.shape[0]
        nt = -(-(n // 2) // 16) if gated else -(-n // 32)
        kc = -(-k // 128)
        per = 128 // group  # groups of a record

        def tiles(t: torch.Tensor, cols: int) -> torch.Tensor:
            """[E, N, c] -> [E, Nt, half, 2, 8, KC, cols]: rows g and g + 8 of every half, zeros beyond the end"""
            t = F.pad(t, (0, kc * cols - t.shape[-1]))
            if gated:
                t = F.pad(t.unflatten(1, (2, n // 2)), (0, 0, 0, nt * 16 - n // 2))
                t = t.unflatten(2, (nt, 2, 8)).permute(0, 2, 3, 1, 4, 5)
            else:
                t = F.pad(t, (0, 0, 0, nt * 32 - n)).unflatten(1, (nt, 2, 2, 8))
            return t.unflatten(-1, (kc, cols))

        data = torch.empty(E, nt, kc, 2048 + per * (64 if zeros is None else 96), dtype=torch.uint8, device=q.device)
        # bytes of a row by (block, word, lane column t, byte i): codes 2i (low) and 2i + 1
        b = tiles(q, 64).unflatten(-1, (2, 4, 4, 2))
        lo, hi = b[:, :, :, 0], b[:, :, :, 1]  # rows g, rows g + 8: [E, Nt, half, 8, KC, block, word, t, i]
        perm = (0, 1, 4, 2, 5, 3, 7, 6, 8)  # -> [E, Nt, KC, half, block, g, t, word, i]
        out = data[..., :2048].unflatten(-1, (2, 2, 8, 4, 4, 2, 2))
        out[..., 0, :] = ((lo & 15) | (hi << 4)).permute(perm)
        out[..., 1, :] = ((lo >> 4) | (hi & 0xF0)).permute(perm)
        side = lambda t: tiles(t, per).permute(0, 1, 5, 6, 4, 2, 3).reshape(E, nt, kc, per * 32)  # noqa: E731
        data[..., 2048 : 2048 + per * 64] = side(scales.view(torch.int16)).view(torch.uint8)
        if zeros is not None:
            data[..., 2048 + per * 64 :] = side(zeros)
        return cls(data, n, k, group, zeros is not None, scales.dtype, gated, experts)

    def codes(self):
        """(q, scales, zeros) as ``pack`` took them."""
        E, nt, kc, _ = self.data.shape
        per = 128 // self.group

        def rows(t: torch.Tensor, cols: int) -> torch.Tensor:
            """[E, Nt, half, 2, 8, ...] -> [E, N, cols]"""
            t = t.flatten(5)[..., :cols]
            if self.gated:
                return t.permute(0, 3, 1, 2, 4, 5).flatten(2, 4)[:, :, : self.n // 2].flatten(1, 2).contiguous()
            return t.flatten(1, 4)[:, : self.n].contiguous()

        c = self.data[..., :2048].unflatten(-1, (2, 2, 8, 4, 4, 2, 2))  # [E, Nt, KC, half, block, g, t, word, c, i]
        c = c.permute(0, 1, 3, 5, 2, 4, 7, 6, 8, 9)  # [E, Nt, half, g, KC, block, word, t, c, i]
        even, odd = c[..., 0, :], c[..., 1, :]
        q = torch.stack([(even & 15) | ((odd & 15) << 4), (even >> 4) | (odd & 0xF0)], dim=3)
        side = lambda t: rows(t.view(E, nt, kc, per, 8, 2, 2).permute(0, 1, 5, 6, 4, 2, 3), self.k // self.group)  # noqa: E731
        s = side(self.data[..., 2048 : 2048 + per * 64].contiguous().view(torch.int16)).view(self.scale_dtype)
        z = side(self.data[..., 2048 + per * 64 :].contiguous()) if self.zeros else None
        got = (rows(q, self.k // 2), s, z)
        return got if self.experts else tuple(t if t is None else t[0] for t in got)

    def dequant(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The ``[(E,) N, K]`` weights that the codes stand for."""
        q, s, z = self.codes()
        v = torch.stack([q & 15, q >> 4], dim=-1).flatten(-2).float().unflatten(-1, (-1, self.group))
        zero = 8.0 if z is None else z.float().unsqueeze(-1)
        return ((v - zero) * s.float().unsqueeze(-1)).flatten(-2).to(dtype)


def quantize_w4(w: torch.Tensor, group: int = 128, symmetric: bool = True, scale_dtype: torch.dtype = torch.bfloat16):
    """Rounds ``w [(E,) N, K]`` to 4 bits, per group of ``group`` inputs: (q, scales, zeros) for
    ``W4Weight.pack``. Symmetric: the largest magnitude becomes 7 steps around a zero point of 8
    (``zeros`` is None); otherwise the group's range, widened to hold 0, is cut into 15 steps. Weights
    that are not finite, or whose scale is beyond ``scale_dtype``, are refused."""
    if scale_dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"4-bit scales must be bf16 or fp16, got {scale_dtype}")
    if group not in GROUP_SIZES or w.shape[-1] % group:
        raise ValueError(f"{w.shape[-1]} inputs do not split into groups of {group} (32, 64 or 128)")
    v = w.float().unflatten(-1, (-1, group))
    if symmetric:
        s = (v.abs().amax(-1) / 7).to(scale_dtype)
        z = None
        zero = 8.0
    else:
        lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).to(scale_dtype)
        step = s.float()
        z = torch.where(step > 0, torch.round(-lo / step), torch.zeros_like(lo)).clamp(0, 15)
        zero = z.unsqueeze(-1)
        z = z.to(torch.uint8)
    if not bool(s.isfinite().all()):
        raise ValueError(f"weights of up to {float(v.abs().max()):.4g} have no finite scale in {scale_dtype}")
    step = s.float().unsqueeze(-1)
    code = torch.where(step > 0, torch.round(v / step), torch.zeros_like(v)) + zero
    code = code.clamp(0, 15).to(torch.uint8).flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), s, z


def _args(w: W4Weight):
    return w.data, w.n, w.k, w.group, w.zeros, w.scale_dtype == torch.float16


# What the kernels' bindings check, for tensors that do not go there.
def _check_rows(op: str, x: torch.Tensor, *weights: W4Weight):
    k = weights[0].k
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != k:
        raise ValueError(f"{op}: x must be bf16 [tokens, {k}], got {x.dtype} {tuple(x.shape)}")
    if any(w.is_cuda for w in weights):
        raise ValueError(f"{op}: weights must be on the activations' device")


def _bias(name: str, b: torch.Tensor | None, shape):
    if b is None:
        return None
    if b.dtype != torch.bfloat16 or b.numel() != math.prod(shape) or b.is_cuda or not b.is_contiguous():
        raise ValueError(f"{name} must be contiguous bf16 {list(shape)} on the activations' device, got {b.dtype} "
                         f"{tuple(b.shape)} on {b.device}")
    return b.view(shape)


def linear_w4(x: torch.Tensor, w: W4Weight, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ w^T (+ bias)`` for bf16 ``x [M, K]`` and a 4-bit ``w [N, K]``; bf16 ``[M, N]``. Sums are
    held in fp32; above 16 tokens every weight ``(code - zero) * scale`` is rounded to bf16 first. ``x`` may
    be strided (rows that overlap or are off the 16-byte grid are copied), ``bias`` is bf16 ``[N]``."""
    if w.experts or w.gated:
        raise ValueError("linear_w4 takes one ungated matrix")
    if not x.is_cuda:
        _check_rows("linear_w4", x, w)
        if x.shape[0] >= 2**30:
            raise ValueError("linear_w4: too many tokens for one call")
        return ref.linear_w4(x, w, _bias("bias", bias, (w.n,)))
    return _cuda().linear_w4(x, *_args(w), bias)


def experts_w4(x: torch.Tensor, w1: W4Weight, w2: W4Weight, weights: torch.Tensor, ids: torch.Tensor, *,
               activation: str = "silu", expert_offset: int = 0, num_experts: int | None = None,
               w1_bias: torch.Tensor | None = None, w2_bias: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * (w2[e] act(w1[e] x[t]))`` with ``e = ids[t, j] - expert_offset``.

    ``w1 [E, 2I, H]`` is packed with ``gated=True``, ``w2 [E, H, I]`` without; ``weights`` fp32 and
    ``ids`` int32 ``[T, k]`` come from ``route_experts``. Ids of experts that are not here (expert
    parallelism) add nothing; ``num_experts`` then says how many experts the ids are of (default: those
    here), by which the GPU estimates how many tokens an expert gets and chooses its form. ``activation``:
    ``silu``, ``gelu`` (tanh form) or ``swiglu_oai``. On the GPU a call takes up to 1024 experts and 2^24
    pairs of a token and an expert.
    The activated values between the two products are held in 16 bits, in bf16 above 12 pairs per expert,
    weights exactly (to 2^-12 of them with fp16 scales and many tokens), sums in fp32. ``x`` may be
    strided; ``weights``, ``ids`` and the bf16 biases ``w1_bias [E, 2I]`` and ``w2_bias [E, H]`` are
    contiguous."""
    if not (w1.experts and w1.gated and w2.experts and not w2.gated):
        raise ValueError("experts_w4 takes w1 [E, 2I, H] packed with gated=True and w2 [E, H, I] without")
    if activation not in _ACT:
        raise ValueError(f"activation must be one of {sorted(_ACT)}, got {activation!r}")
    total = w1.shape[0] if num_experts is None else num_experts
    if total < w1.shape[0]:
        raise ValueError(f"num_experts must be at least the {w1.shape[0]} experts that are here, got {num_experts}")
    if not x.is_cuda:
        _check_rows("experts_w4", x, w1, w2)
        T, E = x.shape[0], w1.shape[0]
        if w2.k != w1.n // 2 or w2.shape[0] != E or E > 1024:
            raise ValueError(f"experts_w4: w1 {w1.shape} and w2 {w2.shape} do not match, or are more than 1024 experts")
        if ids.dim() != 2 or ids.shape[0] != T or ids.shape[1] < 1 or weights.shape != ids.shape:
            raise ValueError(f"experts_w4: weights {tuple(weights.shape)} and ids {tuple(ids.shape)} must be [tokens, top_k]")
        for name, t, dtype in (("weights", weights, torch.float32), ("ids", ids, torch.int32)):
            if t.dtype != dtype or t.is_cuda or not t.is_contiguous():
                raise ValueError(f"experts_w4: {name} must be contiguous {dtype} on the activations' device")
        if ids.numel() >= 2**24:
            raise ValueError("experts_w4: too many tokens for one call")
        if not 0 <= expert_offset < 2**30:
            raise ValueError("expert_offset out of range")
        return ref.experts_w4(x, w1, w2, weights, ids, activation, expert_offset, _bias("w1_bias", w1_bias, (E, w1.n)),
                              _bias("w2_bias", w2_bias, (E, w2.n)))
    return _cuda().experts_w4(x, *_args(w1), *_args(w2), weights, ids, _ACT[activation], expert_offset, total,
                              w1_bias, w2_bias)
