"""8-bit key/value cache: quantising rows as they are written, reading them back, and attention of new
tokens over the paged cache.

``KV8Cache`` is one layer's cache: per kv head and slot (one token) the codes of a key and of a value row,
in int8 or e4m3, and one fp32 scale each. A row's scale is its largest magnitude over 127 (int8) or 448
(e4m3), its codes are the nearest ones to ``value / scale`` (ties to even), and it stands for ``code * scale``.
At head dim 128 a token takes 132 bytes per row instead of the 256 of a bf16 cache.

    cache = ops.KV8Cache.alloc(num_slots, num_kv_heads, head_dim, torch.int8, device)
    ops.store_kv8(k, v, cache, out_loc)                   # bf16 [T, kv heads, head dim] into slots
    q = ops.qk_norm_rope_store_kv8(qkv, positions, cos_sin, q_norm, k_norm, eps, cache, out_loc, num_heads)  # a layer's way in
    o = ops.attention_kv8(q, cache, page_table, rows, cu_q, kv_lens, page_size=64, max_q_len=1)
    k, v = ops.load_kv8(cache, slots)                     # bf16 again

CUDA tensors run the sm_100a kernels, CPU tensors the plain form in ``ops.reference``. Calls may be captured in
CUDA graphs (lengths, tables and slots are read on the device); they keep no state of their own, so calls on
several streams are independent. Equal calls give equal results.

What is rounded on the GPU: codes are held exactly, queries too (for few rows in fp16, scaled by a power of two, where
values below 2^-31 of the row's largest lose bits); scores, maxima and sums are fp32; the product of a
probability and its value's scale is rounded once to fp16, to 2^-11 of it or 2^-31 of the row's largest such product. Indexes that are outside their tables are never
followed: see each operator for what such an entry does; the kernels record them in the device error word
(``minisgl._native.cuda().get_error()``), plain forms raise.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from minisgl._native import cuda as _cuda

from . import reference as ref

KV8_DTYPES = (torch.int8, torch.float8_e4m3fn)


@dataclass
class KV8Cache:
    k: torch.Tensor        # codes [kv heads, slots, head dim], int8 or float8_e4m3fn
    v: torch.Tensor
    k_scale: torch.Tensor  # fp32 [kv heads, slots]
    v_scale: torch.Tensor

    def __post_init__(self):
        k = self.k
        if k.dtype not in KV8_DTYPES or k.dim() != 3:
            raise ValueError(f"8-bit cache codes must be int8 or float8_e4m3fn [kv heads, slots, head dim], got {k.dtype} "
                             f"{tuple(k.shape)}")
        if k.shape[2] not in (64, 128) or k.shape[0] < 1 or k.shape[0] * k.shape[1] >= 2**31:
            raise ValueError(f"8-bit cache: head dim 64 or 128, at least one head, less than 2^31 rows, got {tuple(k.shape)}")
        if k.shape[1] < 16 or k.shape[1] % 16:
            raise ValueError(f"8-bit cache: slots come in pages of 16, got {k.shape[1]}")
        if self.v.dtype != k.dtype or self.v.shape != k.shape:
            raise ValueError(f"8-bit cache: value codes {self.v.dtype} {tuple(self.v.shape)} do not match the keys'")
        for name, t in (("k_scale", self.k_scale), ("v_scale", self.v_scale)):
            if t.dtype != torch.float32 or t.shape != k.shape[:2]:
                raise ValueError(f"8-bit cache: {name} must be fp32 {tuple(k.shape[:2])}, got {t.dtype} {tuple(t.shape)}")
        for t in (k, self.v, self.k_scale, self.v_scale):
            if t.device != k.device or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError("8-bit cache: codes and scales must be contiguous, 16-byte aligned and on one device")
        if _overlap(k, self.v) or _overlap(self.k_scale, self.v_scale):
            raise ValueError("8-bit cache: keys and values must not share memory")

    @classmethod
    def alloc(cls, num_slots: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.int8,
              device: torch.device | str = "cuda") -> "KV8Cache":
        """A cache of zeros."""
        if dtype not in KV8_DTYPES:
            raise ValueError(f"8-bit cache dtype must be int8 or float8_e4m3fn, got {dtype}")
        codes = torch.zeros(2, num_kv_heads, num_slots, head_dim, dtype=torch.uint8, device=device).view(dtype)
        scales = torch.zeros(2, num_kv_heads, num_slots, dtype=torch.float32, device=device)
        return cls(codes[0], codes[1], scales[0], scales[1])

    @property
    def num_kv_heads(self) -> int:
        return self.k.shape[0]

    @property
    def num_slots(self) -> int:
        return self.k.shape[1]

    @property
    def head_dim(self) -> int:
        return self.k.shape[2]

    @property
    def dtype(self) -> torch.dtype:
        return self.k.dtype

    @property
    def is_cuda(self) -> bool:
        return self.k.is_cuda

    @property
    def device(self) -> torch.device:
        return self.k.device

    def nbytes(self) -> int:
        return 2 * (self.k.numel() + 4 * self.k_scale.numel())


# What the kernels' bindings check, for tensors that do not go there.
def _check_like(name: str, t: torch.Tensor, dtype: torch.dtype, shape, cache: KV8Cache):
    if t.dtype != dtype or t.shape != torch.Size(shape) or t.device != cache.device:
        raise ValueError(f"{name} must be {dtype} {list(shape)} on the cache's device, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _check_ids(name: str, t: torch.Tensor, n: int, cache: KV8Cache):
    _check_like(name, t, torch.int32, (n,), cache)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def store_kv8(k: torch.Tensor, v: torch.Tensor, cache: KV8Cache, out_loc: torch.Tensor) -> None:
    """Quantises ``k`` and ``v`` (bf16 ``[T, kv heads, head dim]``, may be strided) into the slots ``out_loc``
    (int32 ``[T]``). A row's quotients are those of exact arithmetic, rounded once; a row of zeros has scale 0,
    and one that holds an infinity or a NaN has scale NaN and codes 0. A negative slot is skipped (padding), one
    beyond the cache is an error and skipped. Slots of one call differ: one that comes twice ends up with either
    row or parts of both."""
    if cache.is_cuda:
        _cuda().store_kv8(k, v, cache.k, cache.v, cache.k_scale, cache.v_scale, out_loc)
        return
    T = k.shape[0] if k.dim() else 0
    for name, t in (("k", k), ("v", v)):
        _check_like(f"store_kv8: {name}", t, torch.bfloat16, (T, cache.num_kv_heads, cache.head_dim), cache)
    _check_ids("store_kv8: out_loc", out_loc, T, cache)
    if T and int(out_loc.max()) >= cache.num_slots:
        raise ValueError(f"store_kv8: slot {int(out_loc.max())} of {cache.num_slots}")
    ref.store_kv8(k, v, cache, out_loc)


def qk_norm_rope_store_kv8(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, q_norm: torch.Tensor | None,
                           k_norm: torch.Tensor | None, eps: float, cache: KV8Cache, out_loc: torch.Tensor, nq: int) -> torch.Tensor:
    """``qk_norm_rope_store`` into an 8-bit cache, in one kernel: splits ``qkv`` (bf16 ``[T, (nq + 2 kv heads) * head
    dim]``) into heads, takes queries and keys through RMSNorm (with weights, bf16 ``[head dim]``) and RoPE
    (``cos_sin`` fp32 ``[positions, head dim]``, ``positions`` int32 ``[T]``), and stores keys and values as ``store_kv8``
    does with their bf16 rows. Returns the queries, bf16 ``[T, nq, head dim]``. A position outside ``cos_sin`` is an
    error: the token's key is not stored, its queries are undefined."""
    if cache.is_cuda:
        return _cuda().qk_norm_rope_store_kv8(qkv, positions, cos_sin, q_norm, k_norm, eps, cache.k, cache.v, cache.k_scale,
                                              cache.v_scale, out_loc, nq)
    T, nkv, hd = qkv.shape[0] if qkv.dim() else 0, cache.num_kv_heads, cache.head_dim
    if nq < 1:
        raise ValueError(f"qk_norm_rope_store_kv8: {nq} query heads")
    _check_like("qk_norm_rope_store_kv8: qkv", qkv, torch.bfloat16, (T, (nq + 2 * nkv) * hd), cache)
    _check_ids("qk_norm_rope_store_kv8: positions", positions, T, cache)
    _check_ids("qk_norm_rope_store_kv8: out_loc", out_loc, T, cache)
    _check_like("qk_norm_rope_store_kv8: cos_sin", cos_sin, torch.float32, (*cos_sin.shape[:1], hd), cache)
    if (q_norm is None) != (k_norm is None):
        raise ValueError("qk_norm_rope_store_kv8: q_norm and k_norm must both be given or both absent")
    for w in (q_norm, k_norm):
        if w is not None:
            _check_like("qk_norm_rope_store_kv8: norm weights", w, torch.bfloat16, (hd,), cache)
    if not all(t.is_contiguous() for t in (qkv, cos_sin, q_norm, k_norm) if t is not None):
        raise ValueError("qk_norm_rope_store_kv8: qkv, cos_sin and norm weights must be contiguous")
    if T and not 0 <= int(positions.min()) <= int(positions.max()) < cos_sin.shape[0]:
        raise ValueError(f"qk_norm_rope_store_kv8: a position outside the {cos_sin.shape[0]} of cos_sin")
    if T and int(out_loc.max()) >= cache.num_slots:
        raise ValueError(f"qk_norm_rope_store_kv8: slot {int(out_loc.max())} of {cache.num_slots}")
    return ref.qk_norm_rope_store_kv8(qkv, positions, cos_sin, q_norm, k_norm, eps, cache, out_loc, nq)


def load_kv8(cache: KV8Cache, slots: torch.Tensor):
    """The rows that the cache's codes at ``slots`` (int32 ``[n]``, in any order, also repeated) stand for:
    (k, v), bf16 ``[n, kv heads, head dim]``, ``code * scale`` rounded to bf16. A negative slot gives zeros, one
    beyond the cache is an error and gives zeros."""
    if cache.is_cuda:
        return _cuda().load_kv8(cache.k, cache.v, cache.k_scale, cache.v_scale, slots)
    _check_ids("load_kv8: slots", slots, slots.numel(), cache)
    if slots.numel() and int(slots.max()) >= cache.num_slots:
        raise ValueError(f"load_kv8: slot {int(slots.max())} of {cache.num_slots}")
    return ref.load_kv8(cache, slots)


def attention_kv8(q: torch.Tensor, cache: KV8Cache, page_table: torch.Tensor, rows: torch.Tensor, cu_q: torch.Tensor,
                  kv_lens: torch.Tensor, *, page_size: int, max_q_len: int | None = None, scale: float | None = None,
                  window: int = -1, sinks: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of new tokens over the paged 8-bit cache, which holds the new tokens' rows already.

    ``q`` (bf16 ``[T, heads, head dim]``, may be strided) holds the queries of B requests one after another, those of
    request b at ``cu_q[b]`` up to ``cu_q[b + 1]`` (int32 ``[B + 1]``, from 0, not falling): one each when decoding, some
    when drafted tokens are verified, many in a prompt's chunk. They are the last ones of the request's ``kv_lens[b]``
    positions (int32 ``[B]``), and position p has its key and value in slot ``page_table[rows[b], p]`` (int32
    ``[R, W]``, token by token as in the engine; ``rows`` int32 ``[B]``). Pages are ``page_size`` consecutive slots that
    start at a multiple of it; a multiple of 16, so the table is read at every 16, 32 or 64 positions only.

    A query at position p sees the keys up to p, with ``window`` > 0 only the last ``window`` of them. The logits are
    ``scale`` (default ``head_dim ** -0.5``) times the products; ``sinks`` (fp32 ``[heads]``) are logits that take their
    share of the softmax without a value. A query that sees no key (a padded request of length 0) gives zeros.
    ``max_q_len`` says how many queries a request has at most: the form is chosen by it, results do not hang on it.

    Returns bf16 ``[T, heads, head dim]``; rows behind ``cu_q[B]`` are zeros, in ``out`` (contiguous, not overlapping
    ``q``) they are left as they were. A request with a row outside the table, a length beyond the table's width or
    queries outside ``q`` is an error and its rows are zeros where they exist; a page that is not in the cache is an
    error and its keys and values count as zeros."""
    if cache.is_cuda:
        return _cuda().attention_kv8(q, cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, rows, cu_q, kv_lens,
                                     page_size, -1 if max_q_len is None else max_q_len, scale, window, sinks, out)
    B = rows.numel()
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[2] != cache.head_dim or q.device != cache.device:
        raise ValueError(f"attention_kv8: q must be bf16 [tokens, heads, {cache.head_dim}] on the cache's device, got {q.dtype} "
                         f"{tuple(q.shape)} on {q.device}")
    T, nq, hd = q.shape
    if nq < 1 or nq % cache.num_kv_heads or nq // cache.num_kv_heads > 128:
        raise ValueError(f"attention_kv8: {nq} query heads over {cache.num_kv_heads} kv heads (1 to 128 each)")
    if T * nq >= 2**30 or B >= 2**24:
        raise ValueError("attention_kv8: too many queries for one call")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != cache.device or (
            page_table.numel() and page_table.stride(1) != 1):
        raise ValueError(f"attention_kv8: page_table must be int32 [rows, positions], got {page_table.dtype} {tuple(page_table.shape)}")
    _check_ids("attention_kv8: rows", rows, B, cache)
    _check_ids("attention_kv8: cu_q", cu_q, B + 1, cache)
    _check_ids("attention_kv8: kv_lens", kv_lens, B, cache)
    if page_size < 16 or page_size % 16:
        raise ValueError(f"attention_kv8: pages must be a multiple of 16 slots, got {page_size}")
    if max_q_len is not None and max_q_len < 0:
        raise ValueError(f"attention_kv8: max_q_len must not be negative, got {max_q_len}")
    if window < 1 and window != -1:
        raise ValueError(f"attention_kv8: window must be positive, or -1 for none, got {window}")
    if scale is not None and not abs(scale) < float("inf"):
        raise ValueError(f"attention_kv8: scale must be finite, got {scale}")
    if sinks is not None:
        _check_like("attention_kv8: sinks", sinks, torch.float32, (nq,), cache)
        if not sinks.is_contiguous():
            raise ValueError("attention_kv8: sinks must be contiguous")
    if out is not None:
        _check_like("attention_kv8: out", out, torch.bfloat16, q.shape, cache)
        if not out.is_contiguous():
            raise ValueError("attention_kv8: out must be contiguous")
        if T and _overlap(q, out):
            raise ValueError("attention_kv8: out must not overlap q")
    return ref.attention_kv8(q, cache, page_table, rows, cu_q, kv_lens, page_size, hd**-0.5 if scale is None else scale, window,
                             sinks, out)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the spans of memory that two tensors lie in meet."""
    def span(t):
        last = sum((n - 1) * abs(s) for n, s in zip(t.shape, t.stride())) + 1
        return t.data_ptr(), t.data_ptr() + last * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1
