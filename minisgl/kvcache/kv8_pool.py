"""Paged KV pool in 8 bits: one ``ops.KV8Cache`` per layer (int8 or e4m3 codes, one fp32 scale per key and per value
row), a little more than half the bytes of a bf16 pool. The engine makes it for ``kv_cache_dtype`` "int8" or
"fp8_e4m3" (this engine's own; the reference's pool, python/minisgl/kvcache/mha_pool.py:10-68, has the model's type only).

Layout: codes ``[layers, 2, kv heads, slots, head_dim]``, scales ``[layers, 2, kv heads, slots]``: a head's page is one
run of codes and one of scales.
"""

from __future__ import annotations

import torch

from minisgl import ops

from .base import BaseKVCachePool

KV8_DTYPES = {"int8": torch.int8, "fp8_e4m3": torch.float8_e4m3fn}


class KV8Pool(BaseKVCachePool):
    def __init__(self, num_kv_heads: int, num_layers: int, head_dim: int, num_pages: int, page_size: int,
                 dtype: torch.dtype, device: torch.device):
        from minisgl.parallel import get_tp_info
        from minisgl.utils import div_even

        tp = get_tp_info()
        self.local_kv_heads = div_even(num_kv_heads, tp.size, allow_replicate=True)
        self.head_dim = head_dim
        self.page_size = page_size
        self.num_slots = num_pages * page_size
        rows = (num_layers, 2, self.local_kv_heads, self.num_slots)
        self._codes = torch.zeros(*rows, head_dim, dtype=torch.uint8, device=device).view(dtype)
        self._scales = torch.zeros(rows, dtype=torch.float32, device=device)
        self._layers = [ops.KV8Cache(c[0], c[1], s[0], s[1]) for c, s in zip(self._codes, self._scales)]

    def layer(self, layer_id: int) -> ops.KV8Cache:
        return self._layers[layer_id]

    def k_cache(self, layer_id: int) -> torch.Tensor:
        """The keys' codes; their scales are ``layer(layer_id).k_scale``."""
        return self._layers[layer_id].k

    def v_cache(self, layer_id: int) -> torch.Tensor:
        return self._layers[layer_id].v

    def store_kv(self, k: torch.Tensor, v: torch.Tensor, out_loc: torch.Tensor, layer_id: int) -> None:
        heads = (k.shape[0], self.local_kv_heads, self.head_dim)
        ops.store_kv8(k.view(heads), v.view(heads), self._layers[layer_id], out_loc)

    def load_kv(self, slots: torch.Tensor, layer_id: int):
        """The rows at ``slots``, as (k, v) in bf16."""
        return ops.load_kv8(self._layers[layer_id], slots)

    @property
    def device(self) -> torch.device:
        return self._codes.device

    @property
    def dtype(self) -> torch.dtype:
        return self._codes.dtype

    @property
    def num_layers(self) -> int:
        return len(self._layers)

    @property
    def bytes_per_token(self) -> int:
        return 2 * self.num_layers * self.local_kv_heads * (self.head_dim + 4)
