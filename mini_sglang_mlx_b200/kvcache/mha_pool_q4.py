"""KV page pool in HBM held in 4 bits: per layer one K and one V pool of ``kv_cache_q4_shape``, written through
``store_kv_cache_q4`` and read back through ``load_kv_cache_q4``.

The interface of ``MHAKVCache`` (no counterpart in the reference, whose pools hold the data type).  Slots go by pages of a multiple
of 16 tokens (``CacheManager(page_size=16)``, slot = page * page_size + offset); a token of a head takes 4.5 bits an
element, scales and biases among them, so the pool of a device holds 3.5 times as many tokens.
"""
from __future__ import annotations

from typing import Tuple

import torch

from ..kernel import KV4_ROWS, kv_cache_q4_shape, load_kv_cache_q4, store_kv_cache_q4


class MHAKVCacheQ4:
    def __init__(self, num_kv_heads: int, num_layers: int, head_dim: int, num_pages: int,
                 dtype: torch.dtype, device="cuda") -> None:
        """``num_pages``: token slots, as in ``MHAKVCache``; rounded up to whole blocks of sixteen.  ``dtype``: of the rows that are
        stored and read, and of the scales and biases."""
        self._num_layers = num_layers
        self._dtype = dtype
        self._shape = kv_cache_q4_shape(num_pages, num_kv_heads, head_dim)
        self._buffer = torch.zeros((2, num_layers, *self._shape), dtype=dtype, device=device)
        self._k_buffer = [self._buffer[0, i] for i in range(num_layers)]
        self._v_buffer = [self._buffer[1, i] for i in range(num_layers)]

    def k_cache(self, index: int) -> torch.Tensor:
        return self._k_buffer[index]

    def v_cache(self, index: int) -> torch.Tensor:
        return self._v_buffer[index]

    def store_kv(self, k: torch.Tensor, v: torch.Tensor, out_loc: torch.Tensor, layer_id: int) -> None:
        assert out_loc.dtype == torch.int32, "out_loc must be int32"
        if len(out_loc) != k.shape[0] or len(out_loc) != v.shape[0]:
            raise ValueError(
                f"store_kv shape mismatch: len(out_loc)={len(out_loc)}, "
                f"k.shape={tuple(k.shape)}, v.shape={tuple(v.shape)}")
        store_kv_cache_q4(self._k_buffer[layer_id], self._v_buffer[layer_id], out_loc, k, v)

    def load_kv(self, slots: torch.Tensor, layer_id: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """The rows at ``slots`` as ``(len(slots), num_kv_heads, head_dim)`` keys and values (to hand a prefix to another pool)."""
        return load_kv_cache_q4(self._k_buffer[layer_id], self._v_buffer[layer_id], slots)

    @property
    def dtype(self) -> torch.dtype:
        return self._dtype

    @property
    def num_layers(self) -> int:
        return self._num_layers

    @property
    def num_pages(self) -> int:
        return self._shape[0] * KV4_ROWS
