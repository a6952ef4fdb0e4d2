"""Physical KV tensors: per layer K and V of shape
(num_blocks, block_size, num_kv_heads, head_dim), the reference layout
(cache/kv_cache.py:41-50) that the HIP kernels read and write in place.
All layers live in one allocation [num_layers, 2, num_blocks, ...].

With ``kv_cache_dtype`` "int8" or "fp8" the cache holds 8-bit codes and one
fp32 scale per token and kv head instead (ops.QuantKV): each head's rows of a
block in one run, [num_layers, 2, num_blocks, num_kv_heads, block_size, ...]."""

from __future__ import annotations

from typing import Union

import torch

from .. import ops


class KVCache:
    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int,
                 head_dim: int, dtype: torch.dtype = torch.float16, device: str = "cuda",
                 kv_cache_dtype: str = "auto") -> None:
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = device
        self.kv_cache_dtype = kv_cache_dtype
        self.scales = None
        if kv_cache_dtype != "auto":
            shape = (num_layers, 2, num_blocks, num_kv_heads, block_size)
            self.storage = torch.zeros((*shape, head_dim), dtype=torch.int8,
                                       device=device).view(ops.QUANT_DTYPES[kv_cache_dtype])
            self.scales = torch.zeros(shape, dtype=torch.float32, device=device)
            codes, scales = self.storage.transpose(3, 4), self.scales.transpose(3, 4)
            self.quant_caches = [ops.QuantKV(codes[i, 0], codes[i, 1], scales[i, 0], scales[i, 1])
                                 for i in range(num_layers)]
            return
        self.storage = torch.zeros((num_layers, 2, num_blocks, block_size, num_kv_heads, head_dim),
                                   dtype=dtype, device=device)
        self.key_caches = [self.storage[i, 0] for i in range(num_layers)]
        self.value_caches = [self.storage[i, 1] for i in range(num_layers)]

    def get_kv(self, layer_idx: int) -> Union[tuple[torch.Tensor, torch.Tensor], ops.QuantKV]:
        """A layer's (key, value) caches, or its QuantKV."""
        if self.scales is not None:
            return self.quant_caches[layer_idx]
        return self.key_caches[layer_idx], self.value_caches[layer_idx]

    @property
    def total_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.storage, self.scales)
                   if t is not None)

    @classmethod
    def profile_num_blocks(cls, available_memory_bytes: int, num_layers: int, block_size: int,
                           num_kv_heads: int, head_dim: int,
                           dtype: torch.dtype = torch.float16,
                           kv_cache_dtype: str = "auto") -> int:
        row = head_dim * torch.tensor([], dtype=dtype).element_size()
        if kv_cache_dtype != "auto":
            row = head_dim + 4
        per_block = 2 * block_size * num_kv_heads * row * num_layers
        return max(1, int(available_memory_bytes // per_block))
