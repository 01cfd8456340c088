"""KV-pool sizing from free HBM (src/nanovllm_ascend/model_runner.py:113-125)."""

from __future__ import annotations

import torch

from ._lib import FP4_UNIT_BYTES, FP4_UNIT_TOKENS, FP8_UNIT_BYTES, FP8_UNIT_TOKENS


def bytes_per_block(num_layers: int, block_size: int, num_kv_heads: int, head_dim: int,
                    dtype: torch.dtype = torch.bfloat16) -> int:
    """K and V bytes of one pool block across all layers."""
    return 2 * num_layers * block_size * num_kv_heads * head_dim * torch.tensor([], dtype=dtype).element_size()


def fp4_bytes_per_block(num_layers: int, block_size: int, num_kv_heads: int) -> int:
    """K and V bytes of one block of a 4-bit pool (head_dim 128) across all layers."""
    return num_layers * num_kv_heads * (block_size // FP4_UNIT_TOKENS) * FP4_UNIT_BYTES


def fp8_bytes_per_block(num_layers: int, block_size: int, num_kv_heads: int) -> int:
    """K and V bytes of one block of an 8-bit pool (head_dim 128) across all layers."""
    return num_layers * num_kv_heads * (block_size // FP8_UNIT_TOKENS) * FP8_UNIT_BYTES


def num_blocks_for_budget(free_bytes: int, total_bytes: int, memory_utilization: float, num_layers: int,
                          block_size: int, num_kv_heads: int, head_dim: int,
                          dtype: torch.dtype = torch.bfloat16, block_bytes: int | None = None) -> int:
    """(total * utilization - used) // bytes_per_block, as the reference sizes its pool
    (``block_bytes``: the bytes of a block, where they are not those of a ``dtype`` pool)."""
    used = total_bytes - free_bytes
    budget = int(total_bytes * memory_utilization) - used
    return max(0, budget // (block_bytes or bytes_per_block(num_layers, block_size, num_kv_heads, head_dim, dtype)))


def num_blocks_from_memory(memory_utilization: float, num_layers: int, block_size: int, num_kv_heads: int,
                           head_dim: int, dtype: torch.dtype = torch.bfloat16,
                           device: torch.device | str | None = None, block_bytes: int | None = None) -> int:
    free, total = torch.cuda.mem_get_info(device)
    return num_blocks_for_budget(free, total, memory_utilization, num_layers, block_size, num_kv_heads, head_dim,
                                 dtype, block_bytes)
