"""Physical KV pool held in 8 bits, with the interface of ``PagedKVCache``.

A token's K and V rows of one head take 258 bytes instead of 512. 16 tokens of
a block's KV head share an exponent for K and one for V, and hold e4m3 codes
over it (``ops_fp8``): no constants have to be chosen, and rows keep four
significant bits over 15 powers of two. Blocks, slots, block tables and prefix
reuse are those of the bf16 pool: the ``BlockManager`` needs no change. The
reference has no counterpart (its pool is bf16).

``get_physical_cache(layer)`` returns the layer's ``Fp8Layer`` in place of both
views, so the call order of the reference's attention layer (append, fetch the
views, attend) stays: ``PagedAttention`` and ``BatchPrefillAttention`` take it
for ``key_cache`` and ``value_cache``. ``read`` gives rows back.

A sequence's tokens are appended in order (any number a call): writing the
first of a unit's 16 tokens starts the unit anew. Slots outside the pool raise
as in ``PagedKVCache``.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import device_errors, ops_fp8
from .fp4_kv_cache import QuantisedKVCache
from .pool import fp8_bytes_per_block


@dataclass(frozen=True)
class Fp8Layer:
    """One layer of an 8-bit pool: K and V together."""

    pool: torch.Tensor  # uint8, ops_fp8.pool_shape

    @property
    def shape(self) -> tuple[int, int, int, int]:
        """[num_blocks, block_size, num_kv_heads, head_dim], as of a bf16 layer's views."""
        nb, kvh, units, _ = self.pool.shape
        return nb, units * 16, kvh, ops_fp8.HEAD_DIM

    @property
    def device(self) -> torch.device:
        return self.pool.device

    # The calls over this layer, as the attention classes and the cache make them.
    def append(self, key, value, slots, error_word) -> None:
        ops_fp8.kv_append_fp8(self.pool, key, value, slots, error_word=error_word)

    def read(self, slots, dtype, error_word):
        return ops_fp8.kv_read_fp8(self.pool, slots, dtype=dtype, error_word=error_word)

    def decode(self, out, query, block_tables, context_lens, scale, workspace, num_ctas, error_word) -> None:
        ops_fp8.paged_decode_fp8(out, query, self.pool, block_tables, context_lens, scale, workspace, num_ctas,
                                 error_word)

    def prefill(self, out, query, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale, error_word) -> None:
        ops_fp8.paged_prefill_fp8(out, query, self.pool, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale,
                                  error_word=error_word)

    def check_pair(self, value_cache) -> None:
        """Raises unless ``value_cache`` is this layer too (it holds K and V together)."""
        if not isinstance(value_cache, Fp8Layer) or value_cache.pool is not self.pool:
            raise ValueError("key_cache and value_cache must be the same layer of a PagedKVCacheFp8")


class PagedKVCacheFp8(QuantisedKVCache):
    def __init__(
        self,
        num_layers: int,
        num_blocks: int,
        block_size: int,
        num_kv_heads: int,
        head_dim: int,
        device: torch.device | str,
    ):
        if head_dim != ops_fp8.HEAD_DIM:
            raise ValueError(f"head_dim {head_dim} unsupported ({ops_fp8.HEAD_DIM} only)")
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.device = torch.device(device)
        # Zero bytes are zero values; rows that were never written read as zeros.
        shape = (num_layers, *ops_fp8.pool_shape(num_blocks, block_size, num_kv_heads))
        self.kv_cache = torch.zeros(shape, dtype=torch.uint8, device=self.device)
        if self.device.type == "cuda":
            device_errors.state(self.device)  # its word exists before any call over this cache is captured
        self.layers = [Fp8Layer(pool) for pool in self.kv_cache]

    @property
    def bytes_per_block(self) -> int:
        """K + V bytes of one block across all layers."""
        return fp8_bytes_per_block(self.num_layers, self.block_size, self.num_kv_heads)
