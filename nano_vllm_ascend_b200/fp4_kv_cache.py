"""Physical KV pool held in 4 bits, with the interface of ``PagedKVCache``.

A token's K and V rows of one head take 144 bytes instead of 512, so the same
HBM holds 3.56 times the tokens and decode attention reads that much less. A
row's 128 dims are 8 groups of 16; each group has an e4m3 scale and e2m1 codes
(``ops_fp4``), relative to a constant of its layer, a power of two that moves
rows of unusual magnitude into the scales' range. Blocks, slots, block tables
and prefix reuse are those of the bf16 pool: the ``BlockManager`` needs no
change. The reference has no counterpart (its pool is bf16).

``get_physical_cache(layer)`` returns the layer's ``Fp4Layer`` in place of both
views, so the call order of the reference's attention layer (append, fetch the
views, attend) stays: ``PagedAttention`` and ``BatchPrefillAttention`` take it
for ``key_cache`` and ``value_cache``. ``read`` gives rows back.

Slots outside the pool raise as in ``PagedKVCache``.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Sequence

import torch

from . import device_errors, ops_fp4
from .paged_kv_cache import _packed_rows, copy_pool_blocks
from .pool import fp4_bytes_per_block


@dataclass(frozen=True)
class Fp4Layer:
    """One layer of a 4-bit pool: K and V together, and the layer's constants."""

    pool: torch.Tensor  # uint8, ops_fp4.pool_shape
    k_scale: float = 1.0
    v_scale: float = 1.0

    @property
    def shape(self) -> tuple[int, int, int, int]:
        """[num_blocks, block_size, num_kv_heads, head_dim], as of a bf16 layer's views."""
        nb, kvh, units, _ = self.pool.shape
        return nb, units * 16, kvh, ops_fp4.HEAD_DIM

    @property
    def device(self) -> torch.device:
        return self.pool.device

    # The calls over this layer, as the attention classes and the cache make them.
    def append(self, key, value, slots, error_word) -> None:
        ops_fp4.kv_append_fp4(self.pool, key, value, slots, self.k_scale, self.v_scale, error_word=error_word)

    def read(self, slots, dtype, error_word):
        return ops_fp4.kv_read_fp4(self.pool, slots, self.k_scale, self.v_scale, dtype=dtype, error_word=error_word)

    def decode(self, out, query, block_tables, context_lens, scale, workspace, num_ctas, error_word) -> None:
        ops_fp4.paged_decode_fp4(out, query, self.pool, block_tables, context_lens, scale, workspace, num_ctas,
                                 self.k_scale, self.v_scale, error_word)

    def prefill(self, out, query, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale, error_word) -> None:
        ops_fp4.paged_prefill_fp4(out, query, self.pool, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale,
                                  self.k_scale, self.v_scale, error_word=error_word)

    def check_pair(self, value_cache) -> None:
        """Raises unless ``value_cache`` is this layer too (it holds K and V together)."""
        if not isinstance(value_cache, Fp4Layer) or value_cache.pool is not self.pool:
            raise ValueError("key_cache and value_cache must be the same layer of a PagedKVCacheFp4")


def _constants(name: str, value: float | Sequence[float], layers: int) -> list[float]:
    values = [float(value)] * layers if isinstance(value, (int, float)) else [float(v) for v in value]
    if len(values) != layers:
        raise ValueError(f"{name}: {len(values)} constants for {layers} layers")
    for v in values:
        if not (v > 0 and math.isfinite(v) and math.frexp(v)[0] == 0.5 and 2.0 ** -60 <= v <= 2.0 ** 60):
            raise ValueError(f"{name}: {v} is not a power of two in [2^-60, 2^60]")
    return values


class QuantisedKVCache:
    """What the pools held in fewer bits share: their checks, and calls that report into the device's error word.
    ``kv_cache`` is [num_layers, num_blocks, ...], ``layers`` the layers that attention takes."""

    def _device_slots(self, slot_mapping: torch.Tensor) -> torch.Tensor:
        if not slot_mapping.is_cuda and slot_mapping.numel():
            lo, hi = int(slot_mapping.min()), int(slot_mapping.max())
            if lo < 0 or hi >= self.num_blocks * self.block_size:
                bad = lo if lo < 0 else hi
                raise IndexError(f"index_copy_(): index {bad} is out of bounds for dimension 0 with size "
                                 f"{self.num_blocks * self.block_size}")
        return slot_mapping.to(device=self.device, dtype=torch.long)

    def write(self, layer_idx: int, key_states: torch.Tensor, value_states: torch.Tensor,
              slot_mapping: torch.Tensor) -> None:
        """Quantises the rows (bf16 or fp16) into ``layer_idx`` at ``slot_mapping``. Slots must differ."""
        total_tokens, num_kv_heads, head_dim = key_states.shape
        if num_kv_heads != self.num_kv_heads or head_dim != self.head_dim:
            raise ValueError(f"kv shape mismatch: got {tuple(key_states.shape)}")
        if slot_mapping.numel() != total_tokens:
            raise ValueError(f"slot_mapping numel {slot_mapping.numel()} != total_tokens {total_tokens}")
        if value_states.shape != key_states.shape:
            raise ValueError(f"kv shape mismatch: got {tuple(value_states.shape)}")
        if total_tokens == 0:
            return
        slots = self._device_slots(slot_mapping)
        layer = self.layers[layer_idx]
        with torch.cuda.device(self.device):
            errors = device_errors.state(self.device)
            errors.raise_if_flagged()
            layer.append(_packed_rows(key_states.to(self.device)), _packed_rows(value_states.to(self.device)), slots,
                         errors.word)
            errors.launched()

    def read(self, layer_idx: int, slot_mapping: torch.Tensor,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """The K and V rows [slots, kv_heads, head_dim] that ``layer_idx`` holds at ``slot_mapping``."""
        slots = self._device_slots(slot_mapping)
        layer = self.layers[layer_idx]
        with torch.cuda.device(self.device):
            errors = device_errors.state(self.device)
            errors.raise_if_flagged()
            rows = layer.read(slots, dtype, errors.word)
            errors.launched()
        return rows

    def get_physical_cache(self, layer_idx: int):
        return self.layers[layer_idx], self.layers[layer_idx]

    def copy_blocks(self, pairs) -> None:
        """Copies blocks, (source, destination) each, in every layer; source -1
        clears the destination (see ``copy_pool_blocks``)."""
        copy_pool_blocks([self.kv_cache], pairs)


class PagedKVCacheFp4(QuantisedKVCache):
    def __init__(
        self,
        num_layers: int,
        num_blocks: int,
        block_size: int,
        num_kv_heads: int,
        head_dim: int,
        device: torch.device | str,
        k_scale: float | Sequence[float] = 1.0,
        v_scale: float | Sequence[float] = 1.0,
    ):
        if head_dim != ops_fp4.HEAD_DIM:
            raise ValueError(f"head_dim {head_dim} unsupported ({ops_fp4.HEAD_DIM} only)")
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.device = torch.device(device)
        # Zero bytes are zero values; rows that were never written read as zeros.
        shape = (num_layers, *ops_fp4.pool_shape(num_blocks, block_size, num_kv_heads))
        constants = zip(_constants("k_scale", k_scale, num_layers), _constants("v_scale", v_scale, num_layers))
        self.kv_cache = torch.zeros(shape, dtype=torch.uint8, device=self.device)
        if self.device.type == "cuda":
            device_errors.state(self.device)  # its word exists before any call over this cache is captured
        self.layers = [Fp4Layer(self.kv_cache[i], ks, vs) for i, (ks, vs) in enumerate(constants)]

    @property
    def bytes_per_block(self) -> int:
        """K + V bytes of one block across all layers."""
        return fp4_bytes_per_block(self.num_layers, self.block_size, self.num_kv_heads)
