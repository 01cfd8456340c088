"""Tensor-level wrappers over the kernels of the 4-bit KV pool.

As in ``ops``, each function validates devices, dtypes, shapes and strides,
then calls the matching ``nvk_fp4_*`` entry point (include/nvk_paged_kv.h) on
the tensors' current CUDA stream, and there is no non-CUDA path.

``kv_cache`` is ONE layer of the pool, K and V together: contiguous uint8
[num_blocks, kv_heads, block_size / 16, 2304] (``pool_shape``), zero-filled
once when it is allocated. A row's 128 dims are 8 groups of 16 with an e4m3
scale ``s = rn(amax / 6)`` and e2m1 codes ``rn(x / s)`` each, of the row
divided by the layer's constant ``k_scale`` or ``v_scale`` (a power of two);
the values that the codes stand for are exact in bf16. Slots, block tables
and lengths are those of the bf16 pool.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _require_cuda, _require_rows

_BF16 = torch.bfloat16
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
HEAD_DIM = 128


def pool_shape(num_blocks: int, block_size: int, num_kv_heads: int) -> tuple[int, int, int, int]:
    """The shape of one layer's uint8 pool."""
    if block_size not in (16, 32, 64, 128, 256):
        raise ValueError(f"block_size {block_size} unsupported (a power of two in [16, 256])")
    return num_blocks, num_kv_heads, block_size // _lib.FP4_UNIT_TOKENS, _lib.FP4_UNIT_BYTES


def _call(dev: torch.device, name: str, *args) -> None:
    """Calls ``name`` on ``dev`` and its current stream (the last argument)."""
    if dev.index == torch.cuda.current_device():
        _lib.call(name, *args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, torch.cuda.current_stream().cuda_stream)


def _check_pool(who: str, kv_cache: torch.Tensor) -> tuple[int, int, int]:
    """(blocks, block size, KV heads) of a layer's pool."""
    if kv_cache.dtype != torch.uint8 or kv_cache.dim() != 4 or kv_cache.shape[3] != _lib.FP4_UNIT_BYTES \
            or not kv_cache.is_contiguous():
        raise ValueError(f"{who}: kv_cache must be contiguous uint8 [blocks, kv_heads, block_size / 16, "
                         f"{_lib.FP4_UNIT_BYTES}], got {kv_cache.dtype} {tuple(kv_cache.shape)}")
    nb, kvh, units, _ = kv_cache.shape
    return nb, units * _lib.FP4_UNIT_TOKENS, kvh


def _check_index(who: str, name: str, t: torch.Tensor, dtype: torch.dtype, count: int) -> torch.Tensor:
    if t.dtype != dtype or t.numel() != count:
        raise ValueError(f"{who}: {name} must be {dtype} with {count} entries, got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def _error_ptr(who: str, error_word: torch.Tensor | None, dev: torch.device) -> int:
    if error_word is None:
        return 0
    _require_cuda("error_word", error_word, dev)
    if error_word.dtype != torch.int32 or error_word.numel() < 1:
        raise ValueError(f"{who}: error_word must be a device int32")
    return error_word.data_ptr()


def kv_append_fp4(kv_cache: torch.Tensor, key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor,
                  k_scale: float = 1.0, v_scale: float = 1.0, error_word: torch.Tensor | None = None) -> None:
    """Quantises the rows ``key`` / ``value`` ([tokens, kv_heads, 128], bf16 or
    fp16; the token stride may be larger) into the pool at ``slot_mapping``
    (int64). Slots must differ; one outside the pool is skipped and sets bit 4
    of ``error_word``."""
    who = "kv_append_fp4"
    dev = kv_cache.device
    for name, t in (("kv_cache", kv_cache), ("key", key), ("value", value), ("slot_mapping", slot_mapping)):
        _require_cuda(name, t, dev)
    nb, bs, kvh = _check_pool(who, kv_cache)
    if key.dtype not in _DTYPES or value.dtype != key.dtype:
        raise ValueError(f"{who}: key and value must both be bfloat16 or float16, got {key.dtype} and {value.dtype}")
    _require_rows("key", key)
    _require_rows("value", value)
    if key.shape != value.shape or key.shape[1] != kvh or key.shape[2] != HEAD_DIM:
        raise ValueError(f"kv shape mismatch: got {tuple(key.shape)} / {tuple(value.shape)}")
    slots = _check_index(who, "slot_mapping", slot_mapping, torch.int64, key.shape[0])
    _call(dev, "nvk_fp4_append", key.data_ptr(), value.data_ptr(), key.stride(0), value.stride(0),
          kv_cache.data_ptr(), slots.data_ptr(), key.shape[0], nb, bs, kvh, HEAD_DIM, _DTYPES[key.dtype], k_scale,
          v_scale, _error_ptr(who, error_word, dev))


def kv_read_fp4(kv_cache: torch.Tensor, slot_mapping: torch.Tensor, k_scale: float = 1.0, v_scale: float = 1.0,
                dtype: torch.dtype = _BF16, key_out: torch.Tensor | None = None,
                value_out: torch.Tensor | None = None,
                error_word: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows [tokens, kv_heads, 128] that the pool holds at
    ``slot_mapping`` (int64; any order, repeats allowed), as ``dtype``; a slot
    outside the pool gives zeros and sets bit 4 of ``error_word``."""
    who = "kv_read_fp4"
    dev = kv_cache.device
    for name, t in (("kv_cache", kv_cache), ("slot_mapping", slot_mapping)):
        _require_cuda(name, t, dev)
    nb, bs, kvh = _check_pool(who, kv_cache)
    if dtype not in _DTYPES:
        raise ValueError(f"{who}: dtype must be bfloat16 or float16, got {dtype}")
    tokens = slot_mapping.numel()
    slots = _check_index(who, "slot_mapping", slot_mapping, torch.int64, tokens)
    outs = []
    for name, t in (("key_out", key_out), ("value_out", value_out)):
        if t is None:
            t = torch.empty(tokens, kvh, HEAD_DIM, dtype=dtype, device=dev)
        else:
            _require_cuda(name, t, dev)
            if t.shape != (tokens, kvh, HEAD_DIM) or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"{who}: {name} must be contiguous {dtype} [tokens, kv_heads, {HEAD_DIM}]")
        outs.append(t)
    _call(dev, "nvk_fp4_read", outs[0].data_ptr(), outs[1].data_ptr(), kv_cache.data_ptr(), slots.data_ptr(), tokens,
          nb, bs, kvh, HEAD_DIM, _DTYPES[dtype], k_scale, v_scale, _error_ptr(who, error_word, dev))
    return outs[0], outs[1]


def qk_norm_rope_append_fp4(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, q_weight: torch.Tensor,
                            k_weight: torch.Tensor, eps: float, cos_table: torch.Tensor, sin_table: torch.Tensor,
                            positions: torch.Tensor, kv_cache: torch.Tensor, slot_mapping: torch.Tensor,
                            k_scale: float = 1.0, v_scale: float = 1.0, query_out: torch.Tensor | None = None,
                            error_word: torch.Tensor | None = None) -> torch.Tensor:
    """``ops.qk_norm_rope_append`` into a 4-bit pool: per-head RMSNorm of q and
    k, rotary embedding, and the append of the rotated k and of v, in one
    kernel. Returns the rotated query [tokens, heads, 128]."""
    who = "qk_norm_rope_append_fp4"
    dev = query.device
    for name, t in (("query", query), ("key", key), ("value", value), ("q_weight", q_weight),
                    ("k_weight", k_weight), ("cos_table", cos_table), ("sin_table", sin_table),
                    ("positions", positions), ("kv_cache", kv_cache), ("slot_mapping", slot_mapping)):
        _require_cuda(name, t, dev)
    for name, t in (("query", query), ("key", key), ("value", value)):
        _require_rows(name, t)
        if t.dtype != _BF16:
            raise ValueError(f"{who}: {name} must be bfloat16")
    tokens, num_heads, head_dim = query.shape
    nb, bs, kvh = _check_pool(who, kv_cache)
    if key.shape != (tokens, kvh, HEAD_DIM) or value.shape != key.shape or head_dim != HEAD_DIM:
        raise ValueError(f"kv shape mismatch: got {tuple(key.shape)} / {tuple(value.shape)}")
    for t in (q_weight, k_weight):
        if t.numel() != HEAD_DIM or t.dtype != _BF16 or not t.is_contiguous():
            raise ValueError(f"{who}: q_weight/k_weight must be contiguous bfloat16 [head_dim]")
    if cos_table.dtype != torch.float32 or sin_table.dtype != torch.float32 or cos_table.dim() != 2 \
            or sin_table.shape != cos_table.shape or cos_table.shape[1] != HEAD_DIM \
            or not (cos_table.is_contiguous() and sin_table.is_contiguous()):
        raise ValueError(f"{who}: cos/sin tables must be contiguous float32 [max_position, head_dim]")
    pos = _check_index(who, "positions", positions, torch.int64, tokens)
    slots = _check_index(who, "slot_mapping", slot_mapping, torch.int64, tokens)
    if query_out is None:
        query_out = torch.empty(tokens, num_heads, HEAD_DIM, dtype=_BF16, device=dev)
    else:
        _require_cuda("query_out", query_out, dev)
        if query_out.shape != query.shape or not query_out.is_contiguous() or query_out.dtype != _BF16:
            raise ValueError(f"{who}: query_out must be a contiguous bf16 [tokens, heads, head_dim]")
    _call(dev, "nvk_fp4_qk_norm_rope_append", query.data_ptr(), key.data_ptr(), value.data_ptr(), query.stride(0),
          key.stride(0), value.stride(0), q_weight.data_ptr(), k_weight.data_ptr(), eps, cos_table.data_ptr(),
          sin_table.data_ptr(), cos_table.shape[0], pos.data_ptr(), query_out.data_ptr(), kv_cache.data_ptr(),
          slots.data_ptr(), tokens, nb, bs, num_heads, kvh, HEAD_DIM, k_scale, v_scale,
          _error_ptr(who, error_word, dev))
    return query_out


def decode_fp4_workspace_bytes(num_heads: int, num_kv_heads: int, head_dim: int = HEAD_DIM, num_ctas: int = 0) -> int:
    """Workspace bytes of paged_decode_fp4 for any batch (num_ctas 0 = one CTA per SM of the current device)."""
    out = ctypes.c_size_t(0)
    _lib.call("nvk_fp4_paged_decode_workspace_size", num_heads, num_kv_heads, head_dim, num_ctas, ctypes.byref(out))
    return int(out.value)


def _table_stride(block_tables: torch.Tensor) -> int:
    """Elements between the rows (of a single row: its width, whatever its stride says)."""
    return block_tables.stride(0) if block_tables.shape[0] > 1 else block_tables.shape[1]


def _check_attention(who: str, out, query, kv_cache, block_tables, lens) -> tuple[int, int, int, int]:
    """Checks what decode and prefill share; returns (blocks, block size, KV heads, sequences)."""
    dev = query.device
    for name, t in (("out", out), ("query", query), ("kv_cache", kv_cache), ("block_tables", block_tables),
                    ("lens", lens)):
        _require_cuda(name, t, dev)
    if query.dtype != _BF16 or out.dtype != _BF16:
        raise ValueError(f"{who}: query and out must be bfloat16")
    if query.dim() != 3 or query.shape[2] != HEAD_DIM or out.shape != query.shape \
            or not (query.is_contiguous() and out.is_contiguous()):
        raise ValueError(f"{who}: query and out must be contiguous [tokens, heads, {HEAD_DIM}], got "
                         f"{tuple(query.shape)} and {tuple(out.shape)}")
    nb, bs, kvh = _check_pool(who, kv_cache)
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.stride(1) != 1:
        raise ValueError(f"{who}: block_tables must be int32 [batch, max_blocks] with unit column stride")
    if lens.dtype != torch.int32 or lens.numel() != block_tables.shape[0] or not lens.is_contiguous():
        raise ValueError(f"{who}: the sequences' lengths must be a contiguous int32 [batch] device tensor")
    return nb, bs, kvh, block_tables.shape[0]


def paged_decode_fp4(out: torch.Tensor, query: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, scale: float, workspace: torch.Tensor, num_ctas: int = 0,
                     k_scale: float = 1.0, v_scale: float = 1.0) -> torch.Tensor:
    """Paged GQA decode attention over a 4-bit pool into ``out`` ([batch, heads, 128] bf16).

    1 to 8 query heads per KV head. ``workspace`` (uint8, zeroed once) must
    hold decode_fp4_workspace_bytes(heads, kv_heads); calls sharing it must be
    ordered on one stream. Its first int32 is the device error word.
    """
    who = "paged_decode_fp4"
    nb, bs, kvh, batch = _check_attention(who, out, query, kv_cache, block_tables, context_lens)
    dev = query.device
    _require_cuda("workspace", workspace, dev)
    if query.shape[0] != batch or not workspace.is_contiguous():
        raise ValueError(f"{who}: {query.shape[0]} queries for {batch} sequences, or a strided workspace")
    _call(dev, "nvk_fp4_paged_decode", out.data_ptr(), query.data_ptr(), kv_cache.data_ptr(), nb, bs,
          block_tables.data_ptr(), _table_stride(block_tables), block_tables.shape[1],
          context_lens.data_ptr(), batch, query.shape[1], kvh, HEAD_DIM, scale, k_scale, v_scale, num_ctas,
          workspace.data_ptr(), workspace.numel() * workspace.element_size())
    return out


def paged_prefill_fp4(out: torch.Tensor, query: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                      cu_seqlens_q: torch.Tensor, kv_lens: torch.Tensor, max_q_len: int, scale: float,
                      k_scale: float = 1.0, v_scale: float = 1.0,
                      error_word: torch.Tensor | None = None) -> torch.Tensor:
    """Causal (bottom-right) prefill attention over a 4-bit pool into ``out``."""
    who = "paged_prefill_fp4"
    nb, bs, kvh, batch = _check_attention(who, out, query, kv_cache, block_tables, kv_lens)
    dev = query.device
    _require_cuda("cu_seqlens_q", cu_seqlens_q, dev)
    cu = _check_index(who, "cu_seqlens_q", cu_seqlens_q, torch.int32, batch + 1)
    _call(dev, "nvk_fp4_paged_prefill", out.data_ptr(), query.data_ptr(), kv_cache.data_ptr(), nb, bs,
          block_tables.data_ptr(), _table_stride(block_tables), block_tables.shape[1],
          cu.data_ptr(), kv_lens.data_ptr(), batch, query.shape[0], max_q_len, query.shape[1], kvh, HEAD_DIM, scale,
          k_scale, v_scale, _error_ptr(who, error_word, dev))
    return out
