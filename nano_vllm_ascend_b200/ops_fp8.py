"""Tensor-level wrappers over the kernels of the 8-bit KV pool.

As in ``ops`` and ``ops_fp4``, each function validates devices, dtypes, shapes
and strides, then calls the matching ``nvk_fp8_*`` entry point
(include/nvk_paged_kv.h) on the tensors' current CUDA stream, and there is no
non-CUDA path.

``kv_cache`` is ONE layer of the pool, K and V together: contiguous uint8
[num_blocks, kv_heads, block_size / 16, 4128] (``pool_shape``), zero-filled
once when it is allocated. 16 tokens of a block's KV head make a unit with an
exponent for K and one for V; a value is an e4m3 code times 2^exponent, exact in
bf16. Slots, block tables and lengths are those of the bf16 pool.
"""

from __future__ import annotations

import ctypes

import torch

from . import _calls, _lib
from .ops_fp4 import (_BF16, _DTYPES, HEAD_DIM, _check_index, _check_sequences, _error_ptr, _row_stride, _wrong_device,
                      call_on)

_append8, _read8, _decode8, _prefill8 = (_calls.first(name, globals()) for name in
                                         ("append8", "read8", "decode8", "prefill8"))
SCAN_TOKENS = 512  # up to here an append needs no workspace


def pool_shape(num_blocks: int, block_size: int, num_kv_heads: int) -> tuple[int, int, int, int]:
    """The shape of one layer's uint8 pool."""
    if block_size not in (16, 32, 64, 128, 256):
        raise ValueError(f"block_size {block_size} unsupported (a power of two in [16, 256])")
    return num_blocks, num_kv_heads, block_size // _lib.FP8_UNIT_TOKENS, _lib.FP8_UNIT_BYTES


def _check_pool(who: str, kv_cache: torch.Tensor) -> tuple[int, int, int]:
    """(blocks, block size, KV heads) of a layer's pool."""
    shape = kv_cache.shape
    if kv_cache.dtype != torch.uint8 or len(shape) != 4 or shape[3] != _lib.FP8_UNIT_BYTES \
            or not kv_cache.is_contiguous():
        raise ValueError(f"{who}: kv_cache must be contiguous uint8 [blocks, kv_heads, block_size / 16, "
                         f"{_lib.FP8_UNIT_BYTES}], got {kv_cache.dtype} {tuple(shape)}")
    return shape[0], shape[2] * _lib.FP8_UNIT_TOKENS, shape[1]


def kv_append_fp8(kv_cache: torch.Tensor, key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor,
                  error_word: torch.Tensor | None = None) -> None:
    """Quantises the rows ``key`` / ``value`` ([tokens, kv_heads, 128], bf16 or
    fp16; the token stride may be larger) into the pool at ``slot_mapping``
    (int64). Slots must differ; one outside the pool is skipped and sets bit 4
    of ``error_word``. Writing a unit's first token starts the unit anew (its
    other rows become zeros), so a sequence's tokens are appended in order."""
    rc = _append8(kv_cache, key, value, slot_mapping, error_word)
    if rc == 0:
        return
    if rc != _calls.NOT_TAKEN:
        _lib.check("nvk_fp8_append", rc)
    who = "kv_append_fp8"
    dev = kv_cache.device
    if not kv_cache.is_cuda or key.device != dev or value.device != dev or slot_mapping.device != dev:
        _wrong_device(dev, kv_cache=kv_cache, key=key, value=value, slot_mapping=slot_mapping)
    nb, bs, kvh = _check_pool(who, kv_cache)
    dtype, shape = key.dtype, key.shape
    if dtype not in _DTYPES or value.dtype != dtype:
        raise ValueError(f"{who}: key and value must both be bfloat16 or float16, got {dtype} and {value.dtype}")
    k_stride, v_stride = _row_stride("key", key), _row_stride("value", value)
    tokens = shape[0]
    if value.shape != shape or shape[1] != kvh:
        raise ValueError(f"kv shape mismatch: got {tuple(shape)} / {tuple(value.shape)}")
    slots = _check_index(who, "slot_mapping", slot_mapping, torch.int64, tokens)
    # which token writes which slot, for longer calls: of this call alone, so from the allocator
    ws = torch.empty(nb * bs, dtype=torch.int32, device=dev) if tokens > SCAN_TOKENS else None
    call_on(dev, "nvk_fp8_append", key.data_ptr(), value.data_ptr(), k_stride, v_stride, kv_cache.data_ptr(),
            slots.data_ptr(), tokens, nb, bs, kvh, HEAD_DIM, _DTYPES[dtype], 0 if ws is None else ws.data_ptr(),
            0 if ws is None else ws.nbytes, _error_ptr(who, error_word, dev))


def kv_read_fp8(kv_cache: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype = _BF16,
                key_out: torch.Tensor | None = None, value_out: torch.Tensor | None = None,
                error_word: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows [tokens, kv_heads, 128] that the pool holds at
    ``slot_mapping`` (int64; any order, repeats allowed), as ``dtype``; a slot
    outside the pool gives zeros and sets bit 4 of ``error_word``."""
    if key_out is None and value_out is None and dtype in _DTYPES:
        rows = _read8(kv_cache, slot_mapping, dtype is torch.float16, error_word)
        if rows.__class__ is tuple:
            return rows
        if rows != _calls.NOT_TAKEN:
            _lib.check("nvk_fp8_read", rows)
    who = "kv_read_fp8"
    dev = kv_cache.device
    if not kv_cache.is_cuda or slot_mapping.device != dev:
        _wrong_device(dev, kv_cache=kv_cache, slot_mapping=slot_mapping)
    nb, bs, kvh = _check_pool(who, kv_cache)
    if dtype not in _DTYPES:
        raise ValueError(f"{who}: dtype must be bfloat16 or float16, got {dtype}")
    tokens = slot_mapping.numel()
    slots = _check_index(who, "slot_mapping", slot_mapping, torch.int64, tokens)
    for name, t in (("key_out", key_out), ("value_out", value_out)):
        if t is not None and (t.device != dev or t.shape != (tokens, kvh, HEAD_DIM) or t.dtype != dtype
                              or not t.is_contiguous()):
            raise ValueError(f"{who}: {name} must be contiguous {dtype} [tokens, kv_heads, {HEAD_DIM}] on {dev}")
    if key_out is None:
        key_out = torch.empty((tokens, kvh, HEAD_DIM), dtype=dtype, device=dev)
    if value_out is None:
        value_out = torch.empty((tokens, kvh, HEAD_DIM), dtype=dtype, device=dev)
    call_on(dev, "nvk_fp8_read", key_out.data_ptr(), value_out.data_ptr(), kv_cache.data_ptr(), slots.data_ptr(),
            tokens, nb, bs, kvh, HEAD_DIM, _DTYPES[dtype], _error_ptr(who, error_word, dev))
    return key_out, value_out


def decode_fp8_workspace_bytes(num_heads: int, num_kv_heads: int, head_dim: int = HEAD_DIM, num_ctas: int = 0) -> int:
    """Workspace bytes of paged_decode_fp8 for any batch (num_ctas 0 = one CTA per SM of the current device)."""
    out = ctypes.c_size_t(0)
    _lib.call("nvk_fp8_paged_decode_workspace_size", num_heads, num_kv_heads, head_dim, num_ctas, ctypes.byref(out))
    return int(out.value)


def paged_decode_fp8(out: torch.Tensor, query: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, scale: float, workspace: torch.Tensor, num_ctas: int = 0,
                     error_word: torch.Tensor | None = None) -> torch.Tensor:
    """Paged GQA decode attention over an 8-bit pool into ``out`` ([batch, heads, 128] bf16).

    1 to 8 query heads per KV head. ``workspace`` (uint8, zeroed once) must
    hold decode_fp8_workspace_bytes(heads, kv_heads); calls sharing it must be
    ordered on one stream. Device errors are bits of ``error_word``, or of the
    workspace's first int32.
    """
    rc = _decode8(out, query, kv_cache, block_tables, context_lens, scale, workspace, num_ctas, error_word)
    if rc == 0:
        return out
    if rc != _calls.NOT_TAKEN:
        _lib.check("nvk_fp8_paged_decode", rc)
    who = "paged_decode_fp8"
    dev = query.device
    shape, batch, stride, width = _check_sequences(who, dev, out, query, kv_cache, block_tables, context_lens)
    nb, bs, kvh = _check_pool(who, kv_cache)
    if workspace.device != dev:
        _wrong_device(dev, workspace=workspace)
    if shape[0] != batch or not workspace.is_contiguous():
        raise ValueError(f"{who}: {shape[0]} queries for {batch} sequences, or a strided workspace")
    call_on(dev, "nvk_fp8_paged_decode", out.data_ptr(), query.data_ptr(), kv_cache.data_ptr(), nb, bs,
            block_tables.data_ptr(), stride, width, context_lens.data_ptr(), batch, shape[1], kvh, HEAD_DIM, scale,
            num_ctas, workspace.data_ptr(), workspace.nbytes, _error_ptr(who, error_word, dev))
    return out


def paged_prefill_fp8(out: torch.Tensor, query: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                      cu_seqlens_q: torch.Tensor, kv_lens: torch.Tensor, max_q_len: int, scale: float,
                      error_word: torch.Tensor | None = None) -> torch.Tensor:
    """Causal (bottom-right) prefill attention over an 8-bit pool into ``out``."""
    rc = _prefill8(out, query, kv_cache, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale, error_word)
    if rc == 0:
        return out
    if rc != _calls.NOT_TAKEN:
        _lib.check("nvk_fp8_paged_prefill", rc)
    who = "paged_prefill_fp8"
    dev = query.device
    shape, batch, stride, width = _check_sequences(who, dev, out, query, kv_cache, block_tables, kv_lens)
    nb, bs, kvh = _check_pool(who, kv_cache)
    if cu_seqlens_q.device != dev:
        _wrong_device(dev, cu_seqlens_q=cu_seqlens_q)
    cu = _check_index(who, "cu_seqlens_q", cu_seqlens_q, torch.int32, batch + 1)
    call_on(dev, "nvk_fp8_paged_prefill", out.data_ptr(), query.data_ptr(), kv_cache.data_ptr(), nb, bs,
            block_tables.data_ptr(), stride, width, cu.data_ptr(), kv_lens.data_ptr(), batch, shape[0], max_q_len,
            shape[1], kvh, HEAD_DIM, scale, _error_ptr(who, error_word, dev))
    return out
