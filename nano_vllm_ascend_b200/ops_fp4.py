"""Tensor-level wrappers over the kernels of the 4-bit KV pool.

As in ``ops``, each function validates devices, dtypes, shapes and strides,
then calls the matching ``nvk_fp4_*`` entry point (include/nvk_paged_kv.h) on
the tensors' current CUDA stream, and there is no non-CUDA path. Calls whose
arguments need no repair go through ``csrc/fp4_calls.cpp``, which makes the
same checks in a third of the time; what it does not take, the code here checks
again, calls or refuses.

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
import functools

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


# A decode step makes a few of these calls a layer, so the checks are written
# to cost little: tensors' properties are read once, torch's raw stream handle
# is asked for instead of a Stream object (3 us less a call), and entry points
# are looked up once.
_raw_stream = torch._C._cuda_getCurrentRawStream
_NOT_TAKEN = 1
_BOUND = ("nvk_fp4_append", "nvk_fp4_read", "nvk_fp4_qk_norm_rope_append", "nvk_fp4_paged_decode_reporting",
          "nvk_fp4_paged_prefill")


class _EntryPoints(dict):
    def __missing__(self, name: str):
        lib = _lib.load()
        calls = _binding()
        if calls is not None:  # from the first call on
            calls.bind(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _BOUND))
        fn = self[name] = getattr(lib, name)
        return fn


_entry_points = _EntryPoints()


def _leave(*args) -> int:
    return _NOT_TAKEN


@functools.cache
def _binding():
    """The compiled binding, loaded with the first call (importing the package maps no native code); None where it is
    not built, or for another torch: then every call is checked and made here."""
    try:
        from . import _fp4_calls as calls
    except ImportError:
        return None
    return calls if torch.__version__.startswith(calls.TORCH_VERSION) else None


def __getattr__(name: str):
    if name == "_calls":
        return _binding()
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def _first(name: str):
    """Stands for the binding's function until its first call, which puts that in its place."""
    def call(*args):
        calls = _binding()
        fn = _leave if calls is None else getattr(calls, name)
        if globals()[f"_{name}"] is call:
            globals()[f"_{name}"] = fn
        return fn(*args)
    return call


_append, _read, _norm_rope_append, _decode, _prefill = map(
    _first, ("append", "read", "norm_rope_append", "decode", "prefill"))


def _call(dev: torch.device, name: str, *args) -> None:
    """Calls ``name`` on ``dev`` and its current stream (the last argument)."""
    index = dev.index
    if index == torch.cuda.current_device():
        rc = _entry_points[name](*args, _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            rc = _entry_points[name](*args, _raw_stream(index))
    if rc:
        _lib.check(name, rc)


def _wrong_device(dev: torch.device, **tensors: torch.Tensor) -> None:
    """Raises for the first tensor that is not on the CUDA device ``dev``."""
    for name, t in tensors.items():
        _require_cuda(name, t, dev)


def _check_pool(who: str, kv_cache: torch.Tensor) -> tuple[int, int, int]:
    """(blocks, block size, KV heads) of a layer's pool."""
    shape = kv_cache.shape
    if kv_cache.dtype != torch.uint8 or len(shape) != 4 or shape[3] != _lib.FP4_UNIT_BYTES \
            or not kv_cache.is_contiguous():
        raise ValueError(f"{who}: kv_cache must be contiguous uint8 [blocks, kv_heads, block_size / 16, "
                         f"{_lib.FP4_UNIT_BYTES}], got {kv_cache.dtype} {tuple(shape)}")
    return shape[0], shape[2] * _lib.FP4_UNIT_TOKENS, shape[1]


def _row_stride(name: str, t: torch.Tensor) -> int:
    """The token stride of rows [tokens, heads, 128] whose heads and dims are packed."""
    stride = t.stride()
    if len(stride) != 3 or stride[2] != 1 or stride[1] != HEAD_DIM or t.shape[2] != HEAD_DIM:
        _require_rows(name, t)
        raise ValueError(f"{name} must have {HEAD_DIM} dims a head, got shape {tuple(t.shape)} stride {stride}")
    return stride[0]


def _check_index(who: str, name: str, t: torch.Tensor, dtype: torch.dtype, count: int) -> torch.Tensor:
    if t.dtype != dtype or t.numel() != count:
        raise ValueError(f"{who}: {name} must be {dtype} with {count} entries, got {t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _error_ptr(who: str, error_word: torch.Tensor | None, dev: torch.device) -> int:
    if error_word is None:
        return 0
    if error_word.device != dev or error_word.dtype != torch.int32 or error_word.numel() < 1:
        raise ValueError(f"{who}: error_word must be an int32 on {dev}")
    return error_word.data_ptr()


def kv_append_fp4(kv_cache: torch.Tensor, key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor,
                  k_scale: float = 1.0, v_scale: float = 1.0, error_word: torch.Tensor | None = None) -> None:
    """Quantises the rows ``key`` / ``value`` ([tokens, kv_heads, 128], bf16 or
    fp16; the token stride may be larger) into the pool at ``slot_mapping``
    (int64). Slots must differ; one outside the pool is skipped and sets bit 4
    of ``error_word``."""
    rc = _append(kv_cache, key, value, slot_mapping, k_scale, v_scale, error_word)
    if rc == 0:
        return
    if rc != _NOT_TAKEN:
        _lib.check("nvk_fp4_append", rc)
    who = "kv_append_fp4"
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
    _call(dev, "nvk_fp4_append", key.data_ptr(), value.data_ptr(), k_stride, v_stride, kv_cache.data_ptr(),
          slots.data_ptr(), tokens, nb, bs, kvh, HEAD_DIM, _DTYPES[dtype], k_scale, v_scale,
          _error_ptr(who, error_word, dev))


def kv_read_fp4(kv_cache: torch.Tensor, slot_mapping: torch.Tensor, k_scale: float = 1.0, v_scale: float = 1.0,
                dtype: torch.dtype = _BF16, key_out: torch.Tensor | None = None,
                value_out: torch.Tensor | None = None,
                error_word: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows [tokens, kv_heads, 128] that the pool holds at
    ``slot_mapping`` (int64; any order, repeats allowed), as ``dtype``; a slot
    outside the pool gives zeros and sets bit 4 of ``error_word``."""
    if key_out is None and value_out is None and dtype in _DTYPES:
        rows = _read(kv_cache, slot_mapping, k_scale, v_scale, dtype is torch.float16, error_word)
        if rows.__class__ is tuple:
            return rows
        if rows != _NOT_TAKEN:
            _lib.check("nvk_fp4_read", rows)
    who = "kv_read_fp4"
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
    _call(dev, "nvk_fp4_read", key_out.data_ptr(), value_out.data_ptr(), kv_cache.data_ptr(), slots.data_ptr(),
          tokens, nb, bs, kvh, HEAD_DIM, _DTYPES[dtype], k_scale, v_scale, _error_ptr(who, error_word, dev))
    return key_out, value_out


def qk_norm_rope_append_fp4(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, q_weight: torch.Tensor,
                            k_weight: torch.Tensor, eps: float, cos_table: torch.Tensor, sin_table: torch.Tensor,
                            positions: torch.Tensor, kv_cache: torch.Tensor, slot_mapping: torch.Tensor,
                            k_scale: float = 1.0, v_scale: float = 1.0, query_out: torch.Tensor | None = None,
                            error_word: torch.Tensor | None = None) -> torch.Tensor:
    """``ops.qk_norm_rope_append`` into a 4-bit pool: per-head RMSNorm of q and
    k, rotary embedding, and the append of the rotated k and of v, in one
    kernel. Returns the rotated query [tokens, heads, 128]."""
    rotated = _norm_rope_append(query, key, value, q_weight, k_weight, eps, cos_table, sin_table, positions, kv_cache,
                                slot_mapping, k_scale, v_scale, query_out, error_word)
    if rotated.__class__ is not int:
        return rotated
    if rotated != _NOT_TAKEN:
        _lib.check("nvk_fp4_qk_norm_rope_append", rotated)
    who = "qk_norm_rope_append_fp4"
    dev = query.device
    if not query.is_cuda or key.device != dev or value.device != dev or q_weight.device != dev \
            or k_weight.device != dev or cos_table.device != dev or sin_table.device != dev \
            or positions.device != dev or kv_cache.device != dev or slot_mapping.device != dev:
        _wrong_device(dev, query=query, key=key, value=value, q_weight=q_weight, k_weight=k_weight,
                      cos_table=cos_table, sin_table=sin_table, positions=positions, kv_cache=kv_cache,
                      slot_mapping=slot_mapping)
    if query.dtype != _BF16 or key.dtype != _BF16 or value.dtype != _BF16:
        raise ValueError(f"{who}: query, key and value must be bfloat16")
    q_stride, k_stride, v_stride = _row_stride("query", query), _row_stride("key", key), _row_stride("value", value)
    tokens, num_heads, _ = query.shape
    nb, bs, kvh = _check_pool(who, kv_cache)
    shape = key.shape
    if shape[0] != tokens or shape[1] != kvh or value.shape != shape:
        raise ValueError(f"kv shape mismatch: got {tuple(shape)} / {tuple(value.shape)}")
    for t in (q_weight, k_weight):
        if t.numel() != HEAD_DIM or t.dtype != _BF16 or not t.is_contiguous():
            raise ValueError(f"{who}: q_weight/k_weight must be contiguous bfloat16 [head_dim]")
    table = cos_table.shape
    if cos_table.dtype != torch.float32 or sin_table.dtype != torch.float32 or len(table) != 2 \
            or table[1] != HEAD_DIM or sin_table.shape != table \
            or not (cos_table.is_contiguous() and sin_table.is_contiguous()):
        raise ValueError(f"{who}: cos/sin tables must be contiguous float32 [max_position, head_dim]")
    pos = _check_index(who, "positions", positions, torch.int64, tokens)
    slots = _check_index(who, "slot_mapping", slot_mapping, torch.int64, tokens)
    if query_out is None:
        query_out = torch.empty((tokens, num_heads, HEAD_DIM), dtype=_BF16, device=dev)
    elif query_out.device != dev or query_out.shape != query.shape or not query_out.is_contiguous() \
            or query_out.dtype != _BF16:
        raise ValueError(f"{who}: query_out must be a contiguous bf16 [tokens, heads, head_dim] on {dev}")
    _call(dev, "nvk_fp4_qk_norm_rope_append", query.data_ptr(), key.data_ptr(), value.data_ptr(), q_stride, k_stride,
          v_stride, q_weight.data_ptr(), k_weight.data_ptr(), eps, cos_table.data_ptr(), sin_table.data_ptr(),
          table[0], pos.data_ptr(), query_out.data_ptr(), kv_cache.data_ptr(), slots.data_ptr(), tokens, nb, bs,
          num_heads, kvh, HEAD_DIM, k_scale, v_scale, _error_ptr(who, error_word, dev))
    return query_out


def decode_fp4_workspace_bytes(num_heads: int, num_kv_heads: int, head_dim: int = HEAD_DIM, num_ctas: int = 0) -> int:
    """Workspace bytes of paged_decode_fp4 for any batch (num_ctas 0 = one CTA per SM of the current device)."""
    out = ctypes.c_size_t(0)
    _lib.call("nvk_fp4_paged_decode_workspace_size", num_heads, num_kv_heads, head_dim, num_ctas, ctypes.byref(out))
    return int(out.value)


def _check_attention(who: str, dev, out, query, kv_cache, block_tables, lens) -> tuple:
    """Checks what decode and prefill share; returns what their calls take: query's shape, the pool's blocks,
    block size and KV heads, and the table's rows, row stride and columns."""
    if not query.is_cuda or out.device != dev or kv_cache.device != dev or block_tables.device != dev \
            or lens.device != dev:
        _wrong_device(dev, out=out, query=query, kv_cache=kv_cache, block_tables=block_tables, lens=lens)
    if query.dtype != _BF16 or out.dtype != _BF16:
        raise ValueError(f"{who}: query and out must be bfloat16")
    shape = query.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM or out.shape != shape \
            or not (query.is_contiguous() and out.is_contiguous()):
        raise ValueError(f"{who}: query and out must be contiguous [tokens, heads, {HEAD_DIM}], got "
                         f"{tuple(shape)} and {tuple(out.shape)}")
    nb, bs, kvh = _check_pool(who, kv_cache)
    stride = block_tables.stride()
    if block_tables.dtype != torch.int32 or len(stride) != 2 or stride[1] != 1:
        raise ValueError(f"{who}: block_tables must be int32 [batch, max_blocks] with unit column stride")
    batch, width = block_tables.shape
    if lens.dtype != torch.int32 or lens.numel() != batch or not lens.is_contiguous():
        raise ValueError(f"{who}: the sequences' lengths must be a contiguous int32 [batch] device tensor")
    # a single row's stride may be anything
    return shape, nb, bs, kvh, batch, stride[0] if batch > 1 else width, width


def paged_decode_fp4(out: torch.Tensor, query: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, scale: float, workspace: torch.Tensor, num_ctas: int = 0,
                     k_scale: float = 1.0, v_scale: float = 1.0,
                     error_word: torch.Tensor | None = None) -> torch.Tensor:
    """Paged GQA decode attention over a 4-bit pool into ``out`` ([batch, heads, 128] bf16).

    1 to 8 query heads per KV head. ``workspace`` (uint8, zeroed once) must
    hold decode_fp4_workspace_bytes(heads, kv_heads); calls sharing it must be
    ordered on one stream. Device errors are bits of ``error_word``, or of the
    workspace's first int32.
    """
    rc = _decode(out, query, kv_cache, block_tables, context_lens, scale, workspace, num_ctas, k_scale, v_scale,
                 error_word)
    if rc == 0:
        return out
    if rc != _NOT_TAKEN:
        _lib.check("nvk_fp4_paged_decode_reporting", rc)
    who = "paged_decode_fp4"
    dev = query.device
    shape, nb, bs, kvh, batch, stride, width = _check_attention(who, dev, out, query, kv_cache, block_tables,
                                                                context_lens)
    if workspace.device != dev:
        _wrong_device(dev, workspace=workspace)
    if shape[0] != batch or not workspace.is_contiguous():
        raise ValueError(f"{who}: {shape[0]} queries for {batch} sequences, or a strided workspace")
    _call(dev, "nvk_fp4_paged_decode_reporting", out.data_ptr(), query.data_ptr(), kv_cache.data_ptr(), nb, bs,
          block_tables.data_ptr(), stride, width, context_lens.data_ptr(), batch, shape[1], kvh, HEAD_DIM, scale,
          k_scale, v_scale, num_ctas, workspace.data_ptr(), workspace.nbytes, _error_ptr(who, error_word, dev))
    return out


def paged_prefill_fp4(out: torch.Tensor, query: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                      cu_seqlens_q: torch.Tensor, kv_lens: torch.Tensor, max_q_len: int, scale: float,
                      k_scale: float = 1.0, v_scale: float = 1.0,
                      error_word: torch.Tensor | None = None) -> torch.Tensor:
    """Causal (bottom-right) prefill attention over a 4-bit pool into ``out``."""
    rc = _prefill(out, query, kv_cache, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale, k_scale, v_scale,
                  error_word)
    if rc == 0:
        return out
    if rc != _NOT_TAKEN:
        _lib.check("nvk_fp4_paged_prefill", rc)
    who = "paged_prefill_fp4"
    dev = query.device
    shape, nb, bs, kvh, batch, stride, width = _check_attention(who, dev, out, query, kv_cache, block_tables, kv_lens)
    if cu_seqlens_q.device != dev:
        _wrong_device(dev, cu_seqlens_q=cu_seqlens_q)
    cu = _check_index(who, "cu_seqlens_q", cu_seqlens_q, torch.int32, batch + 1)
    _call(dev, "nvk_fp4_paged_prefill", out.data_ptr(), query.data_ptr(), kv_cache.data_ptr(), nb, bs,
          block_tables.data_ptr(), stride, width, cu.data_ptr(), kv_lens.data_ptr(), batch, shape[0], max_q_len,
          shape[1], kvh, HEAD_DIM, scale, k_scale, v_scale, _error_ptr(who, error_word, dev))
    return out
