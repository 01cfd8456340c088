"""The 8-bit KV cache where no GPU is needed: what the C entry points and the
tensor wrappers refuse (before any CUDA call), the pool class's checks and its
sizing, and what the oracle's units hold."""

import ctypes
import re

import numpy as np
import pytest
import torch

from nano_vllm_ascend_b200 import NpuPagedAttention, PagedKVCacheFp4, PagedKVCacheFp8, _lib, ops_fp8
from nano_vllm_ascend_b200.pool import bytes_per_block, fp8_bytes_per_block, num_blocks_for_budget
from oracle import fp8_oracle as orc

INVALID, UNSUPPORTED, WORKSPACE = _lib.NVK_ERR_INVALID_ARGUMENT, _lib.NVK_ERR_UNSUPPORTED, _lib.NVK_ERR_WORKSPACE
P = 1 << 20  # a pointer that is never followed: every call here is refused or empty


def refused(name, args, code, text):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == code, lib.nvk_last_error()
    assert text in lib.nvk_last_error().decode()


def append_args(**kw):
    a = dict(key=P, value=P, ks=1024, vs=1024, pool=P, slots=P, tokens=4, nb=8, bs=128, kvh=8, d=128, dtype=0, ws=0,
             bytes=0, err=0, stream=0)
    a.update(kw)
    return list(a.values())


BAD_POOL = [(dict(d=64), UNSUPPORTED, "head_dim"), (dict(bs=96), UNSUPPORTED, "block_size"),
            (dict(bs=8), UNSUPPORTED, "block_size"), (dict(bs=512), UNSUPPORTED, "block_size"),
            (dict(nb=0), INVALID, "bad pool"), (dict(kvh=0), INVALID, "bad pool"), (dict(kvh=-1), INVALID, "bad pool"),
            (dict(pool=0), INVALID, "null"), (dict(pool=P + 8), INVALID, "aligned")]


@pytest.mark.parametrize("kw,code,text", BAD_POOL + [
    (dict(tokens=-1), INVALID, "tokens"), (dict(dtype=2), UNSUPPORTED, "dtype"), (dict(key=0), INVALID, "null"),
    (dict(value=0), INVALID, "null"), (dict(slots=0), INVALID, "null"), (dict(slots=P + 4), INVALID, "aligned"),
    (dict(key=P + 1), INVALID, "aligned"), (dict(ks=1023), INVALID, "strides"), (dict(vs=0), INVALID, "strides"),
    (dict(tokens=513), WORKSPACE, "workspace"), (dict(tokens=513, ws=P, bytes=8 * 128 * 4 - 1), WORKSPACE, "workspace"),
    (dict(tokens=513, ws=P + 2, bytes=8 * 128 * 4), INVALID, "aligned"),
    (dict(tokens=1 << 31, ws=P, bytes=8 * 128 * 4), UNSUPPORTED, "range")])
def test_append_refuses(kw, code, text):
    refused("nvk_fp8_append", append_args(**kw), code, text)


@pytest.mark.parametrize("kw,code,text", BAD_POOL + [
    (dict(tokens=-1), INVALID, "tokens"), (dict(dtype=2), UNSUPPORTED, "dtype"), (dict(key=0), INVALID, "null"),
    (dict(value=P + 8), INVALID, "aligned"), (dict(slots=P + 4), INVALID, "aligned")])
def test_read_refuses(kw, code, text):
    a = dict(key=P, value=P, pool=P, slots=P, tokens=4, nb=8, bs=128, kvh=8, d=128, dtype=0, err=0, stream=0)
    refused("nvk_fp8_read", list({**a, **kw}.values()), code, text)


def test_empty_calls_are_no_ops():
    lib = _lib.load()
    assert lib.nvk_fp8_append(*append_args(tokens=0, key=0, slots=0)) == _lib.NVK_OK
    assert lib.nvk_fp8_read(0, 0, P, 0, 0, 8, 128, 8, 128, 0, 0, 0) == _lib.NVK_OK
    assert lib.nvk_fp8_paged_decode(*decode_args(batch=0)) == _lib.NVK_OK
    assert lib.nvk_fp8_paged_prefill(*prefill_args(batch=0)) == _lib.NVK_OK


def test_append_workspace_size():
    lib, sz = _lib.load(), ctypes.c_size_t()
    for tokens, slots, want in ((0, 100, 0), (512, 100, 0), (513, 100, 400), (1 << 20, 1 << 33, 4 << 33)):
        assert lib.nvk_fp8_append_workspace_size(tokens, slots, ctypes.byref(sz)) == 0 and sz.value == want
    assert ops_fp8.SCAN_TOKENS == 512
    for args in ((-1, 1, ctypes.byref(sz)), (1, -1, ctypes.byref(sz)), (1, 1, None)):
        assert lib.nvk_fp8_append_workspace_size(*args) == INVALID


def decode_args(**kw):
    a = dict(out=P, q=P, pool=P, nb=8, bs=128, tables=P, stride=4, width=4, ctx=P, batch=2, h=16, kvh=8, d=128,
             scale=0.1, ctas=148, ws=P, bytes=1 << 30, err=0, stream=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code,text", BAD_POOL[:4] + BAD_POOL[7:] + [
    (dict(nb=0), INVALID, "bad pool"), (dict(kvh=0), INVALID, "bad sizes"),
    (dict(batch=-1), INVALID, "batch"), (dict(h=0), INVALID, "bad sizes"), (dict(ctas=-1), INVALID, "bad sizes"),
    (dict(h=12), UNSUPPORTED, "group"), (dict(h=72), UNSUPPORTED, "group"), (dict(scale=0.0), INVALID, "positive"),
    (dict(scale=-1.0), INVALID, "positive"), (dict(scale=float("nan")), INVALID, "positive"),
    (dict(width=0), INVALID, "stride"), (dict(stride=3), INVALID, "stride"), (dict(ws=0), INVALID, "null"),
    (dict(ctx=0), INVALID, "null"), (dict(q=P + 2), INVALID, "aligned"), (dict(ws=P + 8), INVALID, "aligned"),
    (dict(width=1 << 24, stride=1 << 24), UNSUPPORTED, "range"), (dict(bytes=1000), WORKSPACE, "workspace")])
def test_decode_refuses(kw, code, text):
    refused("nvk_fp8_paged_decode", decode_args(**kw), code, text)


def test_decode_workspace_is_that_of_the_4_bit_kernel():
    """PagedAttention keeps one workspace for both."""
    lib, a, b = _lib.load(), ctypes.c_size_t(), ctypes.c_size_t()
    for h, kvh, ctas in ((8, 8, 1), (8, 8, 148), (64, 8, 148), (6, 2, 600)):
        assert lib.nvk_fp8_paged_decode_workspace_size(h, kvh, 128, ctas, ctypes.byref(a)) == 0
        assert lib.nvk_fp4_paged_decode_workspace_size(h, kvh, 128, ctas, ctypes.byref(b)) == 0
        assert a.value == b.value
    assert _lib.FP8_DECODE_ZEROED_BYTES == _lib.FP4_DECODE_ZEROED_BYTES
    assert lib.nvk_fp8_paged_decode_workspace_size(8, 8, 64, 1, ctypes.byref(a)) == UNSUPPORTED
    assert lib.nvk_fp8_paged_decode_workspace_size(8, 8, 128, 1, None) == INVALID


def prefill_args(**kw):
    a = dict(out=P, q=P, pool=P, nb=8, bs=128, tables=P, stride=4, width=4, cu=P, lens=P, batch=2, total=8, max_q=8,
             h=16, kvh=8, d=128, scale=0.1, err=0, stream=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code,text", BAD_POOL + [
    (dict(batch=-1), INVALID, "bad sizes"), (dict(total=-1), INVALID, "bad sizes"), (dict(h=0), INVALID, "bad sizes"),
    (dict(h=12), INVALID, "multiple"), (dict(scale=0.0), INVALID, "positive"), (dict(stride=3), INVALID, "stride"),
    (dict(scale=float("nan")), INVALID, "positive"), (dict(cu=0), INVALID, "null"), (dict(lens=0), INVALID, "null"),
    (dict(out=P + 4), INVALID, "aligned"), (dict(batch=70000), UNSUPPORTED, "grid")])
def test_prefill_refuses(kw, code, text):
    refused("nvk_fp8_paged_prefill", prefill_args(**kw), code, text)


def test_wrappers_refuse_host_tensors_and_bad_shapes():
    pool = torch.zeros(ops_fp8.pool_shape(2, 16, 2), dtype=torch.uint8)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        ops_fp8.kv_append_fp8(pool, k, k, torch.arange(3))
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        ops_fp8.kv_read_fp8(pool, torch.arange(3))
    for bs in (8, 24, 512):
        with pytest.raises(ValueError, match=f"block_size {bs}"):
            ops_fp8.pool_shape(2, bs, 2)
    for wrong in (pool.transpose(0, 1), pool.view(torch.int8), pool[..., :2304], pool[0]):
        with pytest.raises(ValueError, match="kv_cache must be contiguous uint8"):
            ops_fp8._check_pool("x", wrong)


def test_cache_refuses_and_sizes():
    kv = PagedKVCacheFp8(2, 4, 16, 8, 128, "cpu")
    assert kv.kv_cache.shape == (2, 4, 8, 1, 4128) and kv.bytes_per_block == 2 * 8 * 4128
    key, value = kv.get_physical_cache(1)
    assert key is value and key.shape == (4, 16, 8, 128)
    bad = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=re.escape("kv shape mismatch: got (3, 4, 128)")):
        kv.write(0, bad, bad, torch.zeros(3, dtype=torch.long))
    k = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="slot_mapping numel 3 != total_tokens 2"):
        kv.write(0, k, k, torch.zeros(3, dtype=torch.long))
    with pytest.raises(IndexError, match="index 64 is out of bounds for dimension 0 with size 64"):
        kv.write(0, k, k, torch.tensor([3, 64]))
    with pytest.raises(IndexError, match="index -1 is out of bounds"):
        kv.read(0, torch.tensor([-1]))
    kv.write(0, k[:0], k[:0], torch.zeros(0, dtype=torch.long))
    with pytest.raises(ValueError, match="head_dim 64"):
        PagedKVCacheFp8(1, 4, 16, 8, 64, "cpu")
    with pytest.raises(ValueError, match="block_size"):
        PagedKVCacheFp8(1, 4, 24, 8, 128, "cpu")


def test_pool_sizing():
    small, large = fp8_bytes_per_block(28, 128, 8), bytes_per_block(28, 128, 8, 128)
    assert large / small == 512 / 258
    n = num_blocks_for_budget(100 << 30, 180 << 30, 0.8, 28, 128, 8, 128, block_bytes=small)
    assert n == (int((180 << 30) * 0.8) - (80 << 30)) // small


def test_attention_over_an_8_bit_layer_checks_like_the_bf16_one():
    kv = PagedKVCacheFp8(1, 4, 16, 8, 128, "cpu")
    key, value = kv.get_physical_cache(0)
    attn = NpuPagedAttention(16, 8, 128)
    with pytest.raises(ValueError, match=re.escape("query shape mismatch: got (2, 8, 128)")):
        attn(torch.zeros(2, 8, 128, dtype=torch.bfloat16), key, value, torch.zeros(2, 1, dtype=torch.int32),
             torch.ones(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="missing block: context length 33"):
        attn(torch.zeros(2, 16, 128, dtype=torch.bfloat16), key, value, torch.zeros(2, 2, dtype=torch.int32),
             torch.tensor([5, 33], dtype=torch.int32))
    other = PagedKVCacheFp8(2, 4, 16, 8, 128, "cpu").get_physical_cache(1)[0]
    fp4 = PagedKVCacheFp4(1, 4, 16, 8, 128, "cpu").get_physical_cache(0)[0]
    for wrong in (other, fp4, torch.zeros(4, 16, 8, 128, dtype=torch.bfloat16), None):
        with pytest.raises(ValueError, match="must be the same layer"):
            attn(torch.zeros(2, 16, 128, dtype=torch.bfloat16), key, wrong, torch.zeros(2, 2, dtype=torch.int32),
                 torch.tensor([5, 31], dtype=torch.int32))


@pytest.mark.parametrize("spread", [0, 5, 60])
def test_a_value_is_off_by_half_a_step_of_its_code_or_of_its_unit(spread):
    """e4m3's half step is 2^-4 of a value down to 2^-6 of the code's scale, and 2^-10 of a code below: with the
    exponent the least that holds the unit's largest (above 224 as a code), that is below 2^-17 of the largest."""
    g = np.random.default_rng(spread)
    pool = np.zeros(ops_fp8.pool_shape(3, 16, 2), dtype=np.uint8)
    k, v = g.standard_normal((2, 48, 2, 128)) * 2.0 ** g.uniform(-spread, 0, (2, 48, 2, 128))
    orc.append(pool, k, v, np.arange(48))
    for got, want in zip(orc.rows(pool), (k, v)):
        amax = np.abs(want.reshape(3, 16, 2, 128)).max((1, 3), keepdims=True).repeat(16, 1).reshape(48, 2, 1)
        assert (np.abs(got.reshape(48, 2, 128) - want) <= np.maximum(np.abs(want) * 2.0 ** -4, amax * 2.0 ** -17)).all()
