"""The 4-bit KV cache where no GPU is needed: what the C entry points and the
tensor wrappers refuse (before any CUDA call), the pool class's checks, its
sizing, and the decode graph's workspaces by kind."""

import ctypes
import re

import numpy as np
import pytest
import torch

from nano_vllm_ascend_b200 import NpuPagedAttention, PagedKVCacheFp4, _lib, ops_fp4
from nano_vllm_ascend_b200.cuda_graph import GraphSlot
from nano_vllm_ascend_b200.pool import bytes_per_block, fp4_bytes_per_block, num_blocks_for_budget
from oracle import fp4_oracle as orc

INVALID, UNSUPPORTED, WORKSPACE = _lib.NVK_ERR_INVALID_ARGUMENT, _lib.NVK_ERR_UNSUPPORTED, _lib.NVK_ERR_WORKSPACE
P = 1 << 20  # a pointer that is never followed: every call here is refused or empty


def refused(name, args, code, text):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == code, lib.nvk_last_error()
    assert text in lib.nvk_last_error().decode()


def append_args(**kw):
    a = dict(key=P, value=P, ks=1024, vs=1024, pool=P, slots=P, tokens=4, nb=8, bs=128, kvh=8, d=128, dtype=0, kc=1.0,
             vc=1.0, err=0, stream=0)
    a.update(kw)
    return list(a.values())


BAD_POOL = [(dict(d=64), UNSUPPORTED, "head_dim"), (dict(bs=96), UNSUPPORTED, "block_size"),
            (dict(bs=8), UNSUPPORTED, "block_size"), (dict(bs=512), UNSUPPORTED, "block_size"),
            (dict(nb=0), INVALID, "bad pool"), (dict(kvh=0), INVALID, "bad pool"), (dict(kvh=-1), INVALID, "bad pool"),
            (dict(pool=0), INVALID, "null"), (dict(pool=P + 8), INVALID, "aligned"),
            (dict(kc=3.0), INVALID, "powers of two"), (dict(vc=0.0), INVALID, "powers of two"),
            (dict(vc=-2.0), INVALID, "powers of two"), (dict(kc=2.0 ** 61), INVALID, "powers of two"),
            (dict(kc=float("nan")), INVALID, "powers of two"), (dict(vc=float("inf")), INVALID, "powers of two")]


@pytest.mark.parametrize("kw,code,text", BAD_POOL + [
    (dict(tokens=-1), INVALID, "tokens"), (dict(dtype=2), UNSUPPORTED, "dtype"), (dict(key=0), INVALID, "null"),
    (dict(slots=0), INVALID, "null"), (dict(key=P + 2), INVALID, "aligned"), (dict(ks=1023), INVALID, "strides"),
    (dict(vs=1022), INVALID, "strides"), (dict(ks=0), INVALID, "strides")])
def test_append_refuses(kw, code, text):
    refused("nvk_fp4_append", append_args(**kw), code, text)
    if not {"key", "ks", "vs"} & set(kw):  # the same checks, without strides
        a = dict(key=P, value=P, pool=P, slots=P, tokens=4, nb=8, bs=128, kvh=8, d=128, dtype=0, kc=1.0, vc=1.0, err=0,
                 stream=0)
        refused("nvk_fp4_read", list({**a, **kw}.values()), code, text)


def test_empty_calls_are_no_ops():
    lib = _lib.load()
    assert lib.nvk_fp4_append(*append_args(tokens=0, key=0, slots=0)) == _lib.NVK_OK
    assert lib.nvk_fp4_read(0, 0, P, 0, 0, 8, 128, 8, 128, 0, 1.0, 1.0, 0, 0) == _lib.NVK_OK


def norm_args(**kw):
    a = dict(q=P, k=P, v=P, qs=2048, ks=1024, vs=1024, wq=P, wk=P, eps=1e-6, cos=P, sin=P, max_pos=64, pos=P, out=P,
             pool=P, slots=P, tokens=4, nb=8, bs=128, h=16, kvh=8, d=128, kc=1.0, vc=1.0, err=0, stream=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code,text", BAD_POOL + [
    (dict(tokens=-1), INVALID, "bad sizes"), (dict(h=0), INVALID, "bad sizes"), (dict(max_pos=0), INVALID, "bad sizes"),
    (dict(q=0), INVALID, "null"), (dict(out=0), INVALID, "null"), (dict(cos=0), INVALID, "null"),
    (dict(qs=2046), INVALID, "strides"), (dict(vs=1025), INVALID, "strides"), (dict(v=P + 1), INVALID, "aligned"),
    (dict(sin=P + 2), INVALID, "aligned"), (dict(pos=P + 4), INVALID, "aligned"), (dict(slots=P + 4), INVALID, "aligned"),
    (dict(tokens=(1 << 30) + 1), UNSUPPORTED, "range"), (dict(h=(1 << 20) + 1, qs=1 << 28), UNSUPPORTED, "range")])
def test_norm_rope_append_refuses(kw, code, text):
    refused("nvk_fp4_qk_norm_rope_append", norm_args(**kw), code, text)


def decode_args(**kw):
    a = dict(out=P, q=P, pool=P, nb=8, bs=128, tables=P, stride=4, width=4, ctx=P, batch=2, h=16, kvh=8, d=128,
             scale=0.1, kc=1.0, vc=1.0, ctas=148, ws=P, bytes=1 << 30, stream=0)
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
    refused("nvk_fp4_paged_decode", decode_args(**kw), code, text)


def test_decode_workspace_size():
    lib, sz = _lib.load(), ctypes.c_size_t()
    sizes = []
    for h, kvh, ctas in ((8, 8, 1), (8, 8, 148), (64, 8, 148)):
        assert lib.nvk_fp4_paged_decode_workspace_size(h, kvh, 128, ctas, ctypes.byref(sz)) == 0
        sizes.append(sz.value)
        assert sz.value >= 256 + ctas * 2 * (h // kvh) * 128 * 4
    assert sizes[0] < sizes[1] < sizes[2]
    assert lib.nvk_fp4_paged_decode_workspace_size(8, 8, 64, 1, ctypes.byref(sz)) == UNSUPPORTED
    assert lib.nvk_fp4_paged_decode_workspace_size(8, 8, 128, 1, None) == INVALID
    assert lib.nvk_fp4_paged_decode(*decode_args(batch=0)) == _lib.NVK_OK


def prefill_args(**kw):
    a = dict(out=P, q=P, pool=P, nb=8, bs=128, tables=P, stride=4, width=4, cu=P, lens=P, batch=2, total=8, max_q=8,
             h=16, kvh=8, d=128, scale=0.1, kc=1.0, vc=1.0, err=0, stream=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code,text", BAD_POOL + [
    (dict(batch=-1), INVALID, "bad sizes"), (dict(total=-1), INVALID, "bad sizes"), (dict(h=0), INVALID, "bad sizes"),
    (dict(h=12), INVALID, "multiple"), (dict(scale=0.0), INVALID, "positive"), (dict(stride=3), INVALID, "stride"),
    (dict(cu=0), INVALID, "null"), (dict(out=P + 4), INVALID, "aligned"), (dict(batch=70000), UNSUPPORTED, "grid")])
def test_prefill_refuses(kw, code, text):
    refused("nvk_fp4_paged_prefill", prefill_args(**kw), code, text)


def test_wrappers_refuse_host_tensors_and_bad_shapes():
    pool = torch.zeros(ops_fp4.pool_shape(2, 16, 2), dtype=torch.uint8)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        ops_fp4.kv_append_fp4(pool, k, k, torch.arange(3))
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        ops_fp4.kv_read_fp4(pool, torch.arange(3))
    with pytest.raises(ValueError, match="block_size 24"):
        ops_fp4.pool_shape(2, 24, 2)
    with pytest.raises(ValueError, match="kv_cache must be contiguous uint8"):
        ops_fp4._check_pool("x", pool.transpose(0, 1))
    with pytest.raises(ValueError, match="kv_cache must be contiguous uint8"):
        ops_fp4._check_pool("x", pool.view(torch.int8))
    with pytest.raises(ValueError, match="must be \\[tokens, heads, dim\\]"):
        ops_fp4._row_stride("key", k.transpose(0, 1))
    with pytest.raises(ValueError, match="128 dims"):
        ops_fp4._row_stride("key", torch.zeros(3, 2, 64))
    with pytest.raises(ValueError, match="with 4 entries"):
        ops_fp4._check_index("x", "slot_mapping", torch.arange(3), torch.int64, 4)
    with pytest.raises(ValueError, match="error_word"):
        ops_fp4._error_ptr("x", torch.zeros(1, dtype=torch.int64), torch.device("cpu"))


def test_cache_refuses_and_sizes():
    kv = PagedKVCacheFp4(2, 4, 16, 8, 128, "cpu", k_scale=0.5, v_scale=[1.0, 4.0])
    assert kv.kv_cache.shape == (2, 4, 8, 1, 2304) and kv.bytes_per_block == 2 * 8 * 2304
    key, value = kv.get_physical_cache(1)
    assert key is value and key.shape == (4, 16, 8, 128) and (key.k_scale, key.v_scale) == (0.5, 4.0)
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
    for kw in (dict(k_scale=3.0), dict(v_scale=0.0), dict(k_scale=[1.0]), dict(v_scale=float("inf")),
               dict(k_scale=2.0 ** 70)):
        with pytest.raises(ValueError):
            PagedKVCacheFp4(2, 4, 16, 8, 128, "cpu", **kw)
    with pytest.raises(ValueError, match="head_dim 64"):
        PagedKVCacheFp4(1, 4, 16, 8, 64, "cpu")
    with pytest.raises(ValueError, match="block_size"):
        PagedKVCacheFp4(1, 4, 24, 8, 128, "cpu")


def test_pool_sizing():
    small, large = fp4_bytes_per_block(28, 128, 8), bytes_per_block(28, 128, 8, 128)
    assert large / small == 512 / 144
    n = num_blocks_for_budget(100 << 30, 180 << 30, 0.8, 28, 128, 8, 128, block_bytes=small)
    assert n == (int((180 << 30) * 0.8) - (80 << 30)) // small


def test_attention_over_a_4_bit_layer_checks_like_the_bf16_one():
    kv = PagedKVCacheFp4(1, 4, 16, 8, 128, "cpu")
    key, value = kv.get_physical_cache(0)
    attn = NpuPagedAttention(16, 8, 128)
    with pytest.raises(ValueError, match=re.escape("query shape mismatch: got (2, 8, 128)")):
        attn(torch.zeros(2, 8, 128, dtype=torch.bfloat16), key, value, torch.zeros(2, 1, dtype=torch.int32),
             torch.ones(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="missing block: context length 33"):
        attn(torch.zeros(2, 16, 128, dtype=torch.bfloat16), key, value, torch.zeros(2, 2, dtype=torch.int32),
             torch.tensor([5, 33], dtype=torch.int32))
    other = PagedKVCacheFp4(2, 4, 16, 8, 128, "cpu").get_physical_cache(1)[0]
    for wrong in (other, torch.zeros(4, 16, 8, 128, dtype=torch.bfloat16), None):
        with pytest.raises(ValueError, match="must be the same layer"):
            attn(torch.zeros(2, 16, 128, dtype=torch.bfloat16), key, wrong, torch.zeros(2, 2, dtype=torch.int32),
                 torch.tensor([5, 31], dtype=torch.int32))


class Backend:
    def capturing(self):
        return False


def test_graph_slot_keeps_workspaces_of_different_kinds_apart():
    ids = torch.zeros(2, dtype=torch.int64)
    md = type("Md", (), dict(block_tables=torch.zeros(2, 1, dtype=torch.int32),
                             slot_mapping=torch.zeros(2, dtype=torch.int64)))
    slot = GraphSlot(2, ids, ids, md, None, "cpu", Backend())
    assert slot.workspace is None
    a, b = slot.workspace_for(100), slot.workspace_for(200, "(4-bit)")
    assert a.numel() == 100 and b.numel() == 200 and slot.workspace is a
    assert slot.workspace_for(50) is a and slot.workspace_for(200, "(4-bit)") is b
    assert list(slot.error_names()) == ["decode graph batch 2", "decode graph batch 2 (4-bit)"]


def test_oracle_round_trip():
    """The restatement's own borders: every code and scale comes back, and rounding is to nearest."""
    x = np.random.default_rng(0).standard_normal((40, 1, 128)).astype(np.float64)
    code, s = orc.quantise(x)
    assert np.array_equal(orc.e4m3_value(orc.e4m3_byte(s)), s)
    v = orc.values(code, s)
    again, s2 = orc.quantise(v)
    # a group whose largest value became 6 s keeps its scale and codes
    same = np.abs(v.reshape(40, 1, 8, 16)).max(-1) == 6 * s
    assert np.array_equal(s2[same], s[same])
    assert np.array_equal(orc.values(again, s2).reshape(40, 1, 8, 16)[same], v.reshape(40, 1, 8, 16)[same])
    # off by at most half of the largest step, 2 s, or what lies above 6 s
    err = np.abs(v - x).reshape(40, 1, 8, 16)
    assert (err <= s[..., None] * 1.0 + 1e-12).all()
