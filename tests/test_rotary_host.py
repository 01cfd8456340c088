"""Rotary frequencies against their formulas, and what the rotary and page calls refuse, without a GPU."""

import math

import pytest
import torch

from nano_vllm_ascend_b200 import _lib, ops, rotary_frequencies

INVALID, UNSUPPORTED = _lib.NVK_ERR_INVALID_ARGUMENT, _lib.NVK_ERR_UNSUPPORTED
P = 1 << 20  # a pointer that is never followed: every call here is refused or empty


def plain(dim, base):
    return [base ** (-2.0 * i / dim) for i in range(dim // 2)]


@pytest.mark.parametrize("dim,base", [(2, 10000.0), (64, 1e4), (128, 1e6), (96, 5e5)])
def test_frequencies_and_their_scalings(dim, base):
    want = plain(dim, base)
    inv, scale = rotary_frequencies(dim, base)
    close = lambda a, b: torch.allclose(a, torch.tensor(b, dtype=torch.float64), rtol=1e-13, atol=0)
    assert inv.dtype == torch.float64 and scale == 1.0 and close(inv, want)
    inv, scale = rotary_frequencies(dim, base, dict(type="linear", factor=4))
    assert scale == 1.0 and close(inv, [w / 4 for w in want])
    inv, scale = rotary_frequencies(dim, base, dict(type="ntk", factor=8.0))
    assert scale == 1.0 and float(inv[0]) == 1.0
    if dim > 2:
        assert math.isclose(float(inv[-1]), want[-1] / 8, rel_tol=1e-12)
        grown = base * 8 ** (dim / (dim - 2))
        assert close(inv, plain(dim, grown))
    length, low, high = 8192, 1.0, 4.0
    inv, scale = rotary_frequencies(dim, base, dict(type="wavelength", factor=8, original_max_position=length,
                                                    low_freq_factor=low, high_freq_factor=high))
    blended = []
    for w in want:
        wave = 2 * math.pi / w
        if wave < length / high:
            blended.append(w)
        elif wave > length / low:
            blended.append(w / 8)
        else:
            smooth = (length / wave - low) / (high - low)
            blended.append((1 - smooth) * w / 8 + smooth * w)
    assert scale == 1.0 and close(inv, blended)


@pytest.mark.parametrize("dim,base,length,factor", [(128, 1e4, 4096, 16.0), (64, 1e6, 32768, 4.0), (128, 1e6, 2048, 40.0)])
def test_yarn_keeps_what_turns_often_and_scales_what_turns_rarely(dim, base, length, factor):
    want = plain(dim, base)
    inv, scale = rotary_frequencies(dim, base, dict(type="yarn", factor=factor, original_max_position=length))
    assert math.isclose(scale, 0.1 * math.log(factor) + 1)
    turns = [length * w / (2 * math.pi) for w in want]
    # the ramp's ends are whole pairs, below the one of 32 turns and above that of one
    low = max(math.floor(sum(t > 32 for t in turns) - 1e-9) - 1, 0)
    ratio = [float(i) / w for i, w in zip(inv, want)]
    for i, (r, t) in enumerate(zip(ratio, turns)):
        if i <= low:
            assert math.isclose(r, 1.0, rel_tol=1e-12), i
        assert 1 / factor * (1 - 1e-12) <= r <= 1 + 1e-12
        if i and turns[i - 1] < 1:
            assert math.isclose(r, 1 / factor, rel_tol=1e-12), i
    assert all(a >= b - 1e-12 for a, b in zip(ratio, ratio[1:]))
    steps = [a - b for a, b in zip(ratio, ratio[1:]) if a < 1 - 1e-9 and b > 1 / factor + 1e-9]
    assert all(math.isclose(s, steps[0], rel_tol=1e-6) for s in steps)  # a line over the pairs between
    assert rotary_frequencies(dim, base, dict(type="yarn", factor=factor, original_max_position=length,
                                              attention_factor=1.5))[1] == 1.5


@pytest.mark.parametrize("args,text", [
    ((0,), "rotary_dim 0"), ((5,), "rotary_dim 5"), ((-2,), "rotary_dim -2"), ((64, 1.0), "base"), ((64, float("nan")), "base"),
    ((64, 1e4, dict(type="cubic")), "is none of"), ((64, 1e4, dict(factor=2)), "is none of"),
    ((64, 1e4, dict(type="linear")), "takes"), ((64, 1e4, dict(type="linear", factor=2, extra=1)), "takes"),
    ((64, 1e4, dict(type="linear", factor=0.5)), "below 1"), ((64, 1e4, dict(type="ntk", factor=float("nan"))), "below 1"),
    ((64, 1e4, dict(type="yarn", factor=2)), "takes"),
    ((64, 1e4, dict(type="wavelength", factor=2, original_max_position=8, low_freq_factor=4, high_freq_factor=4)),
     "is not below")])
def test_frequencies_refuse(args, text):
    with pytest.raises(ValueError, match=text):
        rotary_frequencies(*args)


def refused(name, args, code, text):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == code, lib.nvk_last_error()
    assert text in lib.nvk_last_error().decode()


def rotary_args(**kw):
    a = dict(qo=P, ko=P, q=P, k=P, qos=2048, kos=1024, qs=2048, ks=1024, wq=P, wk=P, eps=1e-6, inv=P, pos=P, factor=1.0,
             tokens=4, h=16, kvh=8, dim=128, rot=128, inter=0, dtype=0, stream=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(tokens=-1), INVALID, "bad sizes"), (dict(h=-1), INVALID, "bad sizes"), (dict(kvh=-1), INVALID, "bad sizes"),
    (dict(dim=0), UNSUPPORTED, "head_dim"), (dict(dim=127), UNSUPPORTED, "head_dim"), (dict(dim=514), UNSUPPORTED, "head_dim"),
    (dict(rot=0), INVALID, "rotary_dim"), (dict(rot=7), INVALID, "rotary_dim"), (dict(rot=130), INVALID, "rotary_dim"),
    (dict(dtype=2), UNSUPPORTED, "dtype"), (dict(q=0), INVALID, "null"), (dict(ko=0), INVALID, "null"),
    (dict(inv=0), INVALID, "null"), (dict(pos=0), INVALID, "null"), (dict(wq=0), INVALID, "only one"),
    (dict(wk=0), INVALID, "only one"), (dict(inv=P + 4), INVALID, "aligned"), (dict(pos=P + 4), INVALID, "aligned"),
    (dict(q=P + 1), INVALID, "aligned"), (dict(qs=2047), INVALID, "strides"), (dict(kos=0), INVALID, "strides")])
def test_rotary_refuses(kw, code, text):
    refused("nvk_rotary", rotary_args(**kw), code, text)


def test_empty_calls_are_no_ops():
    lib = _lib.load()
    assert lib.nvk_rotary(*rotary_args(tokens=0)) == _lib.NVK_OK
    assert lib.nvk_copy_blocks(P, P, 2, 8, 64, P, 0, 0, 0) == _lib.NVK_OK
    assert lib.nvk_remap_blocks(P, 4, 0, 4, P, 8, 0, 0) == _lib.NVK_OK


@pytest.mark.parametrize("kw,code,text", [
    (dict(layers=-1), INVALID, "bad sizes"), (dict(nb=-1), INVALID, "bad sizes"), (dict(n=-1), INVALID, "bad sizes"),
    (dict(bytes=-16), INVALID, "bad sizes"), (dict(bytes=40), UNSUPPORTED, "multiples of 16"),
    (dict(pool=0), INVALID, "null"), (dict(pairs=0), INVALID, "null"), (dict(pool=P + 8), INVALID, "aligned"),
    (dict(pool2=P + 8), INVALID, "aligned"), (dict(pairs=P + 4), INVALID, "aligned"), (dict(bytes=1 << 60), UNSUPPORTED, "bytes")])
def test_copies_refuse(kw, code, text):
    a = dict(pool=P, pool2=P, layers=2, nb=8, bytes=64, pairs=P, n=3, err=0, stream=0)
    refused("nvk_copy_blocks", list({**a, **kw}.values()), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(rows=-1), INVALID, "bad sizes"), (dict(width=-1), INVALID, "bad sizes"), (dict(stride=3), INVALID, "bad sizes"),
    (dict(nb=0), INVALID, "bad sizes"), (dict(tables=0), INVALID, "null"), (dict(map=0), INVALID, "null")])
def test_remaps_refuse(kw, code, text):
    a = dict(tables=P, stride=4, rows=2, width=4, map=P, nb=8, err=0, stream=0)
    refused("nvk_remap_blocks", list({**a, **kw}.values()), code, text)


def test_wrappers_refuse_host_tensors():
    q = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    inv, _ = rotary_frequencies(128)
    with pytest.raises(ValueError, match="must be a CUDA tensor|CUDA"):
        ops.rotary(q, q, inv, torch.arange(3))
    with pytest.raises(ValueError, match="CUDA"):
        ops.copy_blocks(torch.zeros(1, 4, 16), torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        ops.remap_blocks(torch.zeros(1, 4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    for pools in ([], [q, q, q]):
        with pytest.raises(ValueError, match="one or two"):
            ops.copy_blocks(pools, torch.zeros(1, 2, dtype=torch.int32))
