"""Rotary positions (``ops.rotary``) against the formula in 64 bits.

Tolerance: the result's own rounding (half a step: bf16 2^-8, fp16 2^-11, and
2^-25 where fp16 is subnormal), and of the pair's magnitudes 2^-20: the angle
is within 2^-24 of a turn (2^-21.3 radians), and the norm (2^-22 of its
reciprocal root, 128 sums of 2^-24 whose errors partly cancel), the factor, the
weight and the turn add a few 2^-24.
"""

import numpy as np
import pytest
import torch

from nano_vllm_ascend_b200 import ops

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def formula(x, w, eps, inv, pos, interleaved, factor):
    """(result, magnitudes that its errors are relative to), float64."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    half = inv.numel()
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    angle = pos.double()[:, None, None] * inv
    y, mag = x.clone(), x.abs()
    y[..., a] = (x[..., a] * angle.cos() - x[..., b] * angle.sin()) * factor
    y[..., b] = (x[..., b] * angle.cos() + x[..., a] * angle.sin()) * factor
    mag[..., a] = mag[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(factor)
    return y, mag


def check(got, want, mag):
    err = (got.double() - want).abs()
    tol = want.abs() * HALF[got.dtype] + mag * 2.0 ** -20 + 2.0 ** -25 * (got.dtype == torch.float16) + 1e-37
    assert bool((err <= tol).all()), float((err / tol).max())


def frequencies(half, base=1e4):
    return base ** -(torch.arange(half, dtype=torch.float64) / max(half, 1))


def case(dev, tokens, h, kvh, dim, rotated, interleaved, norm, dtype, far=40960, factor=1.0, seed=0, gap=0, shift=0,
         inplace=False, strided_out=False):
    g = torch.Generator().manual_seed(seed)
    rows = h + kvh

    def strided(t):
        buf = torch.full((shift + tokens * (rows * dim + gap),), float("nan"), dtype=dtype, device=dev)
        view = torch.as_strided(buf, (tokens, rows, dim), (rows * dim + gap, dim, 1), shift)
        if t is not None:
            view.copy_(t)
        return view

    x = strided(torch.randn(tokens, rows, dim, generator=g).to(dtype))
    q, k = x[:, :h], x[:, h:]
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dtype).to(dev) if norm else None for _ in range(2))
    inv = frequencies(rotated // 2).to(dev)
    pos = torch.randint(0, far, (tokens,), generator=g).to(dev)
    if tokens:
        pos[-1] = far - 1
    want = [formula(t, w, 1e-6, inv, pos, interleaved, factor) for t, w in ((q, wq), (k, wk))]
    outs = dict()
    if inplace:
        outs = dict(query_out=q, key_out=k)
    elif strided_out:
        y = strided(None)
        outs = dict(query_out=y[:, :h], key_out=y[:, h:])
    got = ops.rotary(q, k, inv, pos, interleaved=interleaved, attention_scale=factor, q_weight=wq, k_weight=wk,
                     eps=1e-6, **outs)
    for g_, (w_, m_), name in zip(got, want, ("query_out", "key_out")):
        check(g_, w_, m_)
        if outs:
            assert g_ is outs[name]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dim,rotated", [(128, 128), (128, 64), (128, 32), (128, 2), (128, 126), (64, 64), (64, 16),
                                         (256, 256), (256, 64), (80, 80), (80, 20), (96, 48), (2, 2), (512, 512),
                                         (130, 66), (192, 128)])
def test_layouts_and_dims(cuda_device, dim, rotated, interleaved, norm):
    for dtype in HALF:
        case(cuda_device, 5, 3, 1, dim, rotated, interleaved, norm, dtype, seed=dim + rotated)


@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 333, 1500])
@pytest.mark.parametrize("h,kvh", [(16, 8), (1, 1), (5, 2), (32, 8)])
def test_tokens_and_heads(cuda_device, tokens, h, kvh):
    case(cuda_device, tokens, h, kvh, 128, 128, False, True, torch.bfloat16, seed=tokens)
    case(cuda_device, tokens, h, kvh, 128, 64, True, False, torch.float16, seed=tokens, factor=1.2)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dim,rotated", [(128, 128), (64, 32), (80, 40)])
@pytest.mark.parametrize("shift,gap", [(8, 8), (1, 0), (4, 4), (0, 3), (2, 2 * 128)])
def test_strides_and_alignment(cuda_device, dim, rotated, shift, gap, norm):
    for interleaved in (False, True):
        case(cuda_device, 9, 4, 2, dim, rotated, interleaved, norm, torch.bfloat16, shift=shift, gap=gap)
        case(cuda_device, 9, 4, 2, dim, rotated, interleaved, norm, torch.bfloat16, shift=shift, gap=gap,
             strided_out=True)
        case(cuda_device, 9, 4, 2, dim, rotated, interleaved, norm, torch.bfloat16, shift=shift, gap=gap, inplace=True)


@pytest.mark.parametrize("far", [1, 1 << 20, (1 << 31) + 7, 1 << 40])
def test_far_positions_keep_their_angle(cuda_device, far):
    """A position times a frequency in 64 bits; at 2^40 its rounding is 2^-13 of a radian, in the formula too (the same
    product), so that the results still agree."""
    case(cuda_device, 40, 2, 2, 128, 128, False, False, torch.bfloat16, far=far)
    case(cuda_device, 40, 2, 2, 64, 64, True, True, torch.float16, far=far)


def test_negative_positions_and_factors(cuda_device):
    dev = cuda_device
    q = torch.randn(6, 2, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    pos = torch.tensor([-1, 0, -1000, 5, -(1 << 33), 1], device=dev)
    inv = frequencies(32).to(dev)
    got = ops.rotary(q, q, inv, pos, attention_scale=-0.5)
    want, mag = formula(q, None, 0, inv, pos, False, -0.5)
    for g in got:
        check(g, want, mag)


def test_rows_of_zeros_and_values_that_are_no_numbers(cuda_device):
    """A row of zeros under a norm stays zeros; a NaN or an infinity stays in its pair without a norm, and in its row
    with one."""
    dev = cuda_device
    q = torch.randn(3, 4, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    q[0, 1] = 0
    q[1, 2, 5], q[2, 3, 127] = float("nan"), float("inf")
    w = torch.ones(128, dtype=torch.bfloat16, device=dev)
    inv, pos = frequencies(64).to(dev), torch.arange(3, device=dev) + 1
    plain, _ = ops.rotary(q, q, inv, pos)
    normed, _ = ops.rotary(q, q, inv, pos, q_weight=w, k_weight=w)
    assert not normed[0, 1].any() and not plain[0, 1].any()
    bad = ~plain.isfinite()
    assert bad[1, 2, 5] and bad[1, 2, 69] and bad[2, 3, 127] and bad[2, 3, 63] and int(bad.sum()) == 4
    bad = ~normed.isfinite()
    assert bad[1, 2].all() and bad[2, 3, 127] and not bad[0].any() and not bad[1, :2].any() and not bad[1, 3].any()


def test_nothing_to_do(cuda_device):
    dev = cuda_device
    inv = frequencies(64).to(dev)
    q = torch.empty(0, 4, 128, dtype=torch.bfloat16, device=dev)
    a, b = ops.rotary(q, q, inv, torch.empty(0, dtype=torch.int64, device=dev))
    assert a.shape == b.shape == (0, 4, 128)


def test_as_the_norm_rope_append_kernel_but_for_its_roundings(cuda_device):
    """qk_norm_rope_append rounds the norm's result, cos and sin to bf16: within a few of its half steps."""
    dev = cuda_device
    t, h, kvh, bs = 70, 16, 8, 128
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(t, h + 2 * kvh, 128, generator=g).to(torch.bfloat16).to(dev)
    q, k, v = qkv[:, :h], qkv[:, h:h + kvh], qkv[:, h + kvh:]
    w = (1 + 0.1 * torch.randn(128, generator=g)).to(torch.bfloat16).to(dev)
    inv = frequencies(64, 1e6)
    f = torch.outer(torch.arange(4096, dtype=torch.float64), inv)
    f = torch.cat((f, f), -1)
    pos = torch.randint(0, 4096, (t,), generator=g).to(dev)
    kc, vc = (torch.zeros(1, bs, kvh, 128, dtype=torch.bfloat16, device=dev) for _ in range(2))
    slots = torch.arange(t, device=dev)
    want = ops.qk_norm_rope_append(q, k, v, w, w, 1e-6, f.cos().float().to(dev), f.sin().float().to(dev), pos, kc, vc,
                                   slots)
    got, gotk = ops.rotary(q, k, inv.to(dev), pos, q_weight=w, k_weight=w)
    _, mag = formula(q, w, 1e-6, inv.to(dev), pos, False, 1.0)
    _, magk = formula(k, w, 1e-6, inv.to(dev), pos, False, 1.0)
    # the norm's rounding and cos and sin's: two half steps of each product, then both results' own
    for a, b, m in ((got, want, mag), (gotk, kc[0, :t], magk)):
        assert bool(((a.double() - b.double()).abs() <= 2 * 2.0 ** -8 * m + 2 * 2.0 ** -8 * a.double().abs()).all())


def test_in_a_graph_and_on_another_stream(cuda_device):
    dev = cuda_device
    q = torch.randn(33, 4, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    inv, pos = frequencies(64).to(dev), torch.arange(33, device=dev)
    out = [torch.empty_like(q), torch.empty_like(q)]
    ops.rotary(q, q, inv, pos, query_out=out[0], key_out=out[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary(q, q, inv, pos, query_out=out[0], key_out=out[1])
    pos.add_(1000)
    graph.replay()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other, _ = ops.rotary(q, q, inv, pos)
    torch.cuda.synchronize()
    assert torch.equal(other, out[0]) and torch.equal(out[0], out[1])
    want, mag = formula(q, None, 0, inv, pos, False, 1.0)
    check(other, want, mag)
