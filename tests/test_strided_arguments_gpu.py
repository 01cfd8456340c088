"""Index tensors and weights that are strided views: the wrappers copy them, and each copy lives until the launch, so that
the call is the one with packed tensors, bit for bit."""

import pytest
import torch

from nano_vllm_ascend_b200 import ops

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def strided(t):
    """The same values at every third place, wild ones between."""
    wide = torch.full((*t.shape, 3), 1000, dtype=t.dtype, device=t.device)
    wide[..., 0] = t
    return wide[..., 0]


def randn(dev, *shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(BF).to(dev)


def test_norm_rope_append(cuda_device):
    dev, t, h, kvh, d = cuda_device, 40, 4, 2, 128
    q, k, v = randn(dev, t, h, d), randn(dev, t, kvh, d, seed=1), randn(dev, t, kvh, d, seed=2)
    wq, wk = 1 + 0.3 * randn(dev, d, seed=3), 1 + 0.3 * randn(dev, d, seed=4)
    angle = torch.outer(torch.arange(2048.0), 1e4 ** (-torch.arange(64.0) / 64)).repeat(1, 2).to(dev)
    positions, slots = torch.arange(t, device=dev) * 7 % 100, torch.arange(t, device=dev).flip(0)
    results = []
    for view in (lambda x: x, strided):
        kc, vc = (torch.zeros(4, 16, kvh, d, dtype=BF, device=dev) for _ in range(2))
        out = ops.qk_norm_rope_append(q, k, v, view(wq), view(wk), 1e-6, angle.cos(), angle.sin(), view(positions), kc, vc,
                                      view(slots))
        results.append((out, kc, vc))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_prefill(cuda_device):
    dev, h, kvh, d, bs = cuda_device, 4, 2, 128, 128
    kc, vc = randn(dev, 6, bs, kvh, d, seed=1), randn(dev, 6, bs, kvh, d, seed=2)
    q = randn(dev, 90, h, d)
    tables = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 30, 31, 90], dtype=torch.int32, device=dev)
    lens = torch.tensor([150, 256, 60], dtype=torch.int32, device=dev)
    results = [ops.paged_prefill(torch.empty_like(q), q, kc, vc, tables, view(cu), view(lens), 59, d ** -0.5)
               for view in (lambda x: x, strided)]
    assert torch.equal(*results)
    k, v = randn(dev, 130, kvh, d, seed=3), randn(dev, 130, kvh, d, seed=4)
    cu_kv = torch.tensor([0, 50, 61, 130], dtype=torch.int32, device=dev)
    results = [ops.dense_prefill(torch.empty_like(q), q, k, v, view(cu), view(cu_kv), 59, d ** -0.5)
               for view in (lambda x: x, strided)]
    assert torch.equal(*results)
