"""8-bit prefill: how exactly weights and scores are held, by items of one CTA and by items divided over a cluster's.

The kernel holds weights in fp16, times 2^7 and relative to a reference that the
largest product of a weight and its unit's power of two is at least as large as.
So, as in test_fp8_gpu, but with what that means for the weights (half steps):

* a weight's rounding is 2^-11 of it, so 2^-11 A;
* scores (below 2^7 in log2 units) and the exponential, another 2^-11 A; the
  reference's rounding, where that is below 2^10 in log2 units, 2^-15, is in it;
* fp16's smallest step is 2^-24: a product is off by half of it where the
  largest one is held as at least 2^7, so by 2^-32 of that one.
"""

import math

import pytest
import torch

from nano_vllm_ascend_b200 import ops_fp8
from oracle import fp4_oracle
from tests import test_fp8_gpu as base

pytestmark = pytest.mark.gpu

D = 128
HOW = dict(per_a=2.0 ** -11 + 2.0 ** -11, step=2.0 ** -32)
LOG2 = math.log(2.0)  # the scale under which q . k is the score in log2 units
# items of one head: 1 is divided over a cluster where its keys are five tiles or more, 80 are not (B200: 148 SMs)
ITEMS = [1, 80]


def filled(dev, k, v, bs=128):
    """A pool over which `k` and `v` ([n, 1, 128]) are one sequence, and its rows in float64."""
    n = k.shape[0]
    pool = torch.zeros(ops_fp8.pool_shape(-(-n // bs), bs, 1), dtype=torch.uint8, device=dev)
    slots = torch.arange(n, device=dev)
    ops_fp8.kv_append_fp8(pool, k.to(torch.bfloat16).to(dev), v.to(torch.bfloat16).to(dev), slots)
    return (pool, *(t.double() for t in ops_fp8.kv_read_fp8(pool, slots)))


def attend(pool, q, n, scale, items):
    """The rows q [m, 1, 128] as the last m of n tokens, by `items` sequences over the same blocks; all give the same."""
    dev, m = pool.device, q.shape[0]
    queries = q.repeat(items, 1, 1)
    out = torch.full_like(queries, float("nan"))
    table = torch.arange(pool.shape[0], dtype=torch.int32, device=dev).repeat(items, 1)
    ops_fp8.paged_prefill_fp8(out, queries, pool, table, torch.arange(items + 1, dtype=torch.int32, device=dev) * m,
                              torch.full((items,), n, dtype=torch.int32, device=dev), m, scale)
    out = out.view(items, m, 1, D)
    assert bool((out == out[0]).all())
    return out[0]


@pytest.mark.parametrize("q_lens,cached,h,kvh,bs,kw", [
    ([1, 130, 64], [0, 77, 256], 1, 1, 64, {}), ([1, 130, 64], [0, 77, 256], 9, 3, 64, {}),
    ([1, 130, 64], [0, 77, 256], 16, 8, 32, {}), ([1500, 900], [0, 2100], 4, 2, 128, {}), ([40], [7000], 2, 1, 32, {}),
    ([150], [1700], 4, 1, 32, {}), ([200], [100], 4, 1, 32, dict(q_mul=8.0)),
    ([200], [100], 4, 1, 32, dict(q_mul=2.0 ** -6, spread=16)), ([150], [1700], 4, 1, 32, dict(q_mul=8.0)),
    ([150], [1700], 4, 1, 32, dict(q_mul=2.0 ** -6, spread=16)), ([200], [100], 4, 1, 32, dict(q_mul=2.0 ** 30, mul=2.0 ** -30)),
    ([150], [1700], 4, 1, 32, dict(q_mul=2.0 ** -30, mul=2.0 ** 30))])
def test_weights_are_as_exact_as_fp16(cuda_device, monkeypatch, q_lens, cached, h, kvh, bs, kw):
    monkeypatch.setattr(base, "PREFILL", HOW)
    base.prefill_case(cuda_device, q_lens, cached, h, kvh, bs, seed=11, **kw)


@pytest.mark.parametrize("items", ITEMS)
@pytest.mark.parametrize("tail", [-6, -15, -20, -24])
@pytest.mark.parametrize("vexp", [0, 20, -20])
def test_tail_of_small_weights_beside_other_exponents(cuda_device, tail, vexp, items):
    """20000 tokens of weight 2^tail each beside one of weight 1, V of the tail 2^vexp times as large: what the tail
    gives is there, however the units' exponents differ."""
    n = 20000
    k = torch.zeros(n, 1, D)
    v = torch.randn(n, 1, D, generator=torch.Generator().manual_seed(1)).abs() * 2.0 ** vexp
    k[:, 0, 0] = tail
    k[0, 0, 0] = 0.0
    v[0] = 1.0
    q = torch.zeros(1, 1, D, dtype=torch.bfloat16, device=cuda_device)
    q[0, 0, 0] = 1.0
    for heavy in (0, n // 2, n - 16):  # the heavy token's place, the first one of a unit of its own
        kk, vv = k.clone(), v.clone()
        if heavy:
            kk[0], kk[heavy], vv[0], vv[heavy] = k[1], k[0], v[1], v[0]
        unit = torch.arange(n) // 16 == heavy // 16
        unit[heavy] = False
        vv[unit] = 0
        pool, kr, vr = filled(cuda_device, kk, vv, 256)
        out = attend(pool, q, n, LOG2, items)
        want, a = fp4_oracle.attention(q, kr, vr, LOG2)
        err = (out.double() - want).abs()
        # weights are powers of two, so exact where they are 2^-24 or more beside 2^7, or 2^-32 of the largest product off
        tol = want.abs() * 2.0 ** -8 + a * 2.0 ** -10 + 2 * n * 2.0 ** -32 * (vr.abs() * torch.exp2(kr[:, :, :1])).max()
        assert bool((err <= tol).all()), float((err / tol).max())
        # the tail is exact (vexp 0 and 20), or below 2^-11 of the whole (vexp -20: 20000 times at most 2^-25)
        assert bool((err <= want.abs() * 0.01).all()), float((err / want.abs()).max())


@pytest.mark.parametrize("items", ITEMS)
def test_scores_of_any_magnitude(cuda_device, items):
    """Scores of 2^4 to 2^60 in log2 units (products exact in 13 bits), over units of different exponents of K and of V:
    weights go by differences, so that they hold."""
    dev, n, ups = cuda_device, 640, [4, 9, 10, 12, 24, 40, 60]
    g = torch.Generator().manual_seed(2)
    unit = torch.arange(n) // 16
    k = torch.zeros(n, 1, D)
    k[:, 0, 0] = 1.0
    k[:, 0, 1] = torch.randint(0, 9, (n,), generator=g) / 8.0
    k[:, 0, 5] = torch.exp2((unit * 3 % 7).float())  # beside an entry of q that is 0: the unit's exponent alone
    v = torch.randn(n, 1, D, generator=g) * torch.exp2((unit % 5 - 2.0) * 4)[:, None, None]
    pool, kr, vr = filled(dev, k, v)
    q = torch.zeros(len(ups), 1, D, dtype=torch.bfloat16, device=dev)
    for i, up in enumerate(ups):
        q[i, 0, 0], q[i, 0, 1] = 2.0 ** up, 2.0 ** (up - 10)
    out = attend(pool, q, n, LOG2, items)
    want, a = fp4_oracle.attention(q, kr, vr, LOG2)
    base.check(out, want, a, n, float(vr.abs().max()), HOW)


@pytest.mark.parametrize("items", ITEMS)
@pytest.mark.parametrize("n", [32, 1024])
def test_scores_next_to_zero_of_the_largest_keys(cuda_device, n, items):
    """Keys at the format's end, +-448 * 2^40, and queries so small (2^-90) that all scores are within 2^-30 of 0: every
    weight is the same, and values of both signs cancel."""
    k = torch.full((n, 1, D), 448 * 2.0 ** 40)
    k[1::2] *= -1
    v = torch.ones(n, 1, D)
    v[1::2] *= -1
    pool, kr, vr = filled(cuda_device, k, v)
    q = torch.full((1, 1, D), 1.9921875 * 2.0 ** -90, dtype=torch.bfloat16, device=cuda_device)
    out = attend(pool, q, n, D ** -0.5, items)
    want, a = fp4_oracle.attention(q, kr, vr, D ** -0.5)
    base.check(out, want, a, n, float(vr.abs().max()), HOW)
