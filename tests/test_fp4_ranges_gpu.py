"""4-bit attention at the ends of its ranges: constants, scales, queries, scores and V rows of any magnitude.

Compared with 64-bit arithmetic over the values that the codes stand for; tolerances as in tests/test_fp4_gpu.py.
"""

import pytest
import torch

from nano_vllm_ascend_b200 import ops_fp4
from oracle import fp4_oracle as orc
from tests.test_fp4_gpu import D, DECODE, PREFILL, SCALE, check, decode_case, random_rows, workspace

pytestmark = pytest.mark.gpu


def pool_of(dev, k, v, bs, ks=1.0, vs=1.0):
    """A pool that holds rows k and v (times the constants), and what it reads back, in float64."""
    nb = -(-k.shape[0] // bs)
    pool = torch.zeros(ops_fp4.pool_shape(nb, bs, k.shape[1]), dtype=torch.uint8, device=dev)
    slots = torch.arange(k.shape[0], device=dev)
    ops_fp4.kv_append_fp4(pool, (k.to(dev) * ks).contiguous(), (v.to(dev) * vs).contiguous(), slots, ks, vs)
    kr, vr = ops_fp4.kv_read_fp4(pool, slots, ks, vs)
    return pool, kr.double(), vr.double()


def attend(which, q, pool, n, scale, ks=1.0, vs=1.0, num_ctas=0):
    """q [m, heads, 128] over the pool's first n slots: m tokens of one sequence, or one of m == 1 in decode."""
    dev, (nb, kvh) = q.device, pool.shape[:2]
    table = torch.arange(nb, dtype=torch.int32, device=dev)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    out = torch.full_like(q, float("nan"))
    if which == "decode":
        ws = workspace(dev, q.shape[1], kvh, num_ctas)
        ops_fp4.paged_decode_fp4(out, q, pool, table, lens, scale, ws, num_ctas, ks, vs)
        assert int(ws[:4].view(torch.int32).item()) == 0
    else:
        cu = torch.tensor([0, q.shape[0]], dtype=torch.int32, device=dev)
        ops_fp4.paged_prefill_fp4(out, q, pool, table, cu, lens, q.shape[0], scale, ks, vs)
    return out


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("ks,scale", [(2.0 ** -60, SCALE), (2.0 ** -36, SCALE), (1.0, 1e-38), (1.0, 1e-45),
                                      (2.0 ** -60, 1e-38), (2.0 ** 60, 1e-38)])
def test_zero_and_tiny_queries_with_any_constant(cuda_device, which, ks, scale):
    """Rows of zeros and of next to nothing weigh all keys the same, whatever the constant and the scale, with a tile
    that ends inside (150 tokens) and, in prefill, masked rows."""
    dev, h, n = cuda_device, 4, 150
    m = 1 if which == "decode" else 40
    k, v = random_rows(n, 2, 31, spread=False)
    pool, kr, vr = pool_of(dev, k, v, 32, ks)
    q = torch.randn(m, h, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    q = (q * torch.tensor([0.0, 2.0 ** -126, 2.0 ** -133, 1.0], dtype=torch.bfloat16)[None, :, None]).to(dev)
    out = attend(which, q, pool, n, scale, ks)
    want, a = orc.attention(q, kr, vr, scale)
    check(out, want, a, vr, DECODE if which == "decode" else PREFILL)


def exact_scores_case(dev, n, kvh, m, h):
    """K rows and queries whose products q . k are multiples of 1/2 below 2^21, so exact in fp32, about +-2^20.2 and 0
    with differences of a few units; V random."""
    g = torch.Generator().manual_seed(n + m)
    levels = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6])
    k = levels[torch.randint(0, 8, (n, kvh, D), generator=g)] * (torch.randint(0, 2, (n, kvh, D), generator=g) * 2 - 1)
    k[:, :, 16::16] = 6.0  # every group's scale is 1
    k[:, :, :16] = 0.0
    k[:, :, 0] = 2304.0  # 6 * 384
    q = torch.randint(-3, 4, (m, h, D), generator=g).float()
    q[:, :, :16] = 0.0
    q[:, :, 0] = torch.tensor([512.0, -512.0, 0.0, 512.0]).repeat(h // 4)
    _, v = random_rows(n, kvh, n, spread=False)
    return q.to(torch.bfloat16).to(dev), k.to(torch.bfloat16), v


@pytest.mark.parametrize("which,n,num_ctas", [("decode", 150, 1), ("decode", 3000, 7), ("decode", 5000, 148),
                                              ("prefill", 300, 0)])
@pytest.mark.parametrize("e", [-12, -6, 0, 4, 8, 12, 40, 90, 120])
def test_scores_of_any_magnitude(cuda_device, which, n, num_ctas, e):
    """Scores of 2^8 to past fp32's largest, whose differences are exact: the weights go by the differences alone."""
    m = 1 if which == "decode" else 40
    q, k, v = exact_scores_case(cuda_device, n, 2, m, 8)
    pool, kr, vr = pool_of(cuda_device, k, v, 32)
    out = attend(which, q, pool, n, 2.0 ** e, num_ctas=num_ctas)
    want, a = orc.attention(q, kr, vr, 2.0 ** e)
    check(out, want, a, vr, DECODE if which == "decode" else PREFILL, f"scale 2^{e}")


def check_relative(got, want, a, v, how):
    """As ``check``, with what small weights lose counted against the largest |v| of the same KV head: half of fp16's
    smallest step over the power of two that p is held with, and 2^-36 for the products with the scales, which are
    held with the largest of them near fp16's end (half of 2^-24 of a code of 6, over 2^4 p and 2^8 of the scale)."""
    n, kvh, _ = v.shape
    top = v.abs().amax((0, 2)).repeat_interleave(got.shape[1] // kvh)[None, :, None]
    tol = want.abs() * 2.0 ** -8 + a * how["per_a"] + n * (how["step"] + 2.0 ** -36) * top + 1e-30
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"off by up to {float((err / tol).max()):.2f} tolerances"


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("far", [8, 16, 20, 23])
@pytest.mark.parametrize("at", [0, 7000, 20479])
@pytest.mark.parametrize("s", [2.0 ** -9, 3 * 2.0 ** -9, 2.0 ** -6, 1.0, 448.0])
def test_a_long_tail_of_small_rows_behind_one_dominant_token(cuda_device, which, far, at, s):
    """20479 tokens of weight 2^-far beside one whose V is zero: the output is the tail's share, for V of every
    magnitude that the format holds. One CTA, so that a warp has hundreds of the tail beside the dominant token."""
    dev, n, kvh, h = cuda_device, 20480, 1, 4
    g = torch.Generator().manual_seed(far)
    v = s * torch.tensor([3.0, 4.0, 6.0])[torch.randint(0, 3, (n, kvh, D), generator=g)]
    v[:, :, ::16] = 6.0 * s  # every group of the tail has its scale
    k = torch.zeros(n, kvh, D)
    v[at], k[at, :, 5] = 0.0, 6.0
    pool, kr, vr = pool_of(dev, k.to(torch.bfloat16), v.to(torch.bfloat16), 256)
    assert torch.equal(vr.cpu(), v.double())
    q = torch.zeros(1, h, D, dtype=torch.bfloat16, device=dev)
    q[:, :, 5] = 1.0
    scale = far / 6 / 1.4426950408889634
    out = attend(which, q, pool, n, scale, num_ctas=1)
    want, a = orc.attention(q, kr, vr, scale)
    check_relative(out, want, a, vr, DECODE if which == "decode" else PREFILL)


@pytest.mark.parametrize("num_ctas", [1, 5, 148])
@pytest.mark.parametrize("h", [3, 8])
def test_v_groups_whose_scales_grow(cuda_device, num_ctas, h):
    """Groups of random magnitude, larger from token to token here and smaller there, some of zeros, over all splits."""
    n, kvh = 3000, 1
    g = torch.Generator().manual_seed(h)
    k, v = random_rows(n, kvh, 77, spread=False)
    e = torch.randint(-9, 9, (n, kvh, 8, 1), generator=g).float()
    e[:, :, 0] = torch.linspace(-9, 8, n)[:, None, None]  # grows
    e[:, :, 1] = torch.linspace(8, -9, n)[:, None, None]
    e[:, :, 2] = -8.0
    v = (v.float().view(n, kvh, 8, 16) * torch.exp2(e)).view(n, kvh, D)
    v[:, :, 48:64] = 0.0
    pool, kr, vr = pool_of(cuda_device, k, v.to(torch.bfloat16), 32)
    q = torch.randn(1, h, D, generator=g).to(torch.bfloat16).to(cuda_device)
    out = attend("decode", q, pool, n, SCALE, num_ctas=num_ctas)
    want, a = orc.attention(q, kr, vr, SCALE)
    check_relative(out, want, a, vr, DECODE)


@pytest.mark.parametrize("ctx,kvh,most", [([40000, 0, 1, 10, 0], 1, 33), ([3, 9, 0, 20000] + [1] * 60, 2, 2 * 33),
                                          ([20000, 20000, 5], 1, 2 * 33 + 1)])
def test_a_long_sequence_among_short_ones_has_few_pieces(cuda_device, ctx, kvh, most):
    """A pair's pieces are read one after another by the CTA that joins them: about 32 at most, however many short and
    empty sequences come with it. Pieces (csrc/fp4_decode.cu): float4 (product, sum, factor) by CTA, end and head."""
    h, ctas = 2 * kvh, 148
    ws = workspace(cuda_device, h, kvh, ctas)
    decode_case(cuda_device, ctx, h, kvh, 64, seed=len(ctx), num_ctas=ctas, ws=ws)
    sums = ws[4352:4352 + ctas * 2 * 2 * 16].view(torch.float32).view(ctas, 2, 2, 4)[..., 1]
    assert 2 < int((sums[:, :, 0] > 0).sum()) <= most


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 17, 2 ** 31 - 33])
def test_the_longest_context_that_the_range_takes(cuda_device, n):
    """A table of the most columns that the entry point takes (2^31 - 16 tokens), all of them one block: the mean of
    that block's V (keys of zeros), for the longest contexts and one beyond, which is cut to the table's length."""
    dev, width = cuda_device, (2 ** 31 - 16) // 16
    _, v = random_rows(16, 1, 3, spread=False)
    pool, _, vr = pool_of(dev, torch.zeros_like(v), v, 16)
    q = torch.randn(1, 1, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    out = torch.full_like(q, float("nan"))
    ws = workspace(dev, 1, 1)
    ops_fp4.paged_decode_fp4(out, q, pool, torch.zeros(1, width, dtype=torch.int32, device=dev),
                             torch.tensor([n], dtype=torch.int32, device=dev), SCALE, ws)
    assert int(ws[:4].view(torch.int32).item()) == (8 if n > 16 * width else 0)
    # The weights are all the same: what rounds are fp32's sums over a warp's 2^26 / (148 * 16) tiles, and the output. A
    # tile adds two products to O, each off by up to 2^-23 of it (matrix sums may be cut off, not rounded), and twice
    # to the sum of weights, each off by up to 2^-24 of it.
    want, mean = vr.mean(0, keepdim=True), vr.abs().mean(0, keepdim=True)
    tol = want.abs() * 2.0 ** -8 + mean * (2 ** 26 / (148 * 16) * 2 * (2.0 ** -23 + 2.0 ** -24))
    assert bool(((out.double() - want).abs() <= tol).all())


def test_prefill_lengths_beyond_the_table(cuda_device):
    """A length past the table's is cut to it, whatever it is, so that the work is bounded; one below 0 sees nothing."""
    dev, h, m, bs = cuda_device, 4, 40, 32
    k, v = random_rows(3 * bs, 2, 5, spread=False)
    pool, kr, vr = pool_of(dev, k, v, bs)
    q = torch.randn(2 * m, h, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    table = torch.arange(3, dtype=torch.int32, device=dev).expand(2, 3).contiguous()
    cu = torch.tensor([0, m, 2 * m], dtype=torch.int32, device=dev)
    for long, negative in ((2 ** 31 - 1, -2 ** 31), (3 * bs + 1, -1)):
        out = torch.full_like(q, float("nan"))
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        ops_fp4.paged_prefill_fp4(out, q, pool, table, cu, torch.tensor([long, negative], dtype=torch.int32, device=dev),
                                  m, SCALE, error_word=err)
        assert int(err.item()) == 8
        want, a = orc.attention(q[:m], kr, vr, SCALE)
        check(out[:m], want, a, vr, PREFILL)
        assert not out[m:].any()


@pytest.mark.parametrize("m,cached,h", [(300, 100, 4), (40, 0, 3), (257, 0, 2), (1, 90, 4)])
def test_prefill_nan_rows_reach_only_the_queries_that_see_them(cuda_device, m, cached, h):
    """Rows of NaN in V (some groups of them) and in K: a query before such a row comes out as without it, one that
    sees it is NaN in the row's groups, or everywhere for K."""
    dev, kvh, bs = cuda_device, 1, 32
    n = m + cached
    k, v = random_rows(n, kvh, 41, spread=False)
    pool, kr, vr = pool_of(dev, k, v, bs)
    q = torch.randn(m, h, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    want, a = orc.attention(q, kr, vr, SCALE)
    spoilt = sorted({n - 1, cached + m // 2, cached + m // 3, min(cached + m // 2 + 1, n - 1), cached // 2})
    for i, j in enumerate(spoilt):  # V: groups i and i + 2
        row, rest = v[j:j + 1].clone(), vr[j].clone()
        for grp in (i, i + 2):
            row[:, :, 16 * grp + 3 * i] = float("nan")
        ops_fp4.kv_append_fp4(pool, k[j:j + 1].to(dev), row.to(dev), torch.tensor([j], device=dev))
    out = attend("prefill", q, pool, n, SCALE)
    bad = torch.zeros(m, h, 8, 16, dtype=torch.bool, device=dev)
    seen = cached + torch.arange(m, device=dev)  # the last key of each query
    for i, j in enumerate(spoilt):
        bad[seen >= j, :, i] = bad[seen >= j, :, i + 2] = True
    bad = bad.view(m, h, D)
    assert torch.equal(torch.isnan(out), bad)
    fine = torch.where(bad, torch.zeros_like(want), want)
    check(torch.where(bad, torch.zeros_like(out), out), fine, a, vr, PREFILL)
    j = cached + m // 2
    row = k[j:j + 1].clone()
    row[:, :, 77] = float("nan")
    ops_fp4.kv_append_fp4(pool, row.to(dev), v[j:j + 1].to(dev), torch.tensor([j], device=dev))
    out = attend("prefill", q, pool, n, SCALE)
    assert bool(torch.isnan(out[seen >= j]).all()) and not torch.isnan(out[(seen < j) & (seen < min(spoilt))]).any()
