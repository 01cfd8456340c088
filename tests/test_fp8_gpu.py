"""The 8-bit KV pool's kernels against the restatement in oracle/fp8_oracle.py.

Append and read are compared bit for bit. Attention is compared with 64-bit
arithmetic over the values that the codes stand for; its tolerance counts the
roundings on the way (relative half steps: bf16 2^-8, fp16 2^-11):

* the output's own, 2^-8 |o|;
* the weights', held in fp16 (decode) or bf16 (prefill), of the weighted mean
  of |v|, A;
* scores: sums of 128 products in fp32 (in the tests' range below 2^7 in log2
  units, so within 2^-14 of them after 128 roundings of 2^-24 relative to the
  sum of magnitudes), the exponential's 2^-22, fp16's floor for entries of q
  far below the row's largest: together below 2^-12 of a weight, so 2^-11 A
  with the denominator's share;
* decode: fp16's smallest step, 2^-24: a weight times its unit's power of two is
  off by half of it where the largest such product is held as at least 2^12, so
  by 2^-37 of that one's; the codes it multiplies are below 448, and 448 times
  the power of two is below twice the unit's largest |v|.
"""

import numpy as np
import pytest
import torch

from nano_vllm_ascend_b200 import ops_fp8
from oracle import fp4_oracle, fp8_oracle as orc
from tests.helpers import seeded_tables

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5
DECODE = dict(per_a=2.0 ** -11 + 2.0 ** -11, step=2.0 ** -37)
PREFILL = dict(per_a=2.0 ** -8 + 2.0 ** -11, step=0.0)


def check(got, want, a, n, vmax, how, what=""):
    """``want`` and ``a`` from the restatement, ``n`` keys, ``vmax`` the pool's largest |v|."""
    err = (got.double() - want).abs()
    tol = want.abs() * 2.0 ** -8 + a * how["per_a"] + n * how["step"] * 2 * vmax + 1e-30
    assert bool((err <= tol).all()), f"{what}: off by up to {float((err / tol).max()):.2f} tolerances"
    assert not torch.isnan(got).any()


def random_rows(tokens, kvh, seed, dtype=torch.bfloat16, spread=6):
    """K and V rows of magnitudes that differ by up to 2^spread."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, tokens, kvh, D, generator=g)
    x = x * torch.exp2(torch.rand(2, tokens, kvh, 1, generator=g) * spread - spread / 2)
    x = x.to(dtype)
    return x[0], x[1]


def make_pool(dev, nb, bs, kvh, seed, spread=0, mul=1.0):
    """A pool with every slot written (through the kernel), and its rows in float64."""
    k, v = random_rows(nb * bs, kvh, seed, spread=spread)
    pool = torch.zeros(ops_fp8.pool_shape(nb, bs, kvh), dtype=torch.uint8, device=dev)
    every = torch.arange(nb * bs, device=dev)
    ops_fp8.kv_append_fp8(pool, (k * mul).to(dev), (v * mul).to(dev), every)
    kr, vr = ops_fp8.kv_read_fp8(pool, every)
    return pool, kr.double(), vr.double()


def workspace(dev, h, kvh, num_ctas=0):
    return torch.zeros(ops_fp8.decode_fp8_workspace_bytes(h, kvh, D, num_ctas), dtype=torch.uint8, device=dev)


def seq_slots(table, n, bs, dev):
    i = torch.arange(n, device=dev)
    return table.to(dev).long()[i // bs] * bs + i % bs


# ------------------------------------------------------ append and read ---
def append_both(dev, want, pool, k, v, slots, err=None):
    """One call on the kernel and on the restatement; compares the whole pool."""
    ops_fp8.kv_append_fp8(pool, k, v, slots.to(dev), error_word=err)
    orc.append(want, k.cpu().float().numpy(), v.cpu().float().numpy(), slots.cpu().numpy())
    got = pool.cpu().numpy()
    if not np.array_equal(got, want):
        at = tuple(np.argwhere(got != want)[0])
        raise AssertionError(f"byte {at}: {got[at]} and {want[at]} ({int((got != want).sum())} differ)")


@pytest.mark.parametrize("tokens,kvh,bs,dtype", [
    (1, 1, 16, torch.bfloat16), (32, 8, 128, torch.bfloat16), (77, 3, 32, torch.float16),
    (256, 2, 64, torch.bfloat16), (257, 2, 64, torch.bfloat16), (512, 1, 16, torch.float16),
    (513, 1, 256, torch.bfloat16), (1500, 2, 256, torch.float16), (4097, 1, 16, torch.bfloat16)])
def test_append_and_read_are_exact(cuda_device, tokens, kvh, bs, dtype):
    """Rows into scattered slots, twice, so that units are partly written, raised and started anew."""
    dev = cuda_device
    nb = -(-tokens // bs) * 2 + 2
    want = np.zeros(ops_fp8.pool_shape(nb, bs, kvh), dtype=np.uint8)
    pool = torch.from_numpy(want.copy()).to(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    for step in range(3):
        k, v = random_rows(tokens, kvh, tokens + step, dtype)
        slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(step))[:tokens]
        append_both(dev, want, pool, k.to(dev), v.to(dev), slots, err)
    every = torch.randint(0, nb * bs, (tokens,), generator=torch.Generator().manual_seed(9))
    kr, vr = ops_fp8.kv_read_fp8(pool, every.to(dev), dtype=dtype, error_word=err)
    for got, ref in zip((kr, vr), orc.rows(want)):
        assert np.array_equal(got.cpu().double().numpy(), ref[every.numpy()])
    assert int(err.item()) == 0


def test_append_token_by_token_and_in_pieces(cuda_device):
    """A sequence grown token by token, in pieces of any length and in one call: the same rows where no exponent moved,
    and the restatement's bytes each time."""
    dev = cuda_device
    bs, kvh, n = 32, 2, 75
    k, v = random_rows(n, kvh, 5, spread=8)
    table = torch.tensor([3, 0, 2])
    slots = (table[torch.arange(n) // bs] * bs + torch.arange(n) % bs)
    for pieces in ([1] * n, [7, 1, 20, 16, 31], [n]):
        want = np.full(ops_fp8.pool_shape(4, bs, kvh), 0x55, dtype=np.uint8)  # an earlier sequence's bytes
        want[..., 4096:] = 0
        pool = torch.from_numpy(want.copy()).to(dev)
        at = 0
        for m in pieces:
            append_both(dev, want, pool, k[at:at + m].to(dev), v[at:at + m].to(dev), slots[at:at + m])
            at += m


def test_append_borders_of_codes_and_exponents(cuda_device):
    """Ties of every code, amax at and next to the borders of the exponents, the range's ends, zeros of both signs."""
    dev = cuda_device
    bf = torch.bfloat16
    rows = []
    mags = torch.tensor([(m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)
                         if (e, m) != (15, 7)])
    mid = (mags[1:] + mags[:-1]) / 2
    for d in (-1, 0, 1):
        x = mid.to(bf).float()
        x = x + d * torch.exp2(torch.floor(torch.log2(x)) - 7)
        row = torch.zeros(D)
        row[:126] = x
        row[126], row[127] = 448.0, -448.0
        rows.append([row, -row])
    for top in (448.0, 450.0, 446.0, 256.0, 255.0, 2.0 ** -31 * 448, 2.0 ** -32 * 450, 2.0 ** -60, 1e-38, 2.0 ** 48,
                448 * 2.0 ** 40, 450 * 2.0 ** 40, 3e38):
        row = torch.linspace(-1, 1, D) * top
        rows.append([row, torch.zeros(D)])
    rows.append([torch.zeros(D), torch.full((D,), -0.0)])
    n = len(rows)
    want = np.zeros(ops_fp8.pool_shape(n, 16, 1), dtype=np.uint8)
    pool = torch.from_numpy(want.copy()).to(dev)
    x = torch.stack([torch.stack(r) for r in rows]).to(bf)  # two rows a unit
    slots = (torch.arange(n)[:, None] * 16 + torch.arange(2)).reshape(-1)
    x = x.view(-1, 1, D).to(dev)
    append_both(dev, want, pool, x, x.flip(0).contiguous(), slots)
    # and onto those units, so that their rows move to other exponents
    y = (x.float() * torch.exp2(torch.arange(2 * n, device=dev) % 9 - 3.0)[:, None, None]).to(bf)
    append_both(dev, want, pool, y, y, slots + 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_of_infinities_and_nan(cuda_device, dtype):
    dev = cuda_device
    k, v = random_rows(40, 2, 3, dtype)
    inf, nan = float("inf"), float("nan")
    k[3, 0, 7], k[3, 0, 9], k[5, 1, 127], k[20, 0, 0] = inf, -inf, nan, nan
    k[20, 1, :] = inf  # nothing finite in the row, and in the unit below nothing at all
    v[32:, 0, :] = inf
    v[39, 1, 64] = -nan
    want = np.zeros(ops_fp8.pool_shape(3, 16, 2), dtype=np.uint8)
    pool = torch.from_numpy(want.copy()).to(dev)
    append_both(dev, want, pool, k.to(dev), v.to(dev), torch.arange(40))
    append_both(dev, want, pool, k[:3].to(dev) * 64, v[:3].to(dev) * 64, torch.arange(40, 43))  # NaN rows move along
    kr, vr = ops_fp8.kv_read_fp8(pool, torch.arange(48, device=dev), dtype=dtype)
    assert torch.isnan(kr[5, 1]).all() and torch.isnan(kr[20, 0]).all() and torch.isnan(vr[39, 1]).all()
    assert int(torch.isnan(kr).sum()) == 2 * D and int(torch.isnan(vr).sum()) == D


@pytest.mark.parametrize("tokens", [40, 700])
@pytest.mark.parametrize("shift,gap", [(0, 0), (1, 1), (2, 3), (8, 8), (4, 40)])
def test_append_of_strided_and_unaligned_rows(cuda_device, tokens, shift, gap):
    dev = cuda_device
    kvh, bs = 2, 16
    k, v = random_rows(tokens, kvh, 5)
    nb = -(-tokens // bs) + 1
    want = np.zeros(ops_fp8.pool_shape(nb, bs, kvh), dtype=np.uint8)
    pool = torch.from_numpy(want.copy()).to(dev)
    row = kvh * D + gap

    def strided(x):
        buf = torch.full((shift + tokens * row,), float("nan"), dtype=x.dtype, device=dev)
        view = torch.as_strided(buf, (tokens, kvh, D), (row, D, 1), shift)
        view.copy_(x.to(dev))
        return view

    append_both(dev, want, pool, strided(k), strided(v), torch.arange(tokens) + 7)


@pytest.mark.parametrize("tokens", [20, 600])
def test_append_skips_and_flags_bad_slots(cuda_device, tokens):
    dev = cuda_device
    nb, bs, kvh = 40, 16, 1
    k, v = random_rows(tokens, kvh, 2)
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(1))[:tokens]
    slots[1], slots[7], slots[11], slots[13] = -1, nb * bs, 1 << 40, -(1 << 62)
    want = np.zeros(ops_fp8.pool_shape(nb, bs, kvh), dtype=np.uint8)
    pool = torch.from_numpy(want.copy()).to(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    append_both(dev, want, pool, k.to(dev), v.to(dev), slots, err)
    assert int(err.item()) == 4
    err.zero_()
    kr, vr = ops_fp8.kv_read_fp8(pool, slots.to(dev), error_word=err)
    assert int(err.item()) == 4 and not kr[[1, 7, 11, 13]].any() and not vr[[1, 7, 11, 13]].any()
    assert not torch.equal(kr[0], torch.zeros_like(kr[0]))


@pytest.mark.parametrize("tokens", [8, 600])
def test_append_of_one_slot_given_twice_writes_one_of_the_rows(cuda_device, tokens):
    dev = cuda_device
    k, v = random_rows(tokens, 2, 2)
    slots = torch.arange(tokens) + 1
    slots[5] = slots[2]
    results = []
    for keep in (2, 5):
        ref = np.zeros(ops_fp8.pool_shape(40, 16, 2), dtype=np.uint8)
        sel = torch.tensor([i for i in range(tokens) if i != 7 - keep])
        orc.append(ref, k[sel].float().numpy(), v[sel].float().numpy(), slots[sel].numpy())
        results.append(ref)
    pool = torch.zeros(ops_fp8.pool_shape(40, 16, 2), dtype=torch.uint8, device=dev)
    ops_fp8.kv_append_fp8(pool, k.to(dev), v.to(dev), slots.to(dev))
    got = pool.cpu().numpy()
    assert any(np.array_equal(got, r) for r in results)


def test_append_and_read_of_nothing(cuda_device):
    dev = cuda_device
    pool = torch.zeros(ops_fp8.pool_shape(1, 16, 2), dtype=torch.uint8, device=dev)
    none = torch.empty(0, 2, D, dtype=torch.bfloat16, device=dev)
    slots = torch.empty(0, dtype=torch.int64, device=dev)
    ops_fp8.kv_append_fp8(pool, none, none, slots)
    k, v = ops_fp8.kv_read_fp8(pool, slots)
    assert k.shape == v.shape == (0, 2, D)


def test_append_in_a_graph_with_slots_that_change(cuda_device):
    """Captured calls, short and long, replayed on other slots; and two streams at once over two layers."""
    dev = cuda_device
    for tokens in (32, 900):
        kvh, bs, nb = 2, 16, 80
        k, v = (t.to(dev) for t in random_rows(tokens, kvh, 4))
        slots = torch.arange(tokens, device=dev)
        pool = torch.zeros(ops_fp8.pool_shape(nb, bs, kvh), dtype=torch.uint8, device=dev)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            ops_fp8.kv_append_fp8(pool, k, v, slots)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops_fp8.kv_append_fp8(pool, k, v, slots)
        want = np.zeros(ops_fp8.pool_shape(nb, bs, kvh), dtype=np.uint8)
        pool.zero_()
        for seed in range(3):
            new = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(seed))[:tokens]
            slots.copy_(new)
            graph.replay()
            orc.append(want, k.cpu().float().numpy(), v.cpu().float().numpy(), new.numpy())
        assert np.array_equal(pool.cpu().numpy(), want)


def test_appends_on_two_streams(cuda_device):
    dev = cuda_device
    tokens, kvh, bs, nb = 1000, 4, 16, 80
    streams, pools, wants, calls = [torch.cuda.Stream() for _ in range(2)], [], [], []
    for i in range(2):
        k, v = random_rows(tokens, kvh, i)
        slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(i))[:tokens]
        want = np.zeros(ops_fp8.pool_shape(nb, bs, kvh), dtype=np.uint8)
        pools.append(torch.from_numpy(want.copy()).to(dev))
        for _ in range(2):
            orc.append(want, k.float().numpy(), v.float().numpy(), slots.numpy())
        wants.append(want)
        calls.append((k.to(dev), v.to(dev), slots.to(dev)))
    torch.cuda.synchronize()
    for _ in range(2):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                ops_fp8.kv_append_fp8(pools[i], *calls[i])
    torch.cuda.synchronize()
    for pool, want in zip(pools, wants):
        assert np.array_equal(pool.cpu().numpy(), want)


# ----------------------------------------------------------------- decode ---
def decode_case(dev, ctx, h, kvh, bs, seed=0, num_ctas=0, q_mul=1.0, spread=2, ws=None, mul=1.0, scale=SCALE):
    nb = sum(-(-n // bs) for n in ctx) + 2
    pool, kr, vr = make_pool(dev, nb, bs, kvh, seed, spread, mul)
    tables = seeded_tables(ctx, bs, nb, seed)
    q = (torch.randn(len(ctx), h, D, generator=torch.Generator().manual_seed(seed + 1)) * q_mul).to(torch.bfloat16)
    q = q.to(dev)
    out = torch.full_like(q, float("nan"))
    ws = workspace(dev, h, kvh, num_ctas) if ws is None else ws
    lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
    ops_fp8.paged_decode_fp8(out, q, pool, tables.to(dev), lens, scale, ws, num_ctas)
    assert int(ws[:4].view(torch.int32).item()) == 0
    assert not ws[256:4096].any(), "the tickets must be back at zero"
    for b, n in enumerate(ctx):
        sl = seq_slots(tables[b], n, bs, dev)
        want, a = fp4_oracle.attention(q[b:b + 1], kr[sl], vr[sl], scale)
        check(out[b:b + 1], want, a, n, float(vr.abs().max()), DECODE, f"sequence {b} of {n} tokens")
    return pool, tables, q, out


@pytest.mark.parametrize("h,kvh", [(1, 1), (2, 1), (3, 1), (8, 2), (10, 2), (6, 1), (21, 3), (16, 2), (16, 8)])
def test_decode_groups(cuda_device, h, kvh):
    decode_case(cuda_device, [1, 16, 100, 0, 257], h, kvh, 32, seed=h)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_decode_lengths_at_block_and_unit_borders(cuda_device, bs):
    ctx = [1, 2, 15, 16, 17, 31, 32, 33, bs - 1, bs, bs + 1, 2 * bs, 0, 0, 3 * bs + 5, 777]
    decode_case(cuda_device, ctx, 4, 2, bs, seed=bs)


@pytest.mark.parametrize("num_ctas", [1, 2, 7, 148, 600])
@pytest.mark.parametrize("ctx", [[5000], [3000, 1, 700, 0, 45], [16] * 40])
def test_decode_split_over_ctas(cuda_device, num_ctas, ctx):
    decode_case(cuda_device, ctx, 8, 2, 64, seed=7, num_ctas=num_ctas)


def test_decode_scores_that_climb_and_units_of_any_exponent(cuda_device):
    decode_case(cuda_device, [900, 63], 4, 1, 32, seed=1, q_mul=8.0)
    decode_case(cuda_device, [900, 63], 4, 1, 32, seed=2, q_mul=2.0 ** -40)
    decode_case(cuda_device, [300, 63], 4, 1, 32, seed=3, q_mul=2.0 ** -6, spread=16)
    decode_case(cuda_device, [300, 63], 4, 1, 32, seed=4, q_mul=2.0 ** 30, mul=2.0 ** -30)
    decode_case(cuda_device, [300, 63], 4, 1, 32, seed=5, q_mul=2.0 ** -30, mul=2.0 ** 30)


def test_decode_many_sequences(cuda_device):
    """More sequences than one launch takes."""
    g = torch.Generator().manual_seed(1)
    decode_case(cuda_device, torch.randint(0, 40, (1100,), generator=g).tolist(), 2, 1, 16, seed=5)


def test_decode_empty_batch_and_only_empty_sequences(cuda_device):
    dev = cuda_device
    decode_case(dev, [0, 0, 0], 4, 2, 16)
    pool = torch.zeros(ops_fp8.pool_shape(1, 16, 2), dtype=torch.uint8, device=dev)
    q = torch.empty(0, 4, D, dtype=torch.bfloat16, device=dev)
    ops_fp8.paged_decode_fp8(q, q, pool, torch.zeros(0, 1, dtype=torch.int32, device=dev),
                             torch.zeros(0, dtype=torch.int32, device=dev), SCALE, workspace(dev, 4, 2))


def test_decode_over_rows_never_written_attends_over_zeros(cuda_device):
    dev = cuda_device
    pool = torch.zeros(ops_fp8.pool_shape(3, 16, 1), dtype=torch.uint8, device=dev)
    k, v = random_rows(16, 1, 1)
    ops_fp8.kv_append_fp8(pool, k.to(dev), v.to(dev), torch.arange(16, device=dev))
    kr, vr = (t.double() for t in ops_fp8.kv_read_fp8(pool, torch.arange(48, device=dev)))
    q = torch.randn(1, 2, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    out = torch.empty_like(q)
    ops_fp8.paged_decode_fp8(out, q, pool, torch.tensor([[1, 0, 2]], dtype=torch.int32, device=dev),
                             torch.tensor([45], dtype=torch.int32, device=dev), SCALE, workspace(dev, 2, 1))
    want, a = fp4_oracle.attention(q, kr[:45], vr[:45], SCALE)
    check(out, want, a, 45, float(vr.abs().max()), DECODE)


@pytest.mark.parametrize("tail", [-6, -20, -26])
@pytest.mark.parametrize("vexp", [0, 30, -30])
def test_decode_tail_of_small_weights_beside_other_exponents(cuda_device, tail, vexp):
    """20000 tokens of weight 2^tail each beside one of weight 1, V of the tail 2^vexp times as large: what the tail
    gives is there, however the units' exponents differ."""
    dev = cuda_device
    n = 20000
    nb = -(-n // 256) + 1
    k = torch.zeros(n, 1, D)
    v = torch.randn(n, 1, D, generator=torch.Generator().manual_seed(1)).abs() * 2.0 ** vexp
    k[:, 0, 0] = tail
    k[0, 0, 0] = 0.0
    v[0] = 1.0
    for first in (0, n - 16):  # the heavy token first, and last, in a unit of its own
        kk, vv = k.clone(), v.clone()
        if first:
            kk[0], kk[first], vv[0], vv[first] = k[1], k[0], v[1], v[0]
        unit = torch.arange(n) // 16 == first // 16
        unit[first] = False
        vv[unit] = 0  # the heavy token's unit holds nothing else
        pool = torch.zeros(ops_fp8.pool_shape(nb, 256, 1), dtype=torch.uint8, device=dev)
        ops_fp8.kv_append_fp8(pool, kk.to(torch.bfloat16).to(dev), vv.to(torch.bfloat16).to(dev),
                              torch.arange(n, device=dev))
        kr, vr = (t.double() for t in ops_fp8.kv_read_fp8(pool, torch.arange(n, device=dev)))
        q = torch.zeros(1, 1, D, dtype=torch.bfloat16, device=dev)
        q[0, 0, 0] = 1.0
        out = torch.empty_like(q)
        scale = float(np.log(2.0))  # scores in log2 units are k's
        table = torch.arange(nb, dtype=torch.int32, device=dev)[None]
        ops_fp8.paged_decode_fp8(out, q, pool, table, torch.tensor([n], dtype=torch.int32, device=dev), scale,
                                 workspace(dev, 1, 1))
        want, a = fp4_oracle.attention(q, kr, vr, scale)
        # every weight is a power of two within fp16's normal range beside the largest product, or 2^-37 of it off
        err = (out.double() - want).abs()
        tol = want.abs() * 2.0 ** -8 + a * (2.0 ** -10) + 2 * n * 2.0 ** -37 * (vr.abs() * torch.exp2(kr[:, :, :1])).max()
        assert bool((err <= tol).all()), float((err / tol).max())
        assert bool((err <= want.abs() * 0.02).all()), float((err / want.abs()).max())


def test_decode_scores_of_any_magnitude(cuda_device):
    """Products of 2^10 to 2^60: weights go by differences, so that they hold."""
    dev = cuda_device
    for up in (10, 24, 40, 60):
        k = torch.zeros(48, 1, D)
        k[:, 0, 0] = 1.0
        k[:, 0, 1] = torch.arange(48).float() / 16 * 2.0 ** -2
        v = torch.randn(48, 1, D, generator=torch.Generator().manual_seed(up))
        pool = torch.zeros(ops_fp8.pool_shape(3, 16, 1), dtype=torch.uint8, device=dev)
        ops_fp8.kv_append_fp8(pool, k.to(torch.bfloat16).to(dev), v.to(torch.bfloat16).to(dev),
                              torch.arange(48, device=dev))
        kr, vr = (t.double() for t in ops_fp8.kv_read_fp8(pool, torch.arange(48, device=dev)))
        q = torch.zeros(1, 1, D, dtype=torch.bfloat16, device=dev)
        q[0, 0, 0] = 2.0 ** up
        q[0, 0, 1] = 4.0 if up < 20 else 2.0 ** (up - 17)  # so that the sum of both products is exact in fp32
        out = torch.empty_like(q)
        ops_fp8.paged_decode_fp8(out, q, pool, torch.arange(3, dtype=torch.int32, device=dev)[None],
                                 torch.tensor([48], dtype=torch.int32, device=dev), 1.0, workspace(dev, 1, 1))
        want, a = fp4_oracle.attention(q, kr, vr, 1.0)
        check(out, want, a, 48, float(vr.abs().max()), DECODE, f"2^{up}")


def test_decode_ignores_what_lies_behind_the_context(cuda_device):
    """NaN rows behind the last token, wild ids in unused table columns, a strided table."""
    dev = cuda_device
    ctx, h, kvh, bs = [5, 18, 40], 4, 2, 16
    pool, tables, q, out = decode_case(dev, ctx, h, kvh, bs, seed=9)
    before = out.clone()
    nan = torch.full((1, kvh, D), float("nan"), dtype=torch.bfloat16, device=dev)
    for b, n in enumerate(ctx):
        for i in range(n, -(-n // bs) * bs):
            slot = torch.tensor([int(tables[b, i // bs]) * bs + i % bs], device=dev)
            ops_fp8.kv_append_fp8(pool, nan, nan, slot)
    wide = torch.full((3, 11), -12345, dtype=torch.int32)
    for b, n in enumerate(ctx):
        wide[b, :-(-n // bs)] = tables[b, :-(-n // bs)]
    view = wide.to(dev)[:, :7]
    ws = workspace(dev, h, kvh)
    ops_fp8.paged_decode_fp8(out, q, pool, view, torch.tensor(ctx, dtype=torch.int32, device=dev), SCALE, ws)
    assert torch.equal(out, before) and int(ws[:4].view(torch.int32).item()) == 0


def test_decode_propagates_a_nan_that_is_seen(cuda_device):
    dev = cuda_device
    ctx, h, kvh, bs = [40, 40], 4, 2, 16
    for which in (0, 1):
        pool, tables, q, out = decode_case(dev, ctx, h, kvh, bs, seed=9)
        before = out.clone()
        row = torch.zeros(1, kvh, D, dtype=torch.bfloat16, device=dev)
        row[0, 1, 5] = float("nan")  # KV head 1
        kv = [torch.zeros_like(row), torch.zeros_like(row)]
        kv[which] = row
        ops_fp8.kv_append_fp8(pool, *kv, torch.tensor([int(tables[0, 1]) * bs + 3], device=dev))
        ops_fp8.paged_decode_fp8(out, q, pool, tables.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev), SCALE,
                                 workspace(dev, h, kvh))
        nan = torch.isnan(out)
        assert nan[0, 2:].all() and int(nan.sum()) == 2 * D and torch.equal(out[1], before[1])


def test_decode_flags_bad_blocks_and_long_contexts(cuda_device):
    dev = cuda_device
    h, kvh, bs = 2, 1, 16
    pool, kr, vr = make_pool(dev, 4, bs, kvh, 3)
    q = torch.randn(2, h, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    out = torch.empty_like(q)
    ws = workspace(dev, h, kvh)
    tables = torch.tensor([[0, 4], [2, -1]], dtype=torch.int32, device=dev)
    ops_fp8.paged_decode_fp8(out, q, pool, tables, torch.tensor([20, 30], dtype=torch.int32, device=dev), SCALE, ws)
    assert int(ws[:4].view(torch.int32).item()) == 2
    vmax = float(vr.abs().max())
    for b, (blk, n) in enumerate(((0, 4), (2, 14))):  # the bad block's tokens count as rows of zeros
        k = torch.cat([kr[blk * bs:(blk + 1) * bs], torch.zeros(n, kvh, D, device=dev, dtype=torch.float64)])
        v = torch.cat([vr[blk * bs:(blk + 1) * bs], torch.zeros(n, kvh, D, device=dev, dtype=torch.float64)])
        want, a = fp4_oracle.attention(q[b:b + 1], k, v, SCALE)
        check(out[b:b + 1], want, a, v.shape[0], vmax, DECODE)
    ws.zero_()
    word = torch.zeros(1, dtype=torch.int32, device=dev)
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    ops_fp8.paged_decode_fp8(out, q, pool, tables, torch.tensor([33, -5], dtype=torch.int32, device=dev), SCALE, ws,
                             error_word=word)
    assert int(word.item()) == 8 and int(ws[:4].view(torch.int32).item()) == 0
    want, a = fp4_oracle.attention(q[:1], kr[:32], vr[:32], SCALE)
    check(out[:1], want, a, 32, vmax, DECODE)
    assert not out[1].any()


def test_decode_one_workspace_for_many_shapes(cuda_device):
    dev = cuda_device
    ws = workspace(dev, 64, 8)
    for i, (ctx, h, kvh) in enumerate([([3000], 16, 8), ([5, 900], 8, 1), ([1] * 50, 4, 4), ([2000, 2000], 64, 8)]):
        decode_case(dev, ctx, h, kvh, 32, seed=i, ws=ws)


def test_decode_repeats_bit_for_bit_and_in_a_graph(cuda_device):
    dev = cuda_device
    ctx, h, kvh, bs = [3000, 17, 0, 1290], 16, 2, 64
    pool, tables, q, out = decode_case(dev, ctx, h, kvh, bs, seed=2)
    ws, lens, tab = workspace(dev, h, kvh), torch.tensor(ctx, dtype=torch.int32, device=dev), tables.to(dev)
    again = torch.empty_like(out)
    for _ in range(3):
        again.fill_(7.0)
        ops_fp8.paged_decode_fp8(again, q, pool, tab, lens, SCALE, ws)
        assert torch.equal(again, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops_fp8.paged_decode_fp8(again, q, pool, tab, lens, SCALE, ws)
    for n in ([3000, 17, 0, 1290], [1, 16, 0, 64]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        eager = torch.empty_like(out)
        ops_fp8.paged_decode_fp8(eager, q, pool, tab, lens, SCALE, ws)
        assert torch.equal(again, eager)


def test_far_offsets(cuda_device):
    """A pool whose last blocks lie past 4 GiB."""
    dev = cuda_device
    kvh, bs, h = 8, 256, 8
    nb = (4 << 30) // (kvh * bs // 16 * 4128) + 40
    pool = torch.zeros(ops_fp8.pool_shape(nb, bs, kvh), dtype=torch.uint8, device=dev)
    n = 600
    k, v = random_rows(n, kvh, 4, spread=0)
    table = torch.tensor([[nb - 1, nb - 20, nb - 7]], dtype=torch.int32)
    slots = seq_slots(table[0], n, bs, dev)
    ops_fp8.kv_append_fp8(pool, k.to(dev), v.to(dev), slots)
    kr, vr = ops_fp8.kv_read_fp8(pool, slots)
    ref = np.zeros(ops_fp8.pool_shape(3, bs, kvh), dtype=np.uint8)
    orc.append(ref, k.float().numpy(), v.float().numpy(), np.arange(n))
    for got, want in zip((kr, vr), orc.rows(ref)):
        assert np.array_equal(got.cpu().double().numpy(), want[:n])
    q = torch.randn(1, h, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(dev)
    want, a = fp4_oracle.attention(q, kr.double(), vr.double(), SCALE)
    out = torch.empty_like(q)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    ops_fp8.paged_decode_fp8(out, q, pool, table.to(dev), lens, SCALE, workspace(dev, h, kvh))
    check(out, want, a, n, float(vr.abs().max()), DECODE)
    out.fill_(0)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    ops_fp8.paged_prefill_fp8(out, q, pool, table.to(dev), cu, lens, 1, SCALE)
    check(out, want, a, n, float(vr.abs().max()), PREFILL)


# ---------------------------------------------------------------- prefill ---
def prefill_case(dev, q_lens, cached, h, kvh, bs, seed=0, q_mul=1.0, spread=2, mul=1.0):
    kv = [a + b for a, b in zip(q_lens, cached)]
    nb = sum(-(-n // bs) for n in kv) + 2
    pool, kr, vr = make_pool(dev, nb, bs, kvh, seed, spread, mul)
    tables = seeded_tables(kv, bs, nb, seed)
    total = sum(q_lens)
    q = (torch.randn(total, h, D, generator=torch.Generator().manual_seed(seed + 1)) * q_mul).to(torch.bfloat16).to(dev)
    out = torch.full_like(q, float("nan"))
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32).to(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    lens = torch.tensor(kv, dtype=torch.int32, device=dev)
    ops_fp8.paged_prefill_fp8(out, q, pool, tables.to(dev), cu, lens, max(q_lens), SCALE, error_word=err)
    assert int(err.item()) == 0
    at = 0
    for b, (m, n) in enumerate(zip(q_lens, kv)):
        sl = seq_slots(tables[b], n, bs, dev)
        want, a = fp4_oracle.attention(q[at:at + m], kr[sl], vr[sl], SCALE)
        check(out[at:at + m], want, a, n, float(vr.abs().max()), PREFILL, f"sequence {b}: {m} over {n}")
        at += m
    return pool, tables, q, cu, lens, out


@pytest.mark.parametrize("h,kvh", [(1, 1), (2, 1), (3, 1), (9, 3), (4, 1), (10, 2), (16, 8), (12, 1)])
def test_prefill_groups(cuda_device, h, kvh):
    prefill_case(cuda_device, [1, 130, 64], [0, 77, 256], h, kvh, 64, seed=h)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_prefill_lengths_at_borders(cuda_device, bs):
    q = [1, 1, 127, 128, 129, 5, 300, 0, 16]
    c = [0, 127, 1, 128, 383, 250, 0, 40, 1000]
    prefill_case(cuda_device, q, c, 4, 2, bs, seed=bs)


def test_prefill_long(cuda_device):
    prefill_case(cuda_device, [1500, 900], [0, 2100], 4, 2, 128, seed=3)
    prefill_case(cuda_device, [40], [7000], 2, 1, 32, seed=4)


def test_prefill_scores_that_climb_and_units_of_any_exponent(cuda_device):
    prefill_case(cuda_device, [200], [100], 4, 1, 32, seed=5, q_mul=8.0)
    prefill_case(cuda_device, [200], [100], 4, 1, 32, seed=6, q_mul=2.0 ** -6, spread=16)
    prefill_case(cuda_device, [200], [100], 4, 1, 32, seed=7, q_mul=2.0 ** 30, mul=2.0 ** -30)
    prefill_case(cuda_device, [200], [100], 4, 1, 32, seed=8, q_mul=2.0 ** -30, mul=2.0 ** 30)


def test_prefill_many_items_per_cta(cuda_device):
    """More work items than CTAs, one and two query tiles each, with empty sequences between."""
    g = torch.Generator().manual_seed(3)
    q = torch.randint(0, 200, (60,), generator=g).tolist()
    c = torch.randint(0, 300, (60,), generator=g).tolist()
    prefill_case(cuda_device, q, c, 8, 2, 32, seed=8)


def test_prefill_rows_that_see_nothing_and_rows_behind_the_last(cuda_device):
    """Fewer keys than queries (the first rows see none and are zeros), no keys at all, and rows of the output behind
    the last sequence, which stay as they were."""
    dev = cuda_device
    h, kvh, bs = 4, 2, 16
    pool, kr, vr = make_pool(dev, 8, bs, kvh, 3)
    q_lens, kv = [40, 7, 130], [25, 0, 60]
    q = torch.randn(200, h, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    out = torch.full_like(q, 5.0)
    tables = torch.tensor([[1, 0, 9, 9], [9, 9, 9, 9], [2, 3, 7, 5]], dtype=torch.int32)
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32).to(dev)
    ops_fp8.paged_prefill_fp8(out, q, pool, tables.to(dev), cu, torch.tensor(kv, dtype=torch.int32, device=dev), 130,
                              SCALE)
    at = 0
    for b, (m, n) in enumerate(zip(q_lens, kv)):
        sl = seq_slots(tables[b], n, bs, dev)
        want, a = fp4_oracle.attention(q[at:at + m], kr[sl], vr[sl], SCALE)
        check(out[at:at + m], want, a, n, float(vr.abs().max()), PREFILL, f"sequence {b}")
        assert not out[at:at + m - n].any()
        at += m
    assert bool((out[at:] == 5.0).all())


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("token", [0, 70, 129, 199])
def test_prefill_nan_reaches_only_the_queries_that_see_it(cuda_device, which, token):
    dev = cuda_device
    h, kvh, bs, n = 4, 2, 16, 200
    pool, tables, q, cu, lens, out = prefill_case(dev, [n], [0], h, kvh, bs, seed=9)
    before = out.clone()
    row = torch.zeros(1, kvh, D, dtype=torch.bfloat16, device=dev)
    row[0, 1, 5] = float("nan")
    slot = int(tables[0, token // bs]) * bs + token % bs
    # the row's own byte pattern, so that the unit's other rows stay as they are
    unit = pool[slot // bs, 1, slot % bs // 16]
    at = 2048 * which + 128 * (slot % 16)
    unit[at:at + 128] = 0x7F
    ops_fp8.paged_prefill_fp8(out, q, pool, tables.to(dev), cu, lens, n, SCALE)
    nan = torch.isnan(out)
    assert nan[token:, 2:].all() and int(nan.sum()) == (n - token) * 2 * D
    clean = ~nan
    if which == 1:
        assert torch.equal(out[clean], before[clean])
    else:
        assert torch.equal(out[:, :2], before[:, :2]) and torch.equal(out[:token], before[:token])


def test_prefill_ignores_nan_behind_the_length(cuda_device):
    dev = cuda_device
    h, kvh, bs = 4, 2, 16
    pool, tables, q, cu, lens, out = prefill_case(dev, [21, 150], [0, 37], h, kvh, bs, seed=9)
    before = out.clone()
    for b, n in enumerate((21, 187)):
        last = int(tables[b, (n - 1) // bs])
        for i in range((n - 1) % bs + 1, bs):
            pool[last, :, 0, 128 * i:128 * i + 128] = 0x7F
            pool[last, :, 0, 2048 + 128 * i:2048 + 128 * i + 128] = 0xFF
    ops_fp8.paged_prefill_fp8(out, q, pool, tables.to(dev), cu, lens, 150, SCALE)
    assert torch.equal(out, before)


def test_prefill_flags_bad_blocks_and_lengths(cuda_device):
    dev = cuda_device
    h, kvh, bs = 2, 1, 16
    pool, kr, vr = make_pool(dev, 4, bs, kvh, 3)
    q = torch.randn(20, h, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    out = torch.empty_like(q)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    tables = torch.tensor([[0, 4], [2, -1]], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 10, 20], dtype=torch.int32, device=dev)
    ops_fp8.paged_prefill_fp8(out, q, pool, tables, cu, torch.tensor([20, 30], dtype=torch.int32, device=dev), 10, SCALE,
                              error_word=err)
    assert int(err.item()) == 2
    vmax = float(vr.abs().max())
    for b, (blk, n) in enumerate(((0, 4), (2, 14))):
        k = torch.cat([kr[blk * bs:(blk + 1) * bs], torch.zeros(n, kvh, D, device=dev, dtype=torch.float64)])
        v = torch.cat([vr[blk * bs:(blk + 1) * bs], torch.zeros(n, kvh, D, device=dev, dtype=torch.float64)])
        want, a = fp4_oracle.attention(q[10 * b:10 * b + 10], k, v, SCALE)
        check(out[10 * b:10 * b + 10], want, a, v.shape[0], vmax, PREFILL)
    err.zero_()
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    ops_fp8.paged_prefill_fp8(out, q, pool, tables, cu, torch.tensor([1 << 30, -5], dtype=torch.int32, device=dev), 10,
                              SCALE, error_word=err)
    assert int(err.item()) == 8
    want, a = fp4_oracle.attention(q[:10], kr[:32], vr[:32], SCALE)
    check(out[:10], want, a, 32, vmax, PREFILL)
    assert not out[10:].any()


# Few items: a cluster of CTAs shares an item's keys, 8 down to 2 of them by how many items there are.
@pytest.mark.parametrize("items", [1, 14, 20, 25, 30, 40, 60, 74])
def test_prefill_keys_over_clusters(cuda_device, items):
    """Ragged lengths of one to 20 tiles of keys, some sequences empty: parts of two tiles and more, and undivided ones."""
    g = torch.Generator().manual_seed(items)
    q = torch.randint(0, 129, (items,), generator=g).tolist()
    c = (torch.rand(items, generator=g) ** 2 * 2400).int().tolist()
    q[0], c[0] = 128, 2400
    prefill_case(cuda_device, q, c, 1, 1, 64, seed=items)


@pytest.mark.parametrize("cached", list(range(0, 1400, 128)) + [127, 383, 385, 511, 513, 900])
def test_prefill_keys_over_clusters_at_borders(cuda_device, cached):
    prefill_case(cuda_device, [128], [cached], 2, 1, 128, seed=cached)
    prefill_case(cuda_device, [1, 200], [cached, 1000], 3, 3, 16, seed=cached)


def test_prefill_parts_whose_scores_and_exponents_differ(cuda_device):
    for seed, kw in ((5, dict(q_mul=8.0)), (6, dict(q_mul=2.0 ** -6, spread=16)), (7, dict(q_mul=2.0 ** 30, mul=2.0 ** -30)),
                     (8, dict(q_mul=2.0 ** -30, mul=2.0 ** 30)), (9, dict(q_mul=16.0, spread=8))):
        prefill_case(cuda_device, [150], [1700], 4, 1, 32, seed=seed, **kw)


def test_prefill_parts_that_no_row_or_only_some_rows_see(cuda_device):
    """Fewer keys than queries, so that the first rows see none of the item's keys; the last tiles only the last rows."""
    dev, h, kvh, bs = cuda_device, 2, 1, 128
    pool, kr, vr = make_pool(dev, 10, bs, kvh, 3)
    q_lens, kv = [1100, 700], [1000, 700]
    q = torch.randn(1800, h, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    out = torch.full_like(q, 5.0)
    tables = torch.stack([torch.randperm(10, generator=torch.Generator().manual_seed(i))[:8] for i in range(2)]).int()
    cu = torch.tensor([0, 1100, 1800], dtype=torch.int32, device=dev)
    ops_fp8.paged_prefill_fp8(out, q, pool, tables.to(dev), cu, torch.tensor(kv, dtype=torch.int32, device=dev), 1100,
                              SCALE)
    for b, (at, m, n) in enumerate(((0, 1100, 1000), (1100, 700, 700))):
        sl = seq_slots(tables[b], n, bs, dev)
        want, a = fp4_oracle.attention(q[at:at + m], kr[sl], vr[sl], SCALE)
        check(out[at:at + m], want, a, n, float(vr.abs().max()), PREFILL, f"sequence {b}")
    assert not out[:100].any()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("token", [0, 129, 600, 1055, 1150])
def test_prefill_nan_in_any_part(cuda_device, which, token):
    dev, h, kvh, bs, m, n = cuda_device, 4, 2, 16, 160, 1160
    pool, tables, q, cu, lens, out = prefill_case(dev, [m], [n - m], h, kvh, bs, seed=9)
    before = out.clone()
    slot = int(tables[0, token // bs]) * bs + token % bs
    at = 2048 * which + 128 * (slot % 16)
    pool[slot // bs, 1, slot % bs // 16, at:at + 128] = 0x7F
    ops_fp8.paged_prefill_fp8(out, q, pool, tables.to(dev), cu, lens, m, SCALE)
    nan, first = torch.isnan(out), max(0, token - (n - m))  # query i sees keys up to n - m + i
    assert nan[first:, 2:].all() and int(nan.sum()) == (m - first) * 2 * D
    assert torch.equal(out[:, :2], before[:, :2]) and torch.equal(out[:first], before[:first])


def test_prefill_parts_repeat_in_graphs_and_on_two_streams(cuda_device):
    """Bit for bit: eager calls on two streams at once, and captured ones over lengths that change."""
    dev = cuda_device
    pool, tables, q, cu, lens, out = prefill_case(dev, [100, 30], [1500, 2500], 4, 2, 64, seed=3)
    tables = tables.to(dev)
    other = lens - 700

    def run(to, n):
        ops_fp8.paged_prefill_fp8(to, q, pool, tables, cu, n, 100, SCALE)

    want = {id(lens): out.clone(), id(other): torch.empty_like(out)}
    run(want[id(other)], other)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    outs = [[torch.empty_like(out) for _ in range(10)] for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    for i in range(10):
        for s, o, n in zip(streams, outs, (lens, other)):
            with torch.cuda.stream(s):
                run(o[i], n)
    torch.cuda.synchronize()
    for o, n in zip(outs, (lens, other)):
        assert all(torch.equal(x, want[id(n)]) for x in o)
    graph, held = torch.cuda.CUDAGraph(), lens.clone()
    with torch.cuda.graph(graph):
        run(out, held)
        run(outs[0][0], held)
    for n in (other, lens, other):
        held.copy_(n)
        graph.replay()
        assert torch.equal(out, want[id(n)]) and torch.equal(outs[0][0], want[id(n)])


def test_prefill_parts_flag_bad_blocks(cuda_device):
    dev, bs = cuda_device, 128
    pool, kr, vr = make_pool(dev, 12, bs, 1, 3)
    q = torch.randn(20, 1, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    out = torch.empty_like(q)
    for bad in range(12):
        table = torch.arange(12, dtype=torch.int32)[None]
        table[0, bad] = 12 if bad % 2 else -1
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        ops_fp8.paged_prefill_fp8(out, q, pool, table.to(dev), torch.tensor([0, 20], dtype=torch.int32, device=dev),
                                  torch.tensor([1500], dtype=torch.int32, device=dev), 20, SCALE, error_word=err)
        assert int(err.item()) == 2
        k, v = kr[:1500].clone(), vr[:1500].clone()
        k[bad * bs:(bad + 1) * bs] = 0  # what a bad block holds: zeros
        v[bad * bs:(bad + 1) * bs] = 0
        want, a = fp4_oracle.attention(q, k, v, SCALE)
        check(out, want, a, 1500, float(vr.abs().max()), PREFILL, f"block {bad}")


def test_append_decode_and_prefill_together(cuda_device):
    """As they are used: a prompt appended and prefilled, then tokens appended and decoded one by one; each decode is
    the last row of a prefill over the same pool."""
    dev = cuda_device
    h, kvh, bs, n0, steps = 8, 2, 32, 90, 20
    k, v = (t.to(dev) for t in random_rows(n0 + steps, kvh, 8, spread=4))
    q = torch.randn(n0 + steps, h, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    table = torch.tensor([[4, 1, 3, 0]], dtype=torch.int32, device=dev)
    pool = torch.zeros(ops_fp8.pool_shape(5, bs, kvh), dtype=torch.uint8, device=dev)
    slots = seq_slots(table[0].cpu(), n0 + steps, bs, dev)
    ws = workspace(dev, h, kvh)
    ops_fp8.kv_append_fp8(pool, k[:n0], v[:n0], slots[:n0])
    for i in range(n0, n0 + steps):
        ops_fp8.kv_append_fp8(pool, k[i:i + 1], v[i:i + 1], slots[i:i + 1])
        lens = torch.tensor([i + 1], dtype=torch.int32, device=dev)
        one, last = torch.empty_like(q[:1]), torch.empty_like(q[:1])
        ops_fp8.paged_decode_fp8(one, q[i:i + 1], pool, table, lens, SCALE, ws)
        ops_fp8.paged_prefill_fp8(last, q[i:i + 1].contiguous(), pool, table,
                                  torch.tensor([0, 1], dtype=torch.int32, device=dev), lens, 1, SCALE)
        kr, vr = (t.double() for t in ops_fp8.kv_read_fp8(pool, slots[:i + 1]))
        want, a = fp4_oracle.attention(q[i:i + 1], kr, vr, SCALE)
        vmax = 2 * float(vr.abs().max())
        check(one, want, a, i + 1, vmax, DECODE)
        check(last, want, a, i + 1, vmax, PREFILL)
