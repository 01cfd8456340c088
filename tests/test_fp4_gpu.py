"""The 4-bit KV pool's kernels against the restatement in oracle/fp4_oracle.py.

Append, read and norm + RoPE + append are compared bit for bit. Attention is
compared with 64-bit arithmetic over the values that the codes stand for; its
tolerance counts the roundings on the way (relative half steps: bf16 2^-8,
fp16 2^-11):

* the output's own, 2^-8 |o|;
* the weights', which are held in fp16 (in decode rounded, multiplied by V's
  scale and rounded again: two half steps; in prefill once), of the weighted
  mean of |v|, A;
* scores: sums of 128 products in fp32 (in the test's range below 2^7 in log2
  units, so within 2^-14 of them after 128 roundings of 2^-24 relative to the
  sum of magnitudes), the exponential's 2^-22, fp16's floor for entries of q
  far below the row's largest: together below 2^-12 of a weight, so 2^-11 A
  with the denominator's share;
* fp16's smallest step, 2^-24: a weight far below the largest one (which is at
  least 1 in the units of p) is off by half of it, over the power of two that
  p is held with. In prefill that is 2^-25 / 2^7 of |v| a key; in decode
  2^-25 / 2^4 of |v| and, for the product with the scale, of a code of up to 6.
"""

import numpy as np
import pytest
import torch

from nano_vllm_ascend_b200 import ops, ops_fp4
from oracle import fp4_oracle as orc
from tests.helpers import seeded_tables

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5
DECODE = dict(per_a=2 * 2.0 ** -11 + 2.0 ** -11, step=2.0 ** -29, code=6.0)
PREFILL = dict(per_a=2.0 ** -11 + 2.0 ** -11, step=2.0 ** -32, code=0.0)


def check(got, want, a, v, how, what=""):
    """``want`` and ``a`` from the restatement, ``v`` the rows attended over, ``how`` DECODE or PREFILL."""
    err = (got.double() - want).abs()
    far = v.shape[0] * how["step"] * (float(v.abs().max()) + how["code"]) if v.numel() else 0.0
    tol = want.abs() * 2.0 ** -8 + a * how["per_a"] + far + 1e-30
    assert bool((err <= tol).all()), f"{what}: off by up to {float((err / tol).max()):.2f} tolerances"
    assert not torch.isnan(got).any()


def random_rows(tokens, kvh, seed, dtype=torch.bfloat16, spread=True):
    """K and V rows whose groups' magnitudes differ."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, tokens, kvh, 8, 16, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-3, 4, (2, tokens, kvh, 8, 1), generator=g).float())
    x = x.view(2, tokens, kvh, D).to(dtype)
    return x[0], x[1]


def make_pool(dev, nb, bs, kvh, seed, spread=False):
    """A pool with every slot written (through the kernel), and its rows in float64."""
    k, v = random_rows(nb * bs, kvh, seed, spread=spread)
    pool = torch.zeros(ops_fp4.pool_shape(nb, bs, kvh), dtype=torch.uint8, device=dev)
    ops_fp4.kv_append_fp4(pool, k.to(dev), v.to(dev), torch.arange(nb * bs, device=dev))
    kr, vr = ops_fp4.kv_read_fp4(pool, torch.arange(nb * bs, device=dev))
    return pool, kr.double(), vr.double()


def canonical(pool):
    """The pool's bytes with +0 for the codes of -0 (the sign of a zero is not kept)."""
    p = pool.cpu().numpy().copy() if isinstance(pool, torch.Tensor) else pool.copy()
    for part in (p[..., :1024], p[..., 1152:2176]):
        part[(part & 0x0F) == 0x08] &= 0xF0
        part[(part & 0xF0) == 0x80] &= 0x0F
    return p


def workspace(dev, h, kvh, num_ctas=0):
    return torch.zeros(ops_fp4.decode_fp4_workspace_bytes(h, kvh, D, num_ctas), dtype=torch.uint8, device=dev)


def seq_slots(table, n, bs, dev):
    i = torch.arange(n, device=dev)
    return table.to(dev).long()[i // bs] * bs + i % bs


# ------------------------------------------------------ append and read ---
@pytest.mark.parametrize("tokens,kvh,bs,dtype", [
    (1, 1, 16, torch.bfloat16), (32, 8, 128, torch.bfloat16), (77, 3, 32, torch.float16),
    (333, 5, 64, torch.bfloat16), (1500, 2, 256, torch.float16), (4097, 4, 16, torch.bfloat16)])
def test_append_and_read_are_exact(cuda_device, tokens, kvh, bs, dtype):
    dev = cuda_device
    k, v = random_rows(tokens, kvh, tokens, dtype)
    nb = -(-tokens // bs) + 2
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(1))[:tokens]
    before = torch.randint(0, 256, ops_fp4.pool_shape(nb, bs, kvh), dtype=torch.uint8,
                           generator=torch.Generator().manual_seed(2))
    before[before == 0x7F] = 0  # a NaN scale reads as NaN
    before[before == 0xFF] = 0
    pool = before.to(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ops_fp4.kv_append_fp4(pool, k.to(dev), v.to(dev), slots.to(dev), error_word=err)
    want = before.numpy().copy()
    orc.append(want, k.float().numpy(), v.float().numpy(), slots.numpy())
    assert np.array_equal(canonical(pool), canonical(want))
    kr, vr = ops_fp4.kv_read_fp4(pool, slots.to(dev), dtype=dtype, error_word=err)
    for got, ref in zip((kr, vr), orc.rows(want)):
        assert np.array_equal(got.cpu().double().numpy(), ref[slots.numpy()])
    assert int(err.item()) == 0


def test_append_rounds_ties_to_even_and_saturates(cuda_device):
    """Every border of the codes and of the scales, values next to them, and what lies beyond both ranges."""
    dev = cuda_device
    rows = []
    for s in (2.0 ** -9, 3 * 2.0 ** -9, 0.015625, 0.9375, 1.0, 1.125, 1.875, 448.0):
        borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
        b = (borders * s).to(torch.bfloat16)
        ulp = torch.exp2(torch.floor(torch.log2(b.float())) - 7)
        for d in (-1, 0, 1):
            x = torch.zeros(16)
            x[:8] = b.float() + d * ulp
            x[8:] = -x[:8]
            x[15] = 6 * s  # fixes the group's scale
            rows.append(x)
    for m in torch.arange(8, 17).tolist():  # scales between two e4m3 values, and ties
        for f in (0.0, 0.25, 0.5, 0.75):
            x = torch.linspace(-1, 1, 16) * 6 * (m + f) / 8
            x[0] = 6 * (m + f) / 8
            rows.append(x)
    rows += [torch.full((16,), 1e-4), torch.full((16,), 0.0058), torch.full((16,), 0.006), torch.zeros(16),
             torch.full((16,), -0.0), torch.linspace(-1e5, 1e5, 16), torch.full((16,), 3e38)]
    inf = torch.linspace(-3, 3, 16)
    inf[3], inf[4] = float("inf"), float("-inf")
    rows.append(inf)
    while len(rows) % 8:
        rows.append(torch.linspace(0, 1, 16))
    x = torch.stack(rows).view(-1, 1, D).to(torch.bfloat16)
    n = x.shape[0]
    pool = torch.zeros(ops_fp4.pool_shape(-(-n // 16), 16, 1), dtype=torch.uint8, device=dev)
    ops_fp4.kv_append_fp4(pool, x.to(dev), x.flip(0).contiguous().to(dev), torch.arange(n, device=dev))
    want = np.zeros(tuple(pool.shape), dtype=np.uint8)
    orc.append(want, x.float().numpy(), x.flip(0).float().numpy(), np.arange(n))
    assert np.array_equal(canonical(pool), canonical(want))


def test_append_nan_group_reads_as_nan(cuda_device):
    dev = cuda_device
    k, v = random_rows(4, 2, 3)
    k[1, 0, 20] = float("nan")
    v[2, 1, 127] = -float("nan")
    pool = torch.zeros(ops_fp4.pool_shape(1, 16, 2), dtype=torch.uint8, device=dev)
    ops_fp4.kv_append_fp4(pool, k.to(dev), v.to(dev), torch.arange(4, device=dev))
    kr, vr = ops_fp4.kv_read_fp4(pool, torch.arange(4, device=dev))
    nk, nv = torch.isnan(kr).cpu(), torch.isnan(vr).cpu()
    assert nk[1, 0, 16:32].all() and int(nk.sum()) == 16
    assert nv[2, 1, 112:].all() and int(nv.sum()) == 16


def test_append_strided_rows_bad_slots_and_constants(cuda_device):
    """Slices of a fused QKV output (4-byte aligned), slots outside the pool, power-of-two constants, no tokens."""
    dev = cuda_device
    t, kvh, bs, nb = 50, 2, 32, 3
    buf = torch.randn(t, 6 * D + 2, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16) * 40
    qkv = buf.to(dev)[:, :6 * D].unflatten(1, (6, D))
    k, v = qkv[:, 2:4], qkv[:, 4:6]
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(6))[:t]
    slots[3], slots[10], slots[49] = -1, nb * bs, 1 << 40
    pool = torch.zeros(ops_fp4.pool_shape(nb, bs, kvh), dtype=torch.uint8, device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ops_fp4.kv_append_fp4(pool, k, v, slots.to(dev), 8.0, 0.25, error_word=err)
    assert int(err.item()) == 4
    want = np.zeros(tuple(pool.shape), dtype=np.uint8)
    orc.append(want, k.float().cpu().numpy(), v.float().cpu().numpy(), slots.numpy(), 8.0, 0.25)
    assert np.array_equal(canonical(pool), canonical(want))
    err.zero_()
    kr, vr = ops_fp4.kv_read_fp4(pool, slots.to(dev), 8.0, 0.25, error_word=err)
    assert int(err.item()) == 4
    ok = (slots >= 0) & (slots < nb * bs)
    for got, ref in zip((kr, vr), orc.rows(want, 8.0, 0.25)):
        assert np.array_equal(got[ok.to(dev)].cpu().double().numpy(), ref[slots[ok].numpy()])
        assert not got[~ok.to(dev)].any()
    ops_fp4.kv_append_fp4(pool, k[:0], v[:0], slots[:0].to(dev))
    kr, vr = ops_fp4.kv_read_fp4(pool, slots[:0].to(dev))
    assert kr.shape == (0, kvh, D) and np.array_equal(canonical(pool), canonical(want))


# -------------------------------------------------- norm + rope + append ---
def rope_tables(max_pos, theta=1e6):
    inv = 1.0 / (theta ** (torch.arange(0, D, 2, dtype=torch.float32) / D))
    f = torch.outer(torch.arange(max_pos, dtype=torch.float32), inv)
    f = torch.cat((f, f), dim=-1)
    return f.cos(), f.sin()


@pytest.mark.parametrize("tokens,h,kvh,bs", [(1, 16, 8, 128), (33, 5, 1, 16), (7, 9, 3, 64), (2500, 4, 2, 32),
                                              (3000, 7, 1, 128), (2367, 16, 8, 64), (2368, 4, 1, 16),
                                              (300, 16, 8, 32), (2500, 16, 8, 128), (700, 35, 5, 64)])
def test_norm_rope_append_is_exact(cuda_device, tokens, h, kvh, bs):
    dev = cuda_device
    g = torch.Generator().manual_seed(tokens)
    qkv = (torch.randn(tokens, h + 2 * kvh, D, generator=g) * 3).to(torch.bfloat16)
    wq, wk = ((1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16) for _ in range(2))
    cos, sin = rope_tables(4096)
    pos = torch.randint(0, 4096, (tokens,), generator=g)
    nb = -(-tokens // bs) + 1
    slots = torch.randperm(nb * bs, generator=g)[:tokens]
    pool = torch.zeros(ops_fp4.pool_shape(nb, bs, kvh), dtype=torch.uint8, device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    d = qkv.to(dev)
    q_out = ops_fp4.qk_norm_rope_append_fp4(d[:, :h], d[:, h:h + kvh], d[:, h + kvh:], wq.to(dev), wk.to(dev), 1e-6,
                                            cos.to(dev), sin.to(dev), pos.to(dev), pool, slots.to(dev),
                                            error_word=err)
    assert int(err.item()) == 0
    x = qkv.float().numpy()
    args = (1e-6, cos[pos].numpy(), sin[pos].numpy())
    want_q = orc.norm_rope(x[:, :h], wq.float().numpy(), *args)
    want_k = orc.norm_rope(x[:, h:h + kvh], wk.float().numpy(), *args)
    assert torch.equal(q_out.cpu().view(torch.int16), want_q.view(torch.int16))
    want = np.zeros(tuple(pool.shape), dtype=np.uint8)
    orc.append(want, want_k.float().numpy(), x[:, h + kvh:], slots.numpy())
    assert np.array_equal(canonical(pool), canonical(want))


def test_norm_rope_append_bad_slot_and_position(cuda_device):
    dev = cuda_device
    q, kv = torch.randn(3, 4, D, device=dev).to(torch.bfloat16), torch.randn(3, 2, D, device=dev).to(torch.bfloat16)
    cos, sin = (t.to(dev) for t in rope_tables(64))
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    pool = torch.zeros(ops_fp4.pool_shape(2, 16, 2), dtype=torch.uint8, device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ops_fp4.qk_norm_rope_append_fp4(q, kv, kv, w, w, 1e-6, cos, sin, torch.tensor([1, 64, -7], device=dev), pool,
                                    torch.tensor([5, 32, -1], device=dev), error_word=err)
    assert int(err.item()) == 4 + 8
    _, vr = ops_fp4.kv_read_fp4(pool, torch.arange(32, device=dev))
    assert vr[5].any() and not vr[torch.arange(32) != 5].any()


def norm_inputs(dev, tokens, h, kvh, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(tokens, h + 2 * kvh, D, generator=g) * 3).to(torch.bfloat16).to(dev)
    wq, wk = ((1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).to(dev) for _ in range(2))
    pos = torch.randint(0, 512, (tokens,), generator=g).to(dev)
    slots = torch.randperm(tokens + 7, generator=g)[:tokens].to(dev)
    pool = torch.zeros(ops_fp4.pool_shape(-(-(tokens + 7) // 32), 32, kvh), dtype=torch.uint8, device=dev)
    return qkv, wq, wk, pos, slots, pool


@pytest.mark.parametrize("tokens", [5, 3001])
@pytest.mark.parametrize("how", ["rows", "tables", "odd pitch"])
def test_norm_rope_append_of_rows_with_4_byte_alignment(cuda_device, tokens, how):
    """Rows, tables or token strides that only 4-byte accesses may take give the same bits."""
    dev, h, kvh = cuda_device, 6, 3
    qkv, wq, wk, pos, slots, pool = norm_inputs(dev, tokens, h, kvh, tokens)
    cos, sin = (t.to(dev) for t in rope_tables(512))
    split = lambda t: (t[:, :h], t[:, h:h + kvh], t[:, h + kvh:])
    want = ops_fp4.qk_norm_rope_append_fp4(*split(qkv), wq, wk, 1e-6, cos, sin, pos, pool, slots)
    width = (h + 2 * kvh) * D
    if how == "tables":
        cos, sin = (torch.cat((t.new_zeros(1), t.flatten()))[1:].view(512, D) for t in (cos, sin))
        assert cos.data_ptr() % 16 == 4
        rows = qkv
    else:
        pitch, first = (width, 2) if how == "rows" else (width + 2, 0)
        flat = torch.zeros(first + tokens * pitch, dtype=torch.bfloat16, device=dev)
        rows = flat[first:].as_strided((tokens, h + 2 * kvh, D), (pitch, D, 1), first)
        rows.copy_(qkv)
    again = torch.zeros_like(pool)
    got = ops_fp4.qk_norm_rope_append_fp4(*split(rows), wq, wk, 1e-6, cos, sin, pos, again, slots)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16)) and torch.equal(again, pool)


def test_norm_rope_append_of_special_rows_and_in_place(cuda_device):
    """A NaN makes its whole row NaN, an infinity its own place (the others are 0), a row of zeros stays one; other
    rows are not touched by them. The query may be normalised in place."""
    dev, h, kvh, tokens = cuda_device, 4, 2, 40
    qkv, wq, wk, pos, slots, pool = norm_inputs(dev, tokens, h, kvh, 3)
    cos, sin = torch.ones(512, D, device=dev), torch.zeros(512, D, device=dev)  # no rotation: 0 * inf is not asked for
    qkv[4, 1, 77] = float("nan")
    qkv[9, h, 3] = float("nan")
    qkv[11, 0] = 0
    qkv[12, h + 1] = 0
    want = orc.norm_rope(qkv[:, :h].float().cpu().numpy(), wq.float().cpu().numpy(), 1e-6, cos[pos].cpu().numpy(),
                         sin[pos].cpu().numpy())
    q = qkv[:, :h].contiguous()
    got = ops_fp4.qk_norm_rope_append_fp4(q, qkv[:, h:h + kvh], qkv[:, h + kvh:], wq, wk, 1e-6, cos, sin, pos, pool,
                                          slots, query_out=q)
    assert got.data_ptr() == q.data_ptr()
    bad = torch.isnan(want)
    assert bad[4, 1].all() and int(bad.sum()) == D
    got = got.cpu()
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], want[~bad])
    kr, vr = ops_fp4.kv_read_fp4(pool, slots)
    assert torch.isnan(kr[9, 0]).all() and int(torch.isnan(kr).sum()) == D and not torch.isnan(vr).any()
    assert not kr[12, 1].any() and kr[12, 0].any()


# ----------------------------------------------------------------- decode ---
def decode_case(dev, ctx, h, kvh, bs, seed=0, q_mul=1.0, num_ctas=0, ws=None, spread=False):
    nb = sum(-(-n // bs) for n in ctx) + 2
    pool, kr, vr = make_pool(dev, nb, bs, kvh, seed, spread)
    tables = seeded_tables(ctx, bs, nb, seed)
    q = (torch.randn(len(ctx), h, D, generator=torch.Generator().manual_seed(seed + 1)) * q_mul).to(torch.bfloat16)
    q = q.to(dev)
    out = torch.full_like(q, float("nan"))
    ws = workspace(dev, h, kvh, num_ctas) if ws is None else ws
    lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
    ops_fp4.paged_decode_fp4(out, q, pool, tables.to(dev), lens, SCALE, ws, num_ctas)
    assert int(ws[:4].view(torch.int32).item()) == 0
    assert not ws[256:256 + 4096].any(), "the tickets must be back at zero"
    for b, n in enumerate(ctx):
        sl = seq_slots(tables[b], n, bs, dev)
        want, a = orc.attention(q[b:b + 1], kr[sl], vr[sl], SCALE)
        check(out[b:b + 1], want, a, vr[sl], DECODE, f"sequence {b} of {n} tokens")
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


def test_decode_scores_that_climb_and_large_scales(cuda_device):
    """Peaked rows (the running maximum moves often), queries far from 1, groups of very different scales."""
    decode_case(cuda_device, [900, 63], 4, 1, 32, seed=1, q_mul=8.0)
    decode_case(cuda_device, [900, 63], 4, 1, 32, seed=2, q_mul=2.0 ** -40)
    decode_case(cuda_device, [300, 63], 4, 1, 32, seed=3, q_mul=0.25, spread=True)


def test_decode_many_sequences(cuda_device):
    """More sequences than one launch takes."""
    g = torch.Generator().manual_seed(1)
    decode_case(cuda_device, torch.randint(0, 40, (1100,), generator=g).tolist(), 2, 1, 16, seed=5)


def test_decode_empty_batch_and_only_empty_sequences(cuda_device):
    dev = cuda_device
    decode_case(dev, [0, 0, 0], 4, 2, 16)
    pool = torch.zeros(ops_fp4.pool_shape(1, 16, 2), dtype=torch.uint8, device=dev)
    q = torch.empty(0, 4, D, dtype=torch.bfloat16, device=dev)
    ops_fp4.paged_decode_fp4(q, q, pool, torch.zeros(0, 1, dtype=torch.int32, device=dev),
                             torch.zeros(0, dtype=torch.int32, device=dev), SCALE, workspace(dev, 4, 2))


def test_decode_ignores_what_lies_behind_the_context(cuda_device):
    """NaN rows behind the last token, wild ids in unused table columns, a strided table, a longer length than blocks
    elsewhere in the pool: none of it reaches the output."""
    dev = cuda_device
    ctx, h, kvh, bs = [5, 18, 40], 4, 2, 16
    pool, tables, q, out = decode_case(dev, ctx, h, kvh, bs, seed=9)
    before = out.clone()
    nan = torch.full((1, kvh, D), float("nan"), dtype=torch.bfloat16, device=dev)
    for b, n in enumerate(ctx):
        for i in range(n, -(-n // bs) * bs):
            slot = torch.tensor([int(tables[b, i // bs]) * bs + i % bs], device=dev)
            ops_fp4.kv_append_fp4(pool, nan, nan, slot)
    wide = torch.full((3, 11), -12345, dtype=torch.int32)
    for b, n in enumerate(ctx):
        wide[b, :-(-n // bs)] = tables[b, :-(-n // bs)]
    view = wide.to(dev)[:, :7]
    ws = workspace(dev, h, kvh)
    ops_fp4.paged_decode_fp4(out, q, pool, view, torch.tensor(ctx, dtype=torch.int32, device=dev), SCALE, ws)
    assert torch.equal(out, before) and int(ws[:4].view(torch.int32).item()) == 0


def test_decode_propagates_a_nan_that_is_seen(cuda_device):
    dev = cuda_device
    ctx, h, kvh, bs = [40, 40], 4, 2, 16
    pool, tables, q, out = decode_case(dev, ctx, h, kvh, bs, seed=9)
    before = out.clone()
    row = torch.zeros(1, kvh, D, dtype=torch.bfloat16, device=dev)
    row[0, 1, 5] = float("nan")  # one group of KV head 1
    ops_fp4.kv_append_fp4(pool, torch.zeros_like(row), row, torch.tensor([int(tables[0, 1]) * bs], device=dev))
    ops_fp4.paged_decode_fp4(out, q, pool, tables.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev), SCALE,
                             workspace(dev, h, kvh))
    nan = torch.isnan(out)
    assert nan[0, 2:, :16].all() and int(nan.sum()) == 2 * 16 and torch.equal(out[1], before[1])


def test_decode_flags_bad_blocks_and_long_contexts(cuda_device):
    dev = cuda_device
    h, kvh, bs = 2, 1, 16
    pool, kr, vr = make_pool(dev, 4, bs, kvh, 3)
    q = torch.randn(2, h, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    out = torch.empty_like(q)
    ws = workspace(dev, h, kvh)
    tables = torch.tensor([[0, 4], [2, -1]], dtype=torch.int32, device=dev)
    ops_fp4.paged_decode_fp4(out, q, pool, tables, torch.tensor([20, 30], dtype=torch.int32, device=dev), SCALE, ws)
    assert int(ws[:4].view(torch.int32).item()) == 2
    for b, (blk, n) in enumerate(((0, 4), (2, 14))):  # the bad block's tokens count as rows of zeros
        k = torch.cat([kr[blk * bs:(blk + 1) * bs], torch.zeros(n, kvh, D, device=dev, dtype=torch.float64)])
        v = torch.cat([vr[blk * bs:(blk + 1) * bs], torch.zeros(n, kvh, D, device=dev, dtype=torch.float64)])
        want, a = orc.attention(q[b:b + 1], k, v, SCALE)
        check(out[b:b + 1], want, a, v, DECODE)
    ws.zero_()
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    ops_fp4.paged_decode_fp4(out, q, pool, tables, torch.tensor([33, -5], dtype=torch.int32, device=dev), SCALE, ws)
    assert int(ws[:4].view(torch.int32).item()) == 8
    want, a = orc.attention(q[:1], kr[:32], vr[:32], SCALE)
    check(out[:1], want, a, vr[:32], DECODE)
    assert not out[1].any()


def test_decode_one_workspace_for_many_shapes(cuda_device):
    dev = cuda_device
    ws = workspace(dev, 64, 8)
    for i, (ctx, h, kvh) in enumerate([([3000], 16, 8), ([5, 900], 8, 1), ([1] * 50, 4, 4), ([2000, 2000], 64, 8)]):
        decode_case(dev, ctx, h, kvh, 32, seed=i, ws=ws)


def test_decode_constants_scale_the_result(cuda_device):
    """k_scale and v_scale are powers of two that every entry point of a layer takes."""
    dev = cuda_device
    k, v = random_rows(48, 2, 8)
    tables = torch.tensor([[1, 0, 2]], dtype=torch.int32, device=dev)
    q = torch.randn(1, 4, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    outs = []
    for ks, vs in ((1.0, 1.0), (4.0, 2.0 ** -10)):
        pool = torch.zeros(ops_fp4.pool_shape(3, 16, 2), dtype=torch.uint8, device=dev)
        ops_fp4.kv_append_fp4(pool, k.to(dev) * ks, v.to(dev) * vs, torch.arange(48, device=dev), ks, vs)
        out = torch.empty_like(q)
        ops_fp4.paged_decode_fp4(out, q, pool, tables, torch.tensor([48], dtype=torch.int32, device=dev), SCALE / ks,
                                 workspace(dev, 4, 2), k_scale=ks, v_scale=vs)
        outs.append(out / vs)
    assert torch.equal(outs[0], outs[1])


def test_decode_far_offsets(cuda_device):
    """A pool whose last blocks lie past 4 GiB."""
    dev = cuda_device
    kvh, bs, h = 8, 256, 8
    per_block = kvh * bs // 16 * 2304
    nb = (4 << 30) // per_block + 40
    pool = torch.zeros(ops_fp4.pool_shape(nb, bs, kvh), dtype=torch.uint8, device=dev)
    n = 600
    k, v = random_rows(n, kvh, 4, spread=False)
    table = torch.tensor([[nb - 1, nb - 20, nb - 7]], dtype=torch.int32)
    slots = seq_slots(table[0], n, bs, dev)
    ops_fp4.kv_append_fp4(pool, k.to(dev), v.to(dev), slots)
    kr, vr = ops_fp4.kv_read_fp4(pool, slots)
    want_pool = np.zeros(ops_fp4.pool_shape(3, bs, kvh), dtype=np.uint8)
    orc.append(want_pool, k.float().numpy(), v.float().numpy(), np.arange(n))
    for got, ref in zip((kr, vr), orc.rows(want_pool)):
        assert np.array_equal(got.cpu().double().numpy(), ref[:n])
    q = torch.randn(1, h, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(dev)
    want, a = orc.attention(q, kr.double(), vr.double(), SCALE)
    out = torch.empty_like(q)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    ops_fp4.paged_decode_fp4(out, q, pool, table.to(dev), lens, SCALE, workspace(dev, h, kvh))
    check(out, want, a, vr.double(), DECODE)
    out.fill_(0)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    ops_fp4.paged_prefill_fp4(out, q, pool, table.to(dev), cu, lens, 1, SCALE)
    check(out, want, a, vr.double(), PREFILL)


# ---------------------------------------------------------------- prefill ---
def prefill_case(dev, q_lens, cached, h, kvh, bs, seed=0, q_mul=1.0, spread=False):
    kv = [a + b for a, b in zip(q_lens, cached)]
    nb = sum(-(-n // bs) for n in kv) + 2
    pool, kr, vr = make_pool(dev, nb, bs, kvh, seed, spread)
    tables = seeded_tables(kv, bs, nb, seed)
    total = sum(q_lens)
    q = (torch.randn(total, h, D, generator=torch.Generator().manual_seed(seed + 1)) * q_mul).to(torch.bfloat16).to(dev)
    out = torch.full_like(q, float("nan"))
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32).to(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    lens = torch.tensor(kv, dtype=torch.int32, device=dev)
    ops_fp4.paged_prefill_fp4(out, q, pool, tables.to(dev), cu, lens, max(q_lens), SCALE, error_word=err)
    assert int(err.item()) == 0
    at = 0
    for b, (m, n) in enumerate(zip(q_lens, kv)):
        sl = seq_slots(tables[b], n, bs, dev)
        want, a = orc.attention(q[at:at + m], kr[sl], vr[sl], SCALE)
        check(out[at:at + m], want, a, vr[sl], PREFILL, f"sequence {b}: {m} over {n}")
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


def test_prefill_scores_that_climb_and_large_scales(cuda_device):
    prefill_case(cuda_device, [200], [100], 4, 1, 32, seed=5, q_mul=8.0)
    prefill_case(cuda_device, [200], [100], 4, 1, 32, seed=6, q_mul=0.25, spread=True)


def test_prefill_many_items_per_cta(cuda_device):
    """More work items than CTAs, one and two query tiles each, with empty sequences between."""
    g = torch.Generator().manual_seed(3)
    q = torch.randint(0, 200, (60,), generator=g).tolist()
    c = torch.randint(0, 300, (60,), generator=g).tolist()
    prefill_case(cuda_device, q, c, 8, 2, 32, seed=8)


def test_prefill_is_near_the_bf16_kernel_over_the_same_values(cuda_device):
    """The tiles are exact: ops.paged_prefill over the pool that the codes stand for differs by the weights' roundings
    (bf16 there, fp16 here) and the outputs'."""
    dev = cuda_device
    pool, tables, q, cu, lens, out = prefill_case(dev, [130, 50], [200, 0], 8, 4, 128, seed=2)
    nb = pool.shape[0]
    kr, vr = ops_fp4.kv_read_fp4(pool, torch.arange(nb * 128, device=dev))
    got = torch.empty_like(out)
    ops.paged_prefill(got, q, kr.view(nb, 128, 4, D), vr.view(nb, 128, 4, D), tables.to(dev), cu, lens, 130, SCALE)
    a = vr.abs().max().double()
    assert bool(((got.double() - out.double()).abs() <= 2 * 2.0 ** -8 * out.double().abs() + a * 2 * 2.0 ** -8).all())


def test_prefill_rows_that_see_no_key_and_hidden_rows(cuda_device):
    """Fewer keys than queries: the first rows are zeros. NaN rows behind a sequence's end do not get in."""
    dev = cuda_device
    bs, kvh, h = 16, 1, 2
    pool, kr, vr = make_pool(dev, 4, bs, kvh, 11)
    nan = torch.full((12, kvh, D), float("nan"), dtype=torch.bfloat16, device=dev)
    ops_fp4.kv_append_fp4(pool, nan, nan, torch.arange(20, 32, device=dev))  # block 1 from its fifth token
    q = torch.randn(50, h, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    out = torch.full_like(q, float("nan"))
    tables = torch.tensor([[0, 1], [3, 99], [2, 99]], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 30, 40, 50], dtype=torch.int32, device=dev)
    lens = torch.tensor([20, 0, 16], dtype=torch.int32, device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ops_fp4.paged_prefill_fp4(out, q, pool, tables, cu, lens, 30, SCALE, error_word=err)
    assert int(err.item()) == 0
    for lo, hi, k, v in ((0, 30, kr[:20], vr[:20]), (40, 50, kr[32:48], vr[32:48])):
        want, a = orc.attention(q[lo:hi], k, v, SCALE)
        check(out[lo:hi], want, a, v, PREFILL)
    assert not out[:10].any() and not out[30:40].any()


def test_prefill_flags_bad_metadata(cuda_device):
    dev = cuda_device
    bs, kvh, h = 16, 1, 2
    pool, kr, vr = make_pool(dev, 4, bs, kvh, 12)
    q = torch.randn(8, h, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    for tables, lens, cu, bits in (([[0, 4]], [20], [0, 8], 2), ([[0, -3]], [20], [0, 8], 2),
                                   ([[0, 1]], [40], [0, 8], 8), ([[0, 1]], [20], [0, 9], 8),
                                   ([[0, 1]], [20], [-1, 5], 8)):
        out = torch.full((10, h, D), 7.0, dtype=torch.bfloat16, device=dev)
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        ops_fp4.paged_prefill_fp4(out[1:9], q, pool, torch.tensor(tables, dtype=torch.int32, device=dev),
                                  torch.tensor(cu, dtype=torch.int32, device=dev),
                                  torch.tensor(lens, dtype=torch.int32, device=dev), 9, SCALE, error_word=err)
        assert int(err.item()) == bits
        assert bool((out[0] == 7).all()) and bool((out[9] == 7).all()), "rows of others are left as they were"


# ------------------------------------------- together, captured, on streams ---
def test_append_decode_prefill_together_in_a_graph(cuda_device):
    """Prefill a prompt, then decode three tokens by replaying one captured step (norm + RoPE + append, decode), on
    another stream than the default; every step matches attention over the rows read back."""
    dev = cuda_device
    h, kvh, bs, n0 = 8, 2, 32, 70
    g = torch.Generator(device=dev).manual_seed(1)
    cos, sin = (t.to(dev) for t in rope_tables(256))
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    table = torch.tensor([[3, 0, 2]], dtype=torch.int32, device=dev)
    pool = torch.zeros(ops_fp4.pool_shape(4, bs, kvh), dtype=torch.uint8, device=dev)
    new = torch.randn(n0 + 3, h + 2 * kvh, D, generator=g, device=dev).to(torch.bfloat16)
    slots = seq_slots(table[0], n0 + 3, bs, dev)
    pos = torch.arange(n0 + 3, device=dev)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        q = ops_fp4.qk_norm_rope_append_fp4(new[:n0, :h], new[:n0, h:h + kvh], new[:n0, h + kvh:], w, w, 1e-6, cos,
                                            sin, pos[:n0], pool, slots[:n0])
        out = torch.empty_like(q)
        ops_fp4.paged_prefill_fp4(out, q, pool, table, torch.tensor([0, n0], dtype=torch.int32, device=dev),
                                  torch.tensor([n0], dtype=torch.int32, device=dev), n0, SCALE)
        kr, vr = ops_fp4.kv_read_fp4(pool, slots[:n0])
        want, a = orc.attention(q, kr.double(), vr.double(), SCALE)
        check(out, want, a, vr.double(), PREFILL, "prefill")
        ws = workspace(dev, h, kvh)
        x, p, sl = new[n0:n0 + 1].clone(), pos[n0:n0 + 1].clone(), slots[n0:n0 + 1].clone()
        ctx = torch.tensor([n0 + 1], dtype=torch.int32, device=dev)
        qd, od = torch.empty(1, h, D, dtype=torch.bfloat16, device=dev), torch.empty(1, h, D, dtype=torch.bfloat16,
                                                                                      device=dev)

        def step():
            ops_fp4.qk_norm_rope_append_fp4(x[:, :h], x[:, h:h + kvh], x[:, h + kvh:], w, w, 1e-6, cos, sin, p, pool,
                                            sl, query_out=qd)
            ops_fp4.paged_decode_fp4(od, qd, pool, table, ctx, SCALE, ws)

        step()
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(3):
            x.copy_(new[n0 + i:n0 + i + 1])
            p.fill_(n0 + i)
            sl.copy_(slots[n0 + i:n0 + i + 1])
            ctx.fill_(n0 + i + 1)
            graph.replay()
            kr, vr = ops_fp4.kv_read_fp4(pool, slots[:n0 + i + 1])
            want, a = orc.attention(qd, kr.double(), vr.double(), SCALE)
            check(od, want, a, vr.double(), DECODE, f"decode step {i}")
    torch.cuda.current_stream(dev).wait_stream(stream)


def test_decode_repeats_bit_for_bit(cuda_device):
    """The pieces of a split pair are joined in a fixed order: a call gives the same bits each time."""
    dev = cuda_device
    pool, tables, q, out = decode_case(dev, [3000, 40, 900], 8, 1, 32, seed=4)
    ws = workspace(dev, 8, 1)
    lens = torch.tensor([3000, 40, 900], dtype=torch.int32, device=dev)
    for _ in range(20):
        again = torch.empty_like(out)
        ops_fp4.paged_decode_fp4(again, q, pool, tables.to(dev), lens, SCALE, ws)
        assert torch.equal(again, out)


def test_two_calls_at_once(cuda_device):
    """Calls on two streams over one pool, each with a workspace of its own, give what each gives alone."""
    dev = cuda_device
    h, kvh, bs, ctx = 8, 2, 64, [5000, 33, 0, 700]
    nb = sum(-(-n // bs) for n in ctx)
    pool, _, _ = make_pool(dev, nb, bs, kvh, 11)
    tables = seeded_tables(ctx, bs, nb, 11).to(dev)
    lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
    cu = torch.arange(len(ctx) + 1, dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(2)
    qs = [torch.randn(len(ctx), h, D, generator=g, device=dev).to(torch.bfloat16) for _ in range(2)]
    streams, spaces = [torch.cuda.Stream(dev) for _ in range(2)], [workspace(dev, h, kvh) for _ in range(2)]

    def calls(i, n):
        outs = []
        for _ in range(n):
            o, p = torch.empty_like(qs[i]), torch.empty_like(qs[i])
            ops_fp4.paged_decode_fp4(o, qs[i], pool, tables, lens, SCALE, spaces[i])
            ops_fp4.paged_prefill_fp4(p, qs[i], pool, tables, cu, lens, 1, SCALE)
            outs += [o, p]
        return outs

    alone = [calls(i, 1) for i in range(2)]
    torch.cuda.synchronize(dev)
    both = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                both[i] += calls(i, 1)
    torch.cuda.synchronize(dev)
    for i in range(2):
        for k, o in enumerate(both[i]):
            assert torch.equal(o, alone[i][k % 2])


def test_query_may_be_overwritten(cuda_device):
    """out may be the query itself in decode: a row is read before any warp writes it."""
    dev = cuda_device
    pool, tables, q, out = decode_case(dev, [3000, 0, 17], 8, 4, 32, seed=9)
    ops_fp4.paged_decode_fp4(q, q, pool, tables.to(dev), torch.tensor([3000, 0, 17], dtype=torch.int32, device=dev),
                             SCALE, workspace(dev, 8, 4))
    assert torch.equal(q, out)


@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_queries_of_any_magnitude(cuda_device, which):
    """Queries far from 1 (the scale undoes it), rows whose entries span 2^24, rows of zeros, and rows with a NaN or an
    infinity, which come out as NaN and leave the others alone. Heads are rows of one tile, so a neighbour shows."""
    dev, h, kvh, bs, n = cuda_device, 4, 2, 32, 150
    pool, kr, vr = make_pool(dev, 6, bs, kvh, 21)
    table = torch.tensor([[4, 0, 3, 1, 5]], dtype=torch.int32, device=dev)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    sl = seq_slots(table[0], n, bs, dev)
    m = 1 if which == "decode" else 40
    g = torch.Generator().manual_seed(5)
    base = torch.randn(m, h, D, generator=g)
    spread = base * torch.exp2(torch.randint(-24, 1, (m, h, D), generator=g).float())
    for q_mul, x in ((2.0 ** 60, base), (2.0 ** -100, base), (2.0 ** -120, base), (1.0, spread), (0.0, base)):
        q = (x * q_mul).to(torch.bfloat16).to(dev)
        q[0, 1, 7], q[0, 2, 100] = float("nan"), float("inf")
        scale = SCALE / q_mul if 0 < q_mul else SCALE
        if q_mul < 2.0 ** -100:
            scale = SCALE * 2.0 ** 100  # as far as fp32 holds scale * log2(e) * 2^-112 apart: scores near 2^-20
        out = torch.empty_like(q)
        if which == "decode":
            ops_fp4.paged_decode_fp4(out, q, pool, table, lens, scale, workspace(dev, h, kvh))
        else:
            ops_fp4.paged_prefill_fp4(out, q, pool, table, torch.tensor([0, m], dtype=torch.int32, device=dev), lens,
                                      m, scale)
        bad = torch.zeros(m, h, dtype=torch.bool, device=dev)
        bad[0, 1] = bad[0, 2] = True
        assert torch.equal(torch.isnan(out).all(-1), bad) and torch.equal(torch.isnan(out).any(-1), bad)
        clean = torch.where(bad[..., None], torch.zeros_like(q), q)
        want, a = orc.attention(clean, kr[sl], vr[sl], scale)
        keep = ~bad[..., None].expand_as(want)
        check(out[keep], want[keep], a[keep], vr[sl], DECODE if which == "decode" else PREFILL, f"times {q_mul}")
