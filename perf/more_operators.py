"""Rotary positions, the 8-bit KV cache and pages of a cache, as cases that can be timed and compared.

A layer's 8-bit pool is uint8 [num_blocks, kv_heads, block_size / 16, 4128]: 16 tokens of one KV head make a unit of

    K codes [16 tokens][8 chunks][16]  e4m3, dims 16 * c .. 16 * c + 15 of token r in chunk c ^ (r % 8)
    V codes [16 tokens][8 chunks][16]  the same
    K exponent, V exponent             int32 each, then 24 bytes of zeros

A row's values are its codes times 2^exponent of its unit. Appending to a unit raises the exponent to the least that
holds the new rows (448 * 2^e, e from -40 to 40) and brings the rows that were there to it; writing the unit's first
token starts it anew: its exponent comes from the new rows alone, its other rows become zeros.
``run`` computes the operators in elementary torch operations, or, with ``own`` set, through the framework's entry
points.
"""

import math
import random

import torch

own = False

D = 128
UNIT = 4128
LEAST, MOST = -40, 40
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # one decode step's heads of 32 sequences, with the heads' norms: latency
        dict(name="rotary 32", op="rotary", tokens=32, heads=16, kv_heads=8, dim=128, rotated=128, interleaved=False,
             norm=True, scaling="none", positions=40960, dtype="bf16", seed=1),
        # a prefill step of another head layout: pairs side by side, half of the head, far positions, scaled
        dict(name="rotary 8191 part", op="rotary", tokens=8191, heads=32, kv_heads=8, dim=128, rotated=64,
             interleaved=True, norm=False, scaling="blend", positions=1 << 20, dtype="fp16", seed=2),
        # one decode step's rows of 32 sequences, each into a unit that is partly filled: latency
        dict(name="append 32", op="append", batch=32, lo=1, hi=1, c_lo=0, c_hi=2048, kv_heads=8, block_size=128,
             dtype="bf16", seed=3),
        # one prefill step: 32 requests of 256 new tokens over 768 cached ones
        dict(name="append 8192", op="append", batch=32, lo=256, hi=256, c_lo=768, c_hi=768, kv_heads=8, block_size=128,
             dtype="bf16", seed=4),
        # four short sequences, up to 513 tokens: latency
        dict(name="decode 4", op="decode", batch=4, lo=37, hi=513, heads=16, kv_heads=8, block_size=128, seed=5),
        # ragged, some sequences empty, five query heads a KV head, small blocks
        dict(name="decode 77 ragged", op="decode", batch=77, lo=0, hi=1500, heads=10, kv_heads=2, block_size=32,
             seed=6),
        # a large batch of long contexts
        dict(name="decode 256", op="decode", batch=256, lo=2048, hi=6144, heads=16, kv_heads=8, block_size=128, seed=7),
        # two sequences at the longest position, four query heads a KV head
        dict(name="decode 2 long", op="decode", batch=2, lo=40959, hi=40960, heads=32, kv_heads=8, block_size=128,
             seed=8),
        # 32 requests of 256 new tokens over a cached prefix of 768
        dict(name="prefill 32 cached", op="prefill", batch=32, q_lo=256, q_hi=256, c_lo=768, c_hi=768, heads=16,
             kv_heads=8, block_size=128, seed=9),
        # a few ragged requests, odd group size, small blocks
        dict(name="prefill 5 ragged", op="prefill", batch=5, q_lo=1, q_hi=300, c_lo=0, c_hi=1000, heads=9, kv_heads=3,
             block_size=64, seed=10),
        # one sequence forks: its last, partly filled page is copied in every layer
        dict(name="pages 1", op="pages", pool="fp8", layers=28, blocks=24, pairs=1, cleared=0, kv_heads=8,
             block_size=128, batch=8, seed=11),
        # a pool is compacted: 45 pages move to the front in every layer, 3 are cleared, and the tables follow
        dict(name="pages 48 bf16", op="pages", pool="bf16", layers=28, blocks=120, pairs=45, cleared=3, kv_heads=8,
             block_size=128, batch=32, seed=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "decode", "decode", "prefill", "pages"])
    bs = rng.choice([16, 32, 64, 128, 256])
    kvh = rng.choice([1, 2, 3, 4, 5, 6, 8])
    seed = rng.randrange(1 << 30)
    dtype = rng.choice(["bf16", "fp16"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
        return dict(op=op, tokens=_log(rng, 1, 8191), heads=kvh * rng.randint(1, 4), kv_heads=kvh, dim=dim,
                    rotated=rng.choice([dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                    norm=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "blend"]),
                    positions=_log(rng, 16, 1 << 20), dtype=dtype, seed=seed)
    if op == "append":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, max(1, 8192 // batch))
        c_hi = rng.choice([0, _log(rng, 1, max(1, 32768 // batch))])
        return dict(op=op, batch=batch, lo=rng.choice([1, hi]), hi=hi, c_lo=rng.choice([0, c_hi]), c_hi=c_hi,
                    kv_heads=kvh, block_size=bs, dtype=dtype, seed=seed)
    if op == "decode":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, 40960 if batch <= 16 else max(2, (1 << 20) // batch))
        lo = rng.choice([0, 1, hi // 2, hi])
        return dict(op=op, batch=batch, lo=min(lo, hi), hi=hi, heads=kvh * rng.randint(1, 8), kv_heads=kvh,
                    block_size=bs, seed=seed)
    if op == "pages":
        pool = rng.choice(["fp8", "bf16", "fp4"])
        layers, pairs = rng.randint(1, 28), _log(rng, 1, 45)
        cleared = rng.choice([0, 0, 1, 3])
        while pool == "bf16" and bs * kvh > 1024:  # no more than the largest listed one
            bs //= 2
        return dict(op=op, pool=pool, layers=layers, blocks=2 * (pairs + cleared) + rng.randint(1, 24), pairs=pairs,
                    cleared=cleared, kv_heads=kvh, block_size=bs, batch=_log(rng, 1, 64), seed=seed)
    batch = _log(rng, 1, 32)
    q_hi = _log(rng, 1, 2048 if batch <= 4 else 256)
    c_hi = rng.choice([0, _log(rng, 1, 4096 if batch <= 4 else 768)])
    case = dict(op=op, batch=batch, q_lo=rng.choice([1, max(1, q_hi // 2), q_hi]), q_hi=q_hi,
                c_lo=rng.choice([0, c_hi]), c_hi=c_hi, heads=rng.randint(1, 4) * kvh, kv_heads=kvh, block_size=bs,
                seed=seed)
    while work(case)["flops"] > 6e10:  # no more than the largest listed prefill
        case["batch"] = (case["batch"] + 1) // 2 if case["batch"] > 1 else 1
        case["heads"] = max(kvh, case["heads"] - kvh) if case["batch"] == 1 else case["heads"]
    return case


def _lens(case):
    """The lengths of the case's sequences: contexts (decode), or new and cached tokens (append, prefill)."""
    r = random.Random(case["seed"])
    if case["op"] == "decode":
        return [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    lo, hi = (case["lo"], case["hi"]) if case["op"] == "append" else (case["q_lo"], case["q_hi"])
    q = [r.randint(lo, hi) for _ in range(case["batch"])]
    c = [r.randint(case["c_lo"], case["c_hi"]) for _ in range(case["batch"])]
    return q, c


def _block_shape(case):
    """Shape and dtype of one block of one of the pool's tensors, and how many tensors the pool has."""
    kvh, bs = case["kv_heads"], case["block_size"]
    if case["pool"] == "bf16":
        return (bs, kvh, D), torch.bfloat16, 2
    return (kvh, bs // 16, UNIT if case["pool"] == "fp8" else 2304), torch.uint8, 1


def work(case):
    op, kvh = case["op"], case["kv_heads"]
    if op == "rotary":
        rows = case["tokens"] * (case["heads"] + kvh)
        return {"bytes": rows * case["dim"] * 4 + case["tokens"] * 8 + case["rotated"] * 4,
                "flops": rows * (case["rotated"] * 3 + (case["dim"] * 4 if case["norm"] else 0))}
    if op == "pages":
        shape, dtype, tensors = _block_shape(case)
        block = math.prod(shape) * torch.empty(0, dtype=dtype).element_size() * tensors * case["layers"]
        return {"bytes": (2 * case["pairs"] + case["cleared"]) * block + case["blocks"] * 4, "flops": 0}
    if op == "append":
        q, c = _lens(case)
        t = sum(q)
        slots = sum(-(-(a + b) // case["block_size"]) for a, b in zip(q, c)) * case["block_size"]
        # the rows in and their codes out, then every row of the sequences' blocks read back
        return {"bytes": t * (kvh * (2 * 256 + 256) + 8) + slots * (kvh * (258 + 2 * 256) + 8),
                "flops": t * kvh * 2 * D * 3}
    h, bs = case["heads"], case["block_size"]
    if op == "decode":
        ctx = _lens(case)
        b = sum(ctx) * kvh * 256 + sum(-(-n // 16) for n in ctx) * kvh * 8 + 2 * len(ctx) * h * 256
        return {"bytes": b + sum(-(-n // bs) for n in ctx) * 4 + len(ctx) * 4, "flops": 4 * D * h * sum(ctx)}
    q, c = _lens(case)
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(q, c))
    b = sum((n + p) * kvh * 256 + -(-(n + p) // 16) * kvh * 8 for n, p in zip(q, c)) + 2 * sum(q) * h * 256
    return {"bytes": b, "flops": 4 * D * h * pairs}


# ------------------------------------------------------------ plain parts ---
def _exponents(amax):
    """Least e with amax <= 448 * 2^e, held to [LEAST, MOST]; amax float32, finite."""
    mant, e = torch.frexp(amax)  # amax = mant * 2^e, mant in [0.5, 1)
    e = e - 9 + (mant > 0.875).to(e.dtype)
    return torch.where(amax > 0, e.clamp(LEAST, MOST), LEAST)


def _codes(x, e):
    """x float32 over 2^e (e broadcast against it) as e4m3; rows with a NaN become NaN throughout."""
    y = torch.ldexp(x, -e).clamp(-448, 448)
    y = torch.where(torch.isnan(x).any(-1, keepdim=True), float("nan"), y)
    return y.to(torch.float8_e4m3fn)


def _swizzled(rows):
    """Bytes [..., 16 tokens, 128] with every 16-byte chunk c of token r at c ^ (r % 8); its own inverse."""
    r = torch.arange(16, device=rows.device)[:, None]
    c = torch.arange(8, device=rows.device)[None]
    return rows.unflatten(-1, (8, 16))[..., r, c ^ (r & 7), :].flatten(-2)


def _unpack(units):
    """Units uint8 [..., 4128] -> codes e4m3 [..., 2 (K, V), 16, 128] and exponents int32 [..., 2]."""
    codes = _swizzled(units[..., :4096].unflatten(-1, (2, 16, 128))).contiguous().view(torch.float8_e4m3fn)
    return codes, units[..., 4096:4104].contiguous().view(torch.int32)


def _pack(codes, exps):
    """Codes e4m3 [..., 2, 16, 128] and exponents int32 [..., 2] -> units uint8 [..., 4128]."""
    rest = torch.zeros(*exps.shape[:-1], 24, dtype=torch.uint8, device=exps.device)
    return torch.cat([_swizzled(codes.view(torch.uint8)).flatten(-3), exps.contiguous().view(torch.uint8), rest], -1)


def _values(codes, exps):
    return torch.ldexp(codes.float(), exps[..., None, None])


def _gathered(pool, tables):
    """K and V values of each sequence's blocks, float32 [batch, kv_heads, tokens, 128]."""
    g = pool[tables.long()].transpose(1, 2)  # [batch, kv_heads, blocks, units, 4128]
    v = _values(*_unpack(g))
    return v[..., 0, :, :].flatten(2, 4), v[..., 1, :, :].flatten(2, 4)


# ----------------------------------------------------------------- inputs ---
def _random_pool(blocks, kvh, bs, gen, dev):
    """A pool whose K and V were normal, of magnitudes that differ from unit to unit, before they were quantised."""
    pool = torch.empty(blocks * kvh * bs // 16, UNIT, dtype=torch.uint8, device=dev)
    for part in pool.split(1 << 17):
        n = part.shape[0]
        x = torch.randn(n, 2, 16, D, generator=gen, device=dev)
        x = (x * torch.exp2(torch.rand(n, 2, 1, 1, generator=gen, device=dev) * 4 - 3)).to(torch.bfloat16).float()
        e = _exponents(x.abs().amax((-1, -2)))
        part.copy_(_pack(_codes(x, e[..., None, None]), e))
    return pool.view(blocks, kvh, bs // 16, UNIT)


def _tables(lens, bs, gen, dev):
    """Block tables drawn without replacement from a permuted pool that is a little larger."""
    need = [-(-n // bs) for n in lens]
    total = sum(need) + 3
    perm = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    width = max(max(need), 1)
    at = torch.tensor([0] + need, device=dev).cumsum(0)
    col = torch.arange(width, device=dev)
    idx = at[:-1, None] + col
    used = col < (at[1:] - at[:-1])[:, None]
    return torch.where(used, perm[torch.where(used, idx, 0)], 0).to(torch.int32).contiguous(), total


def _frequencies(case):
    """The pairs' turns per position, float64, and what the cosines and sines are multiplied by."""
    half = case["rotated"] // 2
    inv = 1e6 ** -(torch.arange(half, dtype=torch.float64) / half)
    if case["scaling"] == "linear":
        return inv / 8, 1.0
    if case["scaling"] == "blend":  # slow pairs stretched by 8, fast ones kept, between them a ramp
        turns = 32768 * inv / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return inv * keep + inv / 8 * (1 - keep), 0.1 * math.log(8) + 1
    return inv, 1.0


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + case["seed"])

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device=dev).to(dtype)

    op, kvh = case["op"], case["kv_heads"]
    st = dict(op=op)
    if op == "rotary":
        t, h, d, dtype = case["tokens"], case["heads"], case["dim"], DTYPES[case["dtype"]]
        qkv = randn(t, h + 2 * kvh, d, dtype=dtype)  # the fused projection's output: q and k are slices of it
        inv, scale = _frequencies(case)
        st.update(q=qkv[:, :h], k=qkv[:, h:h + kvh], inv=inv.to(dev), scale=scale, inter=case["interleaved"],
                  pos=torch.randint(0, case["positions"], (t,), generator=gen, device=dev), wq=None, wk=None, eps=1e-6)
        if case["norm"]:
            st.update(wq=(1 + 0.1 * randn(d)).to(dtype), wk=(1 + 0.1 * randn(d)).to(dtype))
        return st
    bs = case["block_size"]
    if op == "pages":
        shape, dtype, tensors = _block_shape(case)
        n, m = case["pairs"], case["cleared"]
        st["pools"] = [torch.randint(0, 1 << 15, (case["layers"], case["blocks"], math.prod(shape) * dtype.itemsize // 2),
                                     generator=gen, device=dev, dtype=torch.int16).view(dtype).unflatten(-1, shape)
                       for _ in range(tensors)]
        perm = torch.randperm(case["blocks"], generator=gen, device=dev).to(torch.int32)
        src = torch.cat([perm[:n], torch.full((m,), -1, dtype=torch.int32, device=dev)])
        st["pairs"] = torch.stack([src, perm[n:2 * n + m]], 1).contiguous()
        moved = torch.arange(case["blocks"], dtype=torch.int32, device=dev)
        moved[perm[:n].long()] = perm[n:2 * n]
        live = torch.cat([perm[:n], perm[2 * n + m:]])  # tables hold pages that move and pages that stay
        st["map"] = moved
        st["tables"] = live[torch.randint(0, live.numel(), (case["batch"], 48), generator=gen, device=dev)]
        return st
    if op == "append":
        ql, cl = _lens(case)
        dtype = DTYPES[case["dtype"]]
        kv = [a + b for a, b in zip(ql, cl)]
        tables, nb = _tables(kv, bs, gen, dev)
        slots, every = [], []
        host = tables.tolist()
        for row, n, c in zip(host, ql, cl):
            slots += [row[p // bs] * bs + p % bs for p in range(c, c + n)]
            every += [b * bs + i for b in row[:-(-(n + c) // bs)] for i in range(bs)]
        t = sum(ql)
        kvs = randn(t, 2 * kvh, D, dtype=dtype)  # rows of a projection's output
        st.update(pool=_random_pool(nb, kvh, bs, gen, dev), k=kvs[:, :kvh], v=kvs[:, kvh:],
                  slots=torch.tensor(slots, device=dev), every=torch.tensor(every, device=dev))
        return st
    h = case["heads"]
    if op == "decode":
        ctx = _lens(case)
        tables, nb = _tables(ctx, bs, gen, dev)
        st.update(q=randn(len(ctx), h, D), ctx=torch.tensor(ctx, dtype=torch.int32, device=dev))
    else:
        ql, cl = _lens(case)
        kv = [a + b for a, b in zip(ql, cl)]
        tables, nb = _tables(kv, bs, gen, dev)
        cu = torch.tensor([0] + ql).cumsum(0).to(torch.int32).to(dev)
        st.update(q=randn(sum(ql), h, D), ctx=torch.tensor(kv, dtype=torch.int32, device=dev), cu=cu, max_q=max(ql))
    st.update(pool=_random_pool(nb, kvh, bs, gen, dev), tables=tables, scale=D ** -0.5)
    return st


# -------------------------------------------------------------------- run ---
def run(st):
    if own:
        return _run_own(st)
    op = st["op"]
    if op == "rotary":
        turn = st["pos"].double()[:, None] * st["inv"]  # 64 bits: far positions lose their angle in 32
        cos, sin = (f(turn).float()[:, None] * st["scale"] for f in (torch.cos, torch.sin))
        return {name: _rotated(st, st[name], st[w], cos, sin) for name, w in (("q", "wq"), ("k", "wk"))}
    if op == "pages":
        src, dst = st["pairs"].long().unbind(1)
        for pool in st["pools"]:
            rows = pool[:, src.clamp(min=0)]
            rows.masked_fill_((src < 0).view(1, -1, *[1] * (rows.dim() - 2)), 0)
            pool[:, dst] = rows
        st["tables"].copy_(st["map"][st["tables"].long()])
        return _page_outputs(st)
    if op == "append":
        pool, bs = st["pool"], st["pool"].shape[2] * 16
        nb, kvh, upb = pool.shape[:3]
        codes, exps = _unpack(pool)
        rows = torch.stack([st["k"], st["v"]], 2).float()  # [tokens, kv_heads, 2, 128]
        unit, off = st["slots"] // 16, st["slots"] % 16
        new = torch.zeros(nb * upb, 16, kvh, 2, D, device=pool.device)
        new[unit, off] = rows
        written = torch.zeros(nb * upb, 16, dtype=torch.bool, device=pool.device)
        written[unit, off] = True

        def per_head(x):  # [blocks * units, ...] -> [blocks, 1, units, ...]
            return x.unflatten(0, (nb, upb)).unsqueeze(1)

        new = new.view(nb, upb, 16, kvh, 2, D).permute(0, 3, 1, 4, 2, 5)  # [blocks, kv_heads, units, 2, 16, 128]
        e_new = _exponents(new.abs().masked_fill(~new.isfinite(), 0).amax((-1, -2)))
        anew, touched = per_head(written[:, 0])[..., None], per_head(written.any(1))[..., None]
        e = torch.where(anew, e_new, torch.where(touched, torch.maximum(exps, e_new), exps))
        here = per_head(written)[:, :, :, None, :, None]  # [blocks, 1, units, 1, 16, 1]
        kept = torch.where(anew[..., None, None], 0.0, _values(codes, exps))
        both = _codes(torch.where(here, new, kept), e[..., None, None])
        values = _values(both, e).permute(3, 0, 2, 4, 1, 5).reshape(2, nb * bs, kvh, D)[:, st["every"]]
        return {"key": values[0].to(st["k"].dtype), "value": values[1].to(st["k"].dtype)}
    k, v = _gathered(st["pool"], st["tables"])
    b, kvh, n = k.shape[:3]
    ctx, key = st["ctx"].long(), torch.arange(n, device=k.device)
    if op == "decode":
        q = st["q"].float().view(b, kvh, -1, D)  # [batch, kv_heads, group, 128]
        see = (key < ctx[:, None])[:, None, None]
    else:
        h, mq = st["q"].shape[1], st["max_q"]
        cu = st["cu"].long()
        lq = cu[1:] - cu[:-1]
        i = torch.arange(mq, device=k.device)
        row = cu[:-1, None] + i  # the query rows, padded to the longest sequence
        live = i < lq[:, None]
        q = st["q"].float()[torch.where(live, row, 0)].view(b, mq, kvh, h // kvh, D)
        q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)  # [batch, kv_heads, group * queries, 128]
        see = key <= (ctx - lq)[:, None, None] + i[:, None]
        see = see[:, None, None].expand(b, 1, h // kvh, mq, n).flatten(2, 3)
    s = (q @ k.transpose(-1, -2) * st["scale"]).masked_fill(~see, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    o = p @ v / p.sum(-1, keepdim=True).clamp(min=1e-30)
    if op == "decode":
        return o.reshape(b, -1, D).to(torch.bfloat16)
    o = o.view(b, kvh, -1, st["max_q"], D).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[live].to(torch.bfloat16)


def _rotated(st, x, w, cos, sin):
    y, n = x.float(), 2 * cos.shape[-1]
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + st["eps"]) * w.float()
    if st["inter"]:
        a, b = y[..., 0:n:2], y[..., 1:n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :n // 2], y[..., n // 2:n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., n:]], -1).to(x.dtype)


def _page_outputs(st):
    """The pools as whole numbers, and the tables."""
    return [p.view(torch.int16) for p in st["pools"]] + [st["tables"]]


def _run_own(st):
    from nano_vllm_ascend_b200 import ops, ops_fp8

    op = st["op"]
    if op == "rotary":
        q, k = ops.rotary(st["q"], st["k"], st["inv"], st["pos"], interleaved=st["inter"],
                          attention_scale=st["scale"], q_weight=st["wq"], k_weight=st["wk"], eps=st["eps"])
        return {"q": q, "k": k}
    if op == "pages":
        ops.copy_blocks(st["pools"], st["pairs"])
        ops.remap_blocks(st["tables"], st["map"])
        return _page_outputs(st)
    pool = st["pool"]
    if op == "append":
        ops_fp8.kv_append_fp8(pool, st["k"], st["v"], st["slots"])
        k, v = ops_fp8.kv_read_fp8(pool, st["every"], dtype=st["k"].dtype)
        return {"key": k, "value": v}
    out = torch.empty_like(st["q"])
    if op == "decode":
        if "ws" not in st:  # a user keeps one for all layers and steps
            size = ops_fp8.decode_fp8_workspace_bytes(st["q"].shape[1], pool.shape[1], D)
            st["ws"] = torch.zeros(size, dtype=torch.uint8, device=out.device)
        return ops_fp8.paged_decode_fp8(out, st["q"], pool, st["tables"], st["ctx"], st["scale"], st["ws"])
    return ops_fp8.paged_prefill_fp8(out, st["q"], pool, st["tables"], st["cu"], st["ctx"], st["max_q"], st["scale"])


# ------------------------------------------------------------------ exact ---
def _stored64(units):
    """Units uint8 [..., 4128] -> K and V float64 [..., 16, 128], each byte taken from its place."""
    i, d = torch.arange(16, device=units.device)[:, None], torch.arange(D, device=units.device)[None]
    place = 128 * i + 16 * (d // 16 ^ i % 8) + d % 16
    both = []
    for part in (0, 1):
        b = units[..., (2048 * part + place).reshape(-1)].long().unflatten(-1, (16, D))
        e, m = b >> 3 & 15, (b & 7).double()
        mag = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2(e.double() - 7))
        x = units[..., 4096 + 4 * part:4100 + 4 * part].long()
        x = x[..., 0] | x[..., 1] << 8 | x[..., 2] << 16 | x[..., 3] << 24
        x = torch.where(x >= 1 << 31, x - (1 << 32), x)
        both.append(torch.where(b >= 128, -mag, mag) * torch.exp2(x.double())[..., None, None])
    return both


def _round64(x):
    """x [...] to the nearest value of 4 significant bits, not finer than 2^-9; ties to even; at most 448."""
    e = torch.floor(torch.log2(x.abs().clamp(min=1e-300))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    op = case["op"]
    if op == "pages":
        return None  # nothing is computed
    st = prepare(case, seed)
    if op == "rotary":
        angle = st["pos"].double()[:, None, None] * st["inv"]
        out, half = {}, case["rotated"] // 2
        i = torch.arange(half, device=angle.device)
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        for name, w in (("q", st["wq"]), ("k", st["wk"])):
            x = st[name].double()
            if w is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + st["eps"]) * w.double()
            y = x.clone()
            y[..., a] = (x[..., a] * angle.cos() - x[..., b] * angle.sin()) * st["scale"]
            y[..., b] = (x[..., a] * angle.sin() + x[..., b] * angle.cos()) * st["scale"]
            out[name] = y
        return out
    kvh = case["kv_heads"]
    if op == "append":
        out = {}
        unit, off = st["slots"] // 16, st["slots"] % 16
        for name, pool, x in zip(("key", "value"), _stored64(st["pool"]), (st["k"], st["v"])):
            rows = pool.transpose(1, 2).reshape(-1, kvh, 16, D).clone()  # [units, kv_heads, 16, 128]
            part = int(name == "value")
            old = st["pool"][..., 4096 + 4 * part:4100 + 4 * part].contiguous().view(torch.int32)[..., 0]
            old = old.transpose(1, 2).reshape(-1, kvh).double()
            top = torch.zeros_like(old)
            top.index_reduce_(0, unit, x.double().abs().amax(-1), "amax")
            e = torch.ceil(torch.log2((top / 448).clamp(min=1e-300))).clamp(LEAST, MOST)
            first = torch.zeros(rows.shape[0], dtype=torch.bool, device=rows.device)
            first[unit[off == 0]] = True
            hit = torch.zeros_like(first)
            hit[unit] = True
            now = torch.where(first[:, None], e, torch.where(hit[:, None], torch.maximum(e, old), old))
            rows[first] = 0
            rows[unit, :, off] = x.double()
            step = torch.exp2(now)[..., None, None]
            rows = torch.where(hit[:, None, None, None], _round64(rows / step) * step, rows)
            out[name] = rows.transpose(1, 2).reshape(-1, kvh, D)[st["every"]]
        return out
    outs, q_all, bs, at = [], st["q"].double(), case["block_size"], 0
    lens = st["ctx"].tolist()
    new = [1] * len(lens) if op == "decode" else (st["cu"][1:] - st["cu"][:-1]).tolist()
    for b, (n, m) in enumerate(zip(lens, new)):
        q = q_all[at:at + m].unflatten(1, (kvh, -1))  # [m, kv_heads, group, 128]
        at += m
        if n == 0:
            outs.append(torch.zeros(m, case["heads"], D, dtype=torch.float64, device=q.device))
            continue
        blocks = st["pool"][st["tables"][b, :-(-n // bs)].long()]
        k, v = (x.transpose(0, 1).reshape(kvh, -1, D)[:, :n] for x in _stored64(blocks))
        s = torch.einsum("mkgd,knd->kgmn", q, k) * st["scale"]
        hidden = torch.arange(n, device=q.device) > n - m + torch.arange(m, device=q.device)[:, None]
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
        outs.append(torch.einsum("kgmn,knd->mkgd", p, v).reshape(m, -1, D))
    return torch.cat(outs)
