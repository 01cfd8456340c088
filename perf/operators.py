"""The operators of the 4-bit KV cache, as cases that can be timed and compared.

A layer's pool is uint8 [num_blocks, kv_heads, block_size / 16, 2304]: 16 tokens
of one KV head make a unit of

    K codes  [16 tokens][4 t][8 groups][2 h]   bytes, dims 16 * group + 4 * t + 2 * h + {0 low, 1 high nibble}
    K scales [16 tokens][8 groups]             e4m3
    V codes  [4 quads][8 g][4 tokens][8 groups] bytes, dims 16 * group + 2 * g + {0 low, 1 high nibble}
    V scales [4 quads][8 groups][4 tokens]     e4m3

A group is 16 neighbouring dims of a row: its scale is s = e4m3(amax / 6), its
codes e2m1(x / s), its values k_scale * s * code (v_scale for V).
``run`` computes the operators in elementary torch operations, or, with ``own``
set, through the framework's entry points.
"""

import math
import random

import torch

own = False

D = 128
UNIT = 2304
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # one decode step's rows of 32 sequences: latency
        dict(name="append 32", op="append", tokens=32, kv_heads=8, block_size=16, blocks=16, dtype="bf16", seed=1),
        # rows of another model's heads, fp16, an odd number of tokens
        dict(name="append 777 fp16", op="append", tokens=777, kv_heads=5, block_size=64, blocks=20, dtype="fp16",
             seed=2),
        # one prefill step: 32 requests of 256 new tokens
        dict(name="append 8192", op="append", tokens=8192, kv_heads=8, block_size=128, blocks=66, dtype="bf16",
             seed=3),
        # the attention prologue of a decode step
        dict(name="norm rope append 32", op="norm", tokens=32, heads=16, kv_heads=8, block_size=16, blocks=16, seed=4),
        # the attention prologue of a prefill step
        dict(name="norm rope append 8192", op="norm", tokens=8192, heads=16, kv_heads=8, block_size=128, blocks=66,
             seed=5),
        # four short sequences, up to 513 tokens: latency
        dict(name="decode 4", op="decode", batch=4, lo=37, hi=513, heads=16, kv_heads=8, block_size=128, seed=6),
        # 32 requests of 256 prompt and up to 2048 generated tokens
        dict(name="decode 32", op="decode", batch=32, lo=256, hi=2304, heads=16, kv_heads=8, block_size=128, seed=7),
        # a large batch of long contexts
        dict(name="decode 256", op="decode", batch=256, lo=2048, hi=6144, heads=16, kv_heads=8, block_size=128, seed=8),
        # ragged, some sequences empty, five query heads a KV head, small blocks
        dict(name="decode 77 ragged", op="decode", batch=77, lo=0, hi=1500, heads=10, kv_heads=2, block_size=32,
             seed=9),
        # two sequences at the longest position, four query heads a KV head
        dict(name="decode 2 long", op="decode", batch=2, lo=40959, hi=40960, heads=32, kv_heads=8, block_size=128,
             seed=10),
        # 32 requests of 256 new tokens over a cached prefix of 768
        dict(name="prefill 32 cached", op="prefill", batch=32, q_lo=256, q_hi=256, c_lo=768, c_hi=768, heads=16,
             kv_heads=8, block_size=128, seed=11),
        # a few ragged requests, odd group size, small blocks
        dict(name="prefill 5 ragged", op="prefill", batch=5, q_lo=1, q_hi=300, c_lo=0, c_hi=1000, heads=9, kv_heads=3,
             block_size=64, seed=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "norm", "decode", "decode", "prefill", "prefill"])
    bs = rng.choice([16, 32, 64, 128, 256])
    kvh = rng.choice([1, 2, 3, 4, 5, 6, 8])
    seed = rng.randrange(1 << 30)
    if op in ("append", "norm"):
        tokens = _log(rng, 1, 8192)
        spare = rng.randrange(3)
        blocks = -(-tokens // bs) + spare
        if op == "append":
            return dict(op=op, tokens=tokens, kv_heads=kvh, block_size=bs, blocks=blocks,
                        dtype=rng.choice(["bf16", "fp16"]), seed=seed)
        return dict(op=op, tokens=tokens, heads=kvh * rng.randint(1, 4), kv_heads=kvh, block_size=bs, blocks=blocks,
                    seed=seed)
    if op == "decode":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, min(40960, 1 << 20) if batch <= 16 else max(2, (1 << 20) // batch))
        lo = rng.choice([0, 1, hi // 2, hi])
        return dict(op=op, batch=batch, lo=min(lo, hi), hi=hi, heads=kvh * rng.randint(1, 8), kv_heads=kvh,
                    block_size=bs, seed=seed)
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
    """The lengths of the case's sequences: contexts (decode), or new and cached tokens (prefill)."""
    r = random.Random(case["seed"])
    if case["op"] == "decode":
        return [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    c = [r.randint(case["c_lo"], case["c_hi"]) for _ in range(case["batch"])]
    return q, c


def work(case):
    op, kvh = case["op"], case["kv_heads"]
    if op in ("append", "norm"):
        t, slots = case["tokens"], case["blocks"] * case["block_size"]
        # the rows in and their codes out, then every row of the pool read back
        b = t * (kvh * (2 * 256 + 144) + 8) + slots * (kvh * (144 + 2 * 256) + 8)
        f = t * kvh * 2 * D * 4
        if op == "norm":
            b += t * (case["heads"] * 2 * 256 + 8) + min(t, 40960) * 1024
            f += t * (case["heads"] + kvh) * D * 8
        return {"bytes": b, "flops": f}
    h, bs = case["heads"], case["block_size"]
    if op == "decode":
        ctx = _lens(case)
        b = sum(ctx) * kvh * 144 + 2 * len(ctx) * h * 256 + sum(-(-n // bs) for n in ctx) * 4 + len(ctx) * 4
        return {"bytes": b, "flops": 4 * D * h * sum(ctx)}
    q, c = _lens(case)
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(q, c))
    b = sum(n + p for n, p in zip(q, c)) * kvh * 144 + 2 * sum(q) * h * 256
    return {"bytes": b, "flops": 4 * D * h * pairs}


# ------------------------------------------------------------ plain parts ---
def _quantise(x):
    """x [..., 128] float32 -> (codes uint8 [..., 128], scales e4m3 [..., 8])."""
    g = x.unflatten(-1, (8, 16))
    s = (g.abs().amax(-1) / 6).clamp(max=448).to(torch.float8_e4m3fn)
    a = g.abs() / s.float().unsqueeze(-1)
    a = torch.where(s.float().unsqueeze(-1) > 0, a, torch.zeros_like(a))
    # midpoints between neighbouring levels; a tie goes to the even code
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    return (code | (torch.signbit(g).to(torch.uint8) << 3)).flatten(-2), s


def _values(code, s):
    """codes uint8 [..., 128], scales e4m3 [..., 8] -> float32 [..., 128]."""
    lut = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float32, device=code.device)
    return (lut[code.int()].unflatten(-1, (8, 16)) * s.float().unsqueeze(-1)).flatten(-2)


def _pack(kc, ks, vc, vs):
    """Codes [n, 16 tokens, 128] and scales [n, 16, 8] of K and V -> units uint8 [n, 2304]."""
    n = kc.shape[0]
    kb = kc.view(n, 16, 8, 4, 2, 2).permute(0, 1, 3, 2, 4, 5)  # token, t, group, h, nibble
    vb = vc.view(n, 4, 4, 8, 8, 2).permute(0, 1, 4, 2, 3, 5)   # quad, g, token, group, nibble
    kb, vb = ((b[..., 0] | (b[..., 1] << 4)).reshape(n, 1024) for b in (kb, vb))
    return torch.cat([kb, ks.view(torch.uint8).reshape(n, 128), vb,
                      vs.view(torch.uint8).view(n, 4, 4, 8).permute(0, 1, 3, 2).reshape(n, 128)], dim=1)


def _unpack(units):
    """Units uint8 [..., 2304] -> K and V values float32 [..., 16, 128]."""
    lead, u = units.shape[:-1], units.reshape(-1, UNIT)
    n = u.shape[0]
    kb, vb = u[:, :1024].view(n, 16, 4, 8, 2), u[:, 1152:2176].view(n, 4, 8, 4, 8)
    kc = torch.stack([kb & 15, kb >> 4], -1).permute(0, 1, 3, 2, 4, 5).reshape(n, 16, D)
    vc = torch.stack([vb & 15, vb >> 4], -1).permute(0, 1, 3, 4, 2, 5).reshape(n, 16, D)
    ks = u[:, 1024:1152].contiguous().view(torch.float8_e4m3fn).view(n, 16, 8)
    vs = u[:, 2176:].reshape(n, 4, 8, 4).permute(0, 1, 3, 2).contiguous().view(torch.float8_e4m3fn).view(n, 16, 8)
    return _values(kc, ks).view(*lead, 16, D), _values(vc, vs).view(*lead, 16, D)


def _pool_rows(pool):
    """The pool's K and V as float32 rows [slots, kv_heads, 128]."""
    nb, kvh, u, _ = pool.shape
    return tuple(x.permute(0, 2, 3, 1, 4).reshape(nb * u * 16, kvh, D) for x in _unpack(pool))


def _gathered(pool, tables):
    """K and V values of each sequence's blocks, float32 [batch, kv_heads, tokens, 128]."""
    g = pool[tables.long()].transpose(1, 2)  # [batch, kv_heads, blocks, units, 2304]
    return tuple(x.flatten(2, 4) for x in _unpack(g))


# ----------------------------------------------------------------- inputs ---
def _random_pool(blocks, kvh, bs, gen, dev):
    """A pool whose K and V were normal before they were quantised."""
    pool = torch.empty(blocks * kvh * bs // 16, UNIT, dtype=torch.uint8, device=dev)
    for part in pool.split(1 << 18):
        x = torch.randn(2, part.shape[0], 16, D, generator=gen, device=dev).to(torch.bfloat16).float()
        (kc, ks), (vc, vs) = _quantise(x[0]), _quantise(x[1])
        part.copy_(_pack(kc, ks, vc, vs))
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


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + case["seed"])

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device=dev).to(dtype)

    op, kvh, bs = case["op"], case["kv_heads"], case["block_size"]
    st = dict(op=op)
    if op in ("append", "norm"):
        t, nb = case["tokens"], case["blocks"]
        st["pool"] = _random_pool(nb, kvh, bs, gen, dev)
        st["slots"] = torch.randperm(nb * bs, generator=gen, device=dev)[:t].contiguous()
        st["every"] = torch.arange(nb * bs, device=dev)
        if op == "append":
            dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float16
            st.update(k=randn(t, kvh, D, dtype=dtype), v=randn(t, kvh, D, dtype=dtype))
            return st
        h = case["heads"]
        qkv = randn(t, h + 2 * kvh, D)  # the fused projection's output: q, k and v are slices of it
        inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
        f = torch.outer(torch.arange(40960, dtype=torch.float64), inv)
        f = torch.cat((f, f), -1)
        st.update(q=qkv[:, :h], k=qkv[:, h:h + kvh], v=qkv[:, h + kvh:], wq=1 + 0.1 * randn(D), wk=1 + 0.1 * randn(D),
                  cos=f.cos().float().to(dev), sin=f.sin().float().to(dev), eps=1e-6,
                  pos=torch.randint(0, 40960, (t,), generator=gen, device=dev))
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
    if op in ("append", "norm"):
        k, v = st["k"].float(), st["v"].float()
        out = {}
        if op == "norm":
            out["q"], k = _norm_rope(st, st["q"], st["wq"]), _norm_rope(st, st["k"], st["wk"]).float()
        rows = _pool_rows(st["pool"])
        for name, pool, x in (("key", rows[0], k), ("value", rows[1], v)):
            pool[st["slots"]] = _values(*_quantise(x))
            out[name] = pool.to(st["k"].dtype)
        return out
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


def _norm_rope(st, x, w):
    """RMS norm of each head's row, rounded to bf16, then its rotation, as bf16."""
    # the mean square in 64 bits: the row's bf16 values do not hang on the order of the sum
    ms = (x.double().square().mean(-1, keepdim=True) + st["eps"]).float()
    y = (x.float() * ms.double().rsqrt().float() * w.float()).to(torch.bfloat16).float()
    c, s = (t[st["pos"]].to(torch.bfloat16).float().unsqueeze(1) for t in (st["cos"], st["sin"]))
    half = torch.cat([-y[..., D // 2:], y[..., :D // 2]], -1)
    return (y * c + half * s).to(torch.bfloat16)


def _run_own(st):
    from nano_vllm_ascend_b200 import ops_fp4

    op, pool = st["op"], st["pool"]
    if op == "append":
        ops_fp4.kv_append_fp4(pool, st["k"], st["v"], st["slots"])
        k, v = ops_fp4.kv_read_fp4(pool, st["every"], dtype=st["k"].dtype)
        return {"key": k, "value": v}
    if op == "norm":
        q = ops_fp4.qk_norm_rope_append_fp4(st["q"], st["k"], st["v"], st["wq"], st["wk"], st["eps"], st["cos"],
                                            st["sin"], st["pos"], pool, st["slots"])
        k, v = ops_fp4.kv_read_fp4(pool, st["every"])
        return {"q": q, "key": k, "value": v}
    out = torch.empty_like(st["q"])
    if op == "decode":
        if "ws" not in st:  # a user keeps one for all layers and steps
            size = ops_fp4.decode_fp4_workspace_bytes(st["q"].shape[1], pool.shape[1], D)
            st["ws"] = torch.zeros(size, dtype=torch.uint8, device=out.device)
        return ops_fp4.paged_decode_fp4(out, st["q"], pool, st["tables"], st["ctx"], st["scale"], st["ws"])
    return ops_fp4.paged_prefill_fp4(out, st["q"], pool, st["tables"], st["cu"], st["ctx"], st["max_q"], st["scale"])


# ------------------------------------------------------------------ exact ---
def _places(dev):
    """Byte (and nibble) of every token and dim, and the scale's byte, in a unit: K, then V."""
    i, d = torch.arange(16, device=dev)[:, None], torch.arange(D, device=dev)[None]
    j = d // 16
    k = 64 * i + 16 * (d % 16 // 4) + 2 * j + d % 4 // 2
    v = 1152 + 256 * (i // 4) + 32 * (d % 16 // 2) + 8 * (i % 4) + j
    return (k, 1024 + 8 * i + j), (v, 2176 + 32 * (i // 4) + 4 * j + i % 4)


def _e4m3(b):
    e, m = (b >> 3 & 15).double(), (b & 7).double()
    return torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2(e - 7))


def _stored64(pool):
    """[blocks, kv_heads, units, 2304] -> K and V float64 [blocks, kv_heads, units * 16, 128]."""
    both = []
    for at, sc in _places(pool.device):
        b = pool[..., at.reshape(-1)].long().unflatten(-1, (16, D))
        c = b >> 4 * (torch.arange(D, device=pool.device) % 2) & 15
        mag = torch.tensor(LEVELS, dtype=torch.float64, device=pool.device)[c & 7]
        x = torch.where(c >= 8, -mag, mag) * _e4m3(pool[..., sc.reshape(-1)].long().unflatten(-1, (16, D)))
        both.append(x.flatten(-3, -2))
    return both


def _round64(x, bits, low):
    """x to the nearest number of so many significant bits, and of no less than the step at 2^low; ties to even."""
    e = torch.floor(torch.log2(x.abs().clamp(min=1e-300))).clamp(min=low)
    step = torch.exp2(e - (bits - 1))
    return torch.round(x / step) * step


def _fake64(x):
    """The values that rows [..., 128] stand for once held in 4 bits."""
    g = x.unflatten(-1, (8, 16))
    s = _round64(g.abs().amax(-1, keepdim=True) / 6, 4, -6).clamp(max=448)
    q = torch.where(s > 0, g / torch.where(s > 0, s, 1.0), 0.0)
    return (_round64(q, 2, 0).clamp(-6, 6) * s).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    op, kvh = case["op"], case["kv_heads"]
    if op in ("append", "norm"):
        k, v, out = st["k"].double(), st["v"].double(), {}
        if op == "norm":
            c, s = (t[st["pos"]].bfloat16().double()[:, None] for t in (st["cos"], st["sin"]))

            def turned(x, w):
                x = x.double()
                y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + st["eps"]) * w.double()
                a, b = y.bfloat16().double().chunk(2, -1)  # the norm's result is bf16 by definition
                return torch.cat([a * c[..., :64] - b * s[..., :64], b * c[..., 64:] + a * s[..., 64:]], -1)

            out["q"], k = turned(st["q"], st["wq"]), turned(st["k"], st["wk"]).bfloat16().double()
        for name, rows, x in zip(("key", "value"), _stored64(st["pool"]), (k, v)):
            rows = rows.transpose(1, 2).reshape(-1, kvh, D).clone()
            rows.index_copy_(0, st["slots"], _fake64(x))
            out[name] = rows
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
