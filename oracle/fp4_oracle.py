"""The 4-bit KV pool restated in numpy (the format) and 64-bit torch (attention).

The reference has no counterpart: its pool is bf16. The definition restated
here: a row's 128 dims are 8 groups of 16; a group of x / constant has the
scale s = e4m3(amax / 6) and the codes e2m1(x / s), rounded to nearest, ties
to even, saturating; it stands for constant * s * code. 16 tokens of one KV
head make a unit of 2304 bytes.
"""

from __future__ import annotations

import numpy as np
import torch

D = 128
UNIT = 2304
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _round(x: np.ndarray, bits: int, low: int) -> np.ndarray:
    """To ``bits`` significant bits, with the step of 2**low below it; ties to even."""
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.maximum(np.floor(np.log2(np.abs(x))), low)
    e = np.where(np.isfinite(e), e, low)
    step = np.exp2(e - (bits - 1))
    return np.rint(x / step) * step


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Rows [..., 128] (float64) -> codes uint8 [..., 128] and scales float64 [..., 8] (NaN for a group with one)."""
    g = x.reshape(*x.shape[:-1], 8, 16).astype(np.float64)
    amax = np.abs(g).max(-1)
    s = np.minimum(_round(np.minimum(amax / 6, 1e4), 4, -6), 448.0)
    s = np.where(np.isnan(amax), np.nan, s)
    with np.errstate(divide="ignore", invalid="ignore"):
        a = np.where(s[..., None] > 0, np.abs(g) / s[..., None], 0.0)
    a = np.minimum(_round(np.minimum(a, 1e4), 2, 0), 6.0)
    code = np.searchsorted(LEVELS, a).astype(np.uint8) | (np.signbit(g).astype(np.uint8) << 3)
    return code.reshape(x.shape), s


def values(code: np.ndarray, s: np.ndarray) -> np.ndarray:
    mag = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    return (mag.reshape(*code.shape[:-1], 8, 16) * s[..., None]).reshape(code.shape)


def e4m3_byte(s: np.ndarray) -> np.ndarray:
    """The e4m3 byte of non-negative representable values (NaN: 0x7f)."""
    table = np.array([(m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)])
    table[127] = np.inf
    out = np.searchsorted(table, np.where(np.isnan(s), 0, s)).astype(np.uint8)
    return np.where(np.isnan(s), np.uint8(0x7F), out).astype(np.uint8)


def e4m3_value(b: np.ndarray) -> np.ndarray:
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e.astype(np.float64) - 7))
    return np.where(b == 0x7F, np.nan, v)


def _places(is_v: bool):
    """(byte of each token's dim pairs [16, 64], byte of each token's scales [16, 8]) in a unit."""
    i = np.arange(16)[:, None]
    d, j = np.arange(0, D, 2)[None], np.arange(8)[None]
    grp, r = d // 16, d % 16
    if is_v:
        return 1152 + 256 * (i // 4) + 32 * (r // 2) + 8 * (i % 4) + grp, 2176 + 32 * (i // 4) + 4 * j + i % 4
    return 64 * i + 16 * (r // 4) + 2 * grp + r % 4 // 2, 1024 + 8 * i + j


def append(pool: np.ndarray, key: np.ndarray, value: np.ndarray, slots: np.ndarray, k_scale: float = 1.0,
           v_scale: float = 1.0) -> None:
    """Rows [T, KVH, 128] into pool uint8 [NB, KVH, BS / 16, 2304], in place; slots outside it are skipped."""
    nb, kvh, units, _ = pool.shape
    bs = units * 16
    ok = (slots >= 0) & (slots < nb * bs)
    sl = slots[ok]
    blk, unit, i = sl // bs, sl % bs // 16, sl % 16
    for is_v, x, c in ((False, key, k_scale), (True, value, v_scale)):
        at, sc = _places(is_v)
        code, s = quantise(x[ok].astype(np.float64) / c)
        byte = code[..., 0::2] | (code[..., 1::2] << 4)
        h = np.arange(kvh)[None, :, None]
        pool[blk[:, None, None], h, unit[:, None, None], at[i][:, None, :]] = byte
        pool[blk[:, None, None], h, unit[:, None, None], sc[i][:, None, :]] = e4m3_byte(s)


def rows(pool: np.ndarray, k_scale: float = 1.0, v_scale: float = 1.0) -> tuple[np.ndarray, np.ndarray]:
    """Every slot's K and V rows, float64 [NB * BS, KVH, 128]."""
    nb, kvh, units, _ = pool.shape
    out = []
    for is_v, c in ((False, k_scale), (True, v_scale)):
        at, sc = _places(is_v)
        b = pool[..., at]  # [NB, KVH, U, 16, 64]
        code = np.stack([b & 15, b >> 4], -1).reshape(nb, kvh, units, 16, D)
        v = values(code, e4m3_value(pool[..., sc])) * c
        out.append(v.transpose(0, 2, 3, 1, 4).reshape(nb * units * 16, kvh, D))
    return out[0], out[1]


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """Bottom-right causal attention of q [m, H, 128] over k, v [n, KVH, 128] (float64).

    Returns the output and the same weights' mean of |v|, by which rounding of
    the weights is bounded. Rows that see no key are zeros.
    """
    m, h, _ = q.shape
    n, kvh, _ = k.shape
    qg = q.double().view(m, kvh, h // kvh, D)
    s = torch.einsum("mkgd,nkd->kgmn", qg, k) * scale
    hidden = torch.arange(n, device=q.device) > n - m + torch.arange(m, device=q.device)[:, None]
    p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1).nan_to_num(0.0) if n else s
    if n:
        p = torch.where(torch.isnan(s).any(-1, keepdim=True) & ~hidden.all(-1, keepdim=True), float("nan"), p)
    o = torch.einsum("kgmn,nkd->mkgd", p, v).reshape(m, h, D)
    a = torch.einsum("kgmn,nkd->mkgd", p, v.abs()).reshape(m, h, D)
    return o, a


def norm_rope(x: np.ndarray, w: np.ndarray, eps: float, cos: np.ndarray, sin: np.ndarray) -> torch.Tensor:
    """Rows [T, heads, 128] (float32 holding bf16) -> normalised and rotated bf16 rows; cos/sin [T, 128] float32.

    The mean square in 64 bits, it plus eps and its reciprocal root each
    rounded to 32; the products by it and by w rounded to 32 bits; the norm's
    result, cos and sin rounded to bf16, then the rotation's sum to 32 bits
    and to bf16.
    """
    ms = ((x.astype(np.float64) ** 2).sum(-1, keepdims=True) / D + np.float64(np.float32(eps))).astype(np.float32)
    rinv = (1.0 / np.sqrt(ms.astype(np.float64))).astype(np.float32)
    y = torch.from_numpy((x * rinv).astype(np.float32) * w.astype(np.float32)).to(torch.bfloat16).float()
    c, s = (torch.from_numpy(t).to(torch.bfloat16).float()[:, None] for t in (cos, sin))
    half = torch.cat([-y[..., D // 2:], y[..., :D // 2]], -1)
    return (y * c + half * s).to(torch.bfloat16)
