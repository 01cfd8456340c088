"""The 8-bit KV pool restated in numpy (its attention is that of fp4_oracle).

The reference has no counterpart: its pool is bf16. The definition restated
here: 16 tokens of one KV head make a unit of 4128 bytes, with one exponent for
K and one for V; a value is e4m3(code) * 2^exponent. Rows written into a unit
raise its exponent to the least e in [-40, 40] with amax <= 448 * 2^e over their
finite values, and the unit's other rows are rounded again from their values;
a call that writes the unit's first token takes e from its own rows and makes
the others zeros. Codes round to nearest, ties to even, and saturate; a row with
a NaN is NaN throughout.
"""

from __future__ import annotations

import math

import numpy as np

from oracle.fp4_oracle import _round, e4m3_byte, e4m3_value

D = 128
UNIT = 4128
LEAST, MOST = -40, 40
_PLACE = 128 * np.arange(16)[:, None] + 16 * ((np.arange(D) // 16)[None] ^ (np.arange(16) % 8)[:, None]) + np.arange(D) % 16


def exponent(amax: float) -> int:
    e = LEAST if amax == 0 else math.frexp(amax / 448)[1]
    if amax and amax <= 448 * 2.0 ** (e - 1):
        e -= 1
    return min(max(e, LEAST), MOST)


def codes(x: np.ndarray, e: int) -> np.ndarray:
    """Rows [..., 128] (float64) as e4m3 bytes over 2^e."""
    with np.errstate(invalid="ignore"):
        y = np.clip(x / 2.0 ** e, -1e6, 1e6)
    mag = np.minimum(_round(np.abs(np.nan_to_num(y)), 4, -6), 448.0)
    byte = e4m3_byte(mag) | (np.signbit(x).astype(np.uint8) << 7)
    return np.where(np.isnan(x).any(-1, keepdims=True), np.uint8(0x7F), byte)


def values(byte: np.ndarray, e) -> np.ndarray:
    return e4m3_value(byte & 0x7F) * np.where(byte & 0x80, -1.0, 1.0) * 2.0 ** np.asarray(e, dtype=np.float64)


def _exps(unit: np.ndarray) -> np.ndarray:
    return unit[..., 4096:4104].copy().view(np.int32)


def append(pool: np.ndarray, key: np.ndarray, value: np.ndarray, slots: np.ndarray) -> None:
    """One call: rows [T, KVH, 128] into pool uint8 [NB, KVH, BS / 16, 4128], in place; slots outside it are skipped."""
    nb, kvh, upb, _ = pool.shape
    members: dict[int, dict[int, int]] = {}
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < nb * upb * 16:
            members.setdefault(s // 16, {})[s % 16] = i
    for u, rows in members.items():
        off, tok = list(rows), list(rows.values())
        for h in range(kvh):
            unit = pool[u // upb, h, u % upb]
            for part, x in enumerate((key, value)):
                new = x[tok, h].astype(np.float64)
                old = int(_exps(unit)[part])
                e = exponent(float(np.abs(np.where(np.isfinite(new), new, 0)).max()))
                place = 2048 * part + _PLACE
                if 0 in rows:
                    unit[place] = 0
                elif e > old:
                    unit[place] = codes(values(unit[place], old), e)
                else:
                    e = old
                unit[place[off]] = codes(new, e)
                unit[4096 + 4 * part:4100 + 4 * part] = np.array([e], dtype=np.int32).view(np.uint8)


def rows(pool: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Every slot's K and V rows, float64 [NB * BS, KVH, 128]."""
    nb, kvh, upb, _ = pool.shape
    e = _exps(pool)
    out = []
    for part in (0, 1):
        v = values(pool[..., 2048 * part + _PLACE], e[..., part, None, None])  # [NB, KVH, U, 16, 128]
        out.append(v.transpose(0, 2, 3, 1, 4).reshape(nb * upb * 16, kvh, D))
    return out[0], out[1]
