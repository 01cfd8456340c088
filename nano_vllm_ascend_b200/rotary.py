"""Turns per position of rotary embeddings, for ``ops.rotary``.

The reference makes cosine and sine tables of one base
(src/nanovllm_ascend/layers/rotary_embedding.py:20-40); here the frequencies
themselves are kept, in 64 bits, and the kernel makes the angles, so that no
position is out of a table. Long contexts scale them:

* ``linear``: every position counts 1 / factor;
* ``ntk``: the base grows, so that the slowest pair turns 1 / factor as far and
  the fastest keeps its turns;
* ``yarn`` (Peng et al., "YaRN: Efficient Context Window Extension of Large
  Language Models"): pairs that turn fewer than ``beta_slow`` times within
  ``original_max_position`` are scaled by 1 / factor, those above ``beta_fast``
  kept, with a ramp over the pairs between; the result is multiplied by
  ``attention_factor`` (0.1 ln(factor) + 1 by default);
* ``wavelength``: the same by wavelength: kept below ``original_max_position /
  high_freq_factor``, scaled above ``original_max_position / low_freq_factor``,
  and blended by the turns between.
"""

from __future__ import annotations

import math

import torch

_KEYS = {
    "linear": ({"factor"}, set()),
    "ntk": ({"factor"}, set()),
    "yarn": ({"factor", "original_max_position"}, {"beta_fast", "beta_slow", "attention_factor"}),
    "wavelength": ({"factor", "original_max_position", "low_freq_factor", "high_freq_factor"}, set()),
}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """(inv_freq, attention_scale) for ``ops.rotary``: radians a position of each of the rotary_dim / 2 pairs (float64),
    and what the turned pairs are multiplied by. ``scaling``: {"type": one of the above, ...}, or None."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} is not even and positive")
    if not 1 < base < math.inf:
        raise ValueError(f"base {base} is not above 1 and finite")
    half = rotary_dim // 2
    pair = torch.arange(half, dtype=torch.float64) / half
    inv, scale = float(base) ** -pair, 1.0
    if scaling is not None:
        kind = scaling.get("type")
        if kind not in _KEYS:
            raise ValueError(f"scaling type {kind!r} is none of {sorted(_KEYS)}")
        needed, more = _KEYS[kind]
        given = set(scaling) - {"type"}
        if not needed <= given or not given <= needed | more:
            raise ValueError(f"{kind} scaling takes {sorted(needed)}" + (f" and may have {sorted(more)}" if more else "")
                             + f", got {sorted(given)}")
        factor = float(scaling["factor"])
        if not 1 <= factor < math.inf:
            raise ValueError(f"scaling factor {factor} is below 1 or not finite")
        length = float(scaling.get("original_max_position", 1))
        if not 0 < length < math.inf:
            raise ValueError(f"original_max_position {length} is not positive and finite")
        if kind == "linear":
            inv = inv / factor
        elif kind == "ntk":
            if half > 1:
                inv = (base * factor ** (half / (half - 1))) ** -pair
        elif kind == "yarn":
            fast, slow = float(scaling.get("beta_fast", 32)), float(scaling.get("beta_slow", 1))
            if not 0 < slow <= fast:
                raise ValueError(f"beta_slow {slow} is not positive or above beta_fast {fast}")

            def pair_of(turns: float) -> float:  # the pair that turns so often within the length
                return half * math.log(length / (turns * 2 * math.pi)) / math.log(base)

            low = max(math.floor(pair_of(fast)), 0)
            high = min(math.ceil(pair_of(slow)), rotary_dim - 1)
            ramp = ((torch.arange(half, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
            inv = inv / factor * ramp + inv * (1 - ramp)
            given_scale = scaling.get("attention_factor")
            scale = float(given_scale) if given_scale is not None else 0.1 * math.log(factor) + 1
        else:
            slow, fast = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
            if not 0 < slow < fast:
                raise ValueError(f"low_freq_factor {slow} is not below high_freq_factor {fast}")
            keep = ((length * inv / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
            inv = inv * keep + inv / factor * (1 - keep)
    return inv.to(device) if device is not None else inv, scale
