"""Rotary frequencies, with the usual scalings for long contexts.

After an eviction a token's place in the cache is no longer its position in the text, so a
decode step turns its queries and keys by their true positions
(``ops.block_tables`` gives them, ``ops.rotary`` turns by them).  The frequencies are held in
float64: at position 10^6 a float32 frequency would put the angle off by 0.06.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch


_KEYS = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "finetuned", "mrope_section", "factor",
         "original_max_position_embeddings", "low_freq_factor", "high_freq_factor", "beta_fast", "beta_slow",
         "attention_factor", "mscale", "mscale_all_dim", "truncate"}


def _option(scaling: dict, key: str, default: float) -> float:
    """A number of the dictionary; a key that is absent or None is the default."""
    value = scaling.get(key)
    return default if value is None else float(value)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None,
                       seq_len: Optional[int] = None, device=None) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, factor)``: float64 ``[rotary_dim / 2]`` radians per position of each pair,
    ``base ** (-2 i / rotary_dim)`` before scaling, and the factor on cosine and sine.

    ``scaling``: a model config's ``rope_scaling`` dictionary.  ``rope_type`` (or ``type``):

    * ``"default"``: none;
    * ``"linear"``: every frequency divided by ``factor`` (position interpolation);
    * ``"dynamic"``: the base stretched so that ``seq_len`` tokens fit where
      ``original_max_position_embeddings`` did (NTK-aware), once ``seq_len`` is longer;
    * ``"llama3"``: wavelengths above ``original_max_position_embeddings / low_freq_factor`` are
      divided by ``factor``, those below ``.. / high_freq_factor`` stay, a smooth blend between;
    * ``"yarn"``: the same idea by pair index, a linear ramp between the pairs that make
      ``beta_fast`` and ``beta_slow`` turns over ``original_max_position_embeddings`` (rounded
      outwards to whole pairs unless ``truncate`` is false), with cosine and sine times
      ``attention_factor``; without one, by ``mscale(m) = 0.1 m ln(factor) + 1``: the ratio
      ``mscale(mscale) / mscale(mscale_all_dim)`` where the dictionary has both, else ``mscale(1)``.

    A key that none of these read raises ``ValueError``, rather than being left out quietly.
    ``rope_theta``, if it is there, must be ``base``; ``partial_rotary_factor`` is the caller's
    (``rotary_dim``), and ``finetuned`` and ``mrope_section`` say nothing of the frequencies.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    if not base > 0:
        raise ValueError("base must be positive")
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    unknown = sorted(set(scaling) - _KEYS)
    if unknown:
        raise ValueError(f"rope_scaling keys that are not understood: {unknown}")
    if scaling.get("rope_theta") is not None and float(scaling["rope_theta"]) != float(base):
        raise ValueError(f"rope_theta {scaling['rope_theta']} is not the base {base}")
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    freq = float(base) ** -exponent
    if kind == "default":
        return freq.to(device), 1.0
    if kind not in ("linear", "dynamic", "llama3", "yarn"):
        raise ValueError(f"unknown rope_type {kind!r}")
    by = float(scaling["factor"])
    if not by >= 1.0:
        raise ValueError("the scaling factor must be at least 1")
    if kind == "linear":
        return (freq / by).to(device), 1.0
    original = float(scaling["original_max_position_embeddings"])
    if kind == "dynamic":
        length = max(float(seq_len or 0), original)
        if rotary_dim > 2:
            stretched = base * (by * length / original - (by - 1.0)) ** (rotary_dim / (rotary_dim - 2.0))
            freq = stretched ** -exponent
        return freq.to(device), 1.0
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = original * freq / (2.0 * math.pi)            # whole turns over the original length
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return (freq * (keep + (1.0 - keep) / by)).to(device), 1.0
    fast, slow = _option(scaling, "beta_fast", 32.0), _option(scaling, "beta_slow", 1.0)

    def pair_of(turns: float) -> float:   # the (fractional) pair that makes so many turns
        return rotary_dim * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    def mscale(m: float) -> float:
        return 0.1 * m * math.log(by) + 1.0

    first, last = pair_of(fast), pair_of(slow)
    if scaling.get("truncate", True):
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rotary_dim - 1)
    ramp = (torch.arange(rotary_dim // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)
    keep = 1.0 - ramp.clamp(0.0, 1.0)
    factor = scaling.get("attention_factor")
    if factor is None:
        over, under = _option(scaling, "mscale", 0.0), _option(scaling, "mscale_all_dim", 0.0)
        if bool(over) != bool(under):
            raise ValueError("mscale and mscale_all_dim are given together or not at all")
        factor = mscale(over) / mscale(under) if over else mscale(1.0)
    return (freq * (keep + (1.0 - keep) / by)).to(device), float(factor)
