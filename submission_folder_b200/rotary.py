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
      ``beta_fast`` and ``beta_slow`` turns over ``original_max_position_embeddings``, with
      cosine and sine times ``attention_factor`` (default ``0.1 ln(factor) + 1``).
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    if not base > 0:
        raise ValueError("base must be positive")
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
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
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

    def pair_of(turns: float) -> float:   # the (fractional) pair that makes so many turns
        return rotary_dim * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    first = max(math.floor(pair_of(fast)), 0)
    last = min(math.ceil(pair_of(slow)), rotary_dim - 1)
    ramp = (torch.arange(rotary_dim // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)
    keep = 1.0 - ramp.clamp(0.0, 1.0)
    factor = scaling.get("attention_factor")
    factor = 0.1 * math.log(by) + 1.0 if factor is None else float(factor)
    return (freq * (keep + (1.0 - keep) / by)).to(device), factor
