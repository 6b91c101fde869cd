"""Cosine and sine tables of rotary positions, scaled for long contexts.

Pair ``i`` of a rotary dimension ``R`` turns by ``position * f_i``, ``f_i = base ** (-2 i / R)``. A table is
float32 ``[positions, R]``: the cosines of every pair, then the sines. It is computed in 64 bits, since
``position * f_i`` of a long context has no fraction left in 32, and rounded once.
"""

from __future__ import annotations

import math
from collections.abc import Mapping

import torch


def rotary_frequencies(
    rotary_dim: int, base: float = 10000.0, scaling: Mapping[str, object] | None = None
) -> tuple[torch.Tensor, float]:
    """The frequencies ``f_i`` (float64 ``[R / 2]``) and the factor on cosines and sines.

    ``scaling`` is a model configuration's ``rope_scaling``, by its ``rope_type`` (or ``type``):

    * ``linear``: positions divided by ``factor``;
    * ``llama3``: frequencies whose wavelength exceeds ``original_max_position_embeddings /
      low_freq_factor`` divided by ``factor``, those below ``original / high_freq_factor`` kept, and a
      linear mix by ``original / wavelength`` between them;
    * ``yarn``: a pair that turns ``beta_fast`` times or more over the original context kept, one that
      turns ``beta_slow`` times or less divided by ``factor``, a linear ramp over the pair's number
      between them, its ends rounded outwards to whole pairs unless ``truncate`` is false; cosines and
      sines times ``attention_factor``, by default ``m(mscale) / m(mscale_all_dim)`` where the configuration
      has both and ``m(1)`` where it has neither, ``m(s) = 0.1 s ln(factor) + 1``. One of the two
      alone, and ``attn_factor`` and ``extrapolation_factor`` other than 1, are refused.
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError("rotary dimension must be even and positive")
    if not base > 0.0:
        raise ValueError("base must be positive")
    pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    frequencies = base ** (-pair / rotary_dim)
    if scaling is None:
        return frequencies, 1.0
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind == "default":
        return frequencies, 1.0
    if kind not in ("linear", "llama3", "yarn"):
        raise ValueError(f"unknown rope scaling type: {kind}")
    factor = float(scaling["factor"])
    if not factor >= 1.0:
        raise ValueError("the factor of a rope scaling must be at least 1")
    if kind == "linear":
        return frequencies / factor, 1.0
    original = float(scaling["original_max_position_embeddings"])
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not high > low:
            raise ValueError("high_freq_factor must exceed low_freq_factor")
        turns = original * frequencies / (2 * math.pi)
        kept = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return frequencies * (kept + (1.0 - kept) / factor), 1.0
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

    def pair_of(turns: float) -> float:
        """The (fractional) number of the pair that turns so often over the original context."""
        return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    for other in ("attn_factor", "extrapolation_factor"):
        if scaling.get(other) not in (None, 1):
            raise ValueError(f"unsupported key of a yarn rope scaling: {other}")
    low, high = pair_of(fast), pair_of(slow)
    if scaling.get("truncate", True):
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, rotary_dim - 1)
    ramp = ((pair / 2 - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
    attention = scaling.get("attention_factor")
    if attention is not None:
        attention = float(attention)
    else:
        attention = 0.1 * math.log(factor) + 1.0
        mscale, mscale_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
        if (mscale is None) != (mscale_all is None):
            raise ValueError("mscale and mscale_all_dim of a yarn rope scaling must be given together")
        if mscale is not None:
            attention = (0.1 * float(mscale) * math.log(factor) + 1.0) / (0.1 * float(mscale_all) * math.log(factor) + 1.0)
    return frequencies * ((1.0 - ramp) + ramp / factor), attention


def rotary_cos_sin_cache(
    rotary_dim: int,
    max_position: int,
    base: float = 10000.0,
    scaling: Mapping[str, object] | None = None,
    device: torch.device | str = "cuda",
) -> torch.Tensor:
    """The table of positions ``0 .. max_position - 1``, for :func:`~.extension.rotary_embedding`."""
    if max_position < 1:
        raise ValueError("max_position must be positive")
    frequencies, factor = rotary_frequencies(rotary_dim, base, scaling)
    position = torch.arange(max_position, dtype=torch.float64, device=device)
    angle = position[:, None] * frequencies.to(device)
    return (torch.cat([angle.cos(), angle.sin()], dim=1) * factor).to(torch.float32)
