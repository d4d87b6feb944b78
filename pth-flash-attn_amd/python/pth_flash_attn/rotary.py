"""Frequencies of rotary positions, for ``ops.rotary_embedding``.

A pair of columns turns by its position times its frequency. The op takes the
frequencies as 64-bit fractions of a turn per position, laid out once: the
product with a position, wrapped to 64 bits, is the angle's place in the circle,
exact at every position, without a table that would have to reach to the last.
"""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch

SCALINGS = ("none", "linear", "base", "ramp", "smooth", "factors")


def rotary_frequencies(
    rot_dim: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
    original_max_position: int = 4096, fast_turns: float = 32.0, slow_turns: float = 1.0,
    low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
    factors: Sequence[float] | None = None,
) -> list[float]:
    """Radians per position of the ``rot_dim / 2`` pairs, base^(-2 j / rot_dim), scaled:

    * ``none``;
    * ``linear``: all divided by ``factor`` (positions interpolated);
    * ``base``: the base grows so that the slowest pair is divided by ``factor``
      and the fastest stays (the NTK-aware scaling);
    * ``ramp``: pairs that make ``fast_turns`` turns or more within
      ``original_max_position`` stay, those of ``slow_turns`` or fewer are divided
      by ``factor``, between them (by pair number) a linear mix (YaRN);
    * ``smooth``: pairs whose wavelength is below original_max_position /
      ``high_freq_factor`` stay, above original_max_position / ``low_freq_factor``
      are divided, between them a mix linear in the turns made;
    * ``factors``: pair j divided by ``factors[j]``.
    """
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be even and positive, got {rot_dim}")
    if not (base > 0 and math.isfinite(base) and factor > 0 and math.isfinite(factor)):
        raise ValueError("base and factor must be positive and finite")
    if original_max_position < 1:
        raise ValueError("original_max_position must be positive")
    half = rot_dim // 2
    if scaling == "base":
        if rot_dim < 4:
            raise ValueError("scaling 'base' needs rot_dim of 4 or more")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    f = [base ** (-2.0 * j / rot_dim) for j in range(half)]
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "ramp":
        if not (fast_turns > slow_turns > 0 and base > 1):
            raise ValueError("scaling 'ramp' needs fast_turns > slow_turns > 0 and base > 1")

        def pair_of(turns: float) -> float:
            return (rot_dim * math.log(original_max_position / (turns * 2 * math.pi))
                    / (2 * math.log(base)))

        lo = max(math.floor(pair_of(fast_turns)), 0)
        hi = min(math.ceil(pair_of(slow_turns)), rot_dim - 1)
        out = []
        for j, x in enumerate(f):
            scaled = min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            out.append(x * (1.0 - scaled) + x / factor * scaled)
        return out
    if scaling == "smooth":
        if not high_freq_factor > low_freq_factor > 0:
            raise ValueError("scaling 'smooth' needs high_freq_factor > low_freq_factor > 0")
        out = []
        for x in f:
            turns = original_max_position * x / (2 * math.pi)
            keep = (turns - low_freq_factor) / (high_freq_factor - low_freq_factor)
            keep = min(max(keep, 0.0), 1.0)
            out.append(x * keep + x / factor * (1.0 - keep))
        return out
    if scaling == "factors":
        if factors is None or len(factors) != half or not all(x > 0 for x in factors):
            raise ValueError(f"scaling 'factors' needs {half} positive factors")
        return [x / d for x, d in zip(f, factors)]
    return f


def rotary_turns(rot_dim: int, *, scaling: str = "none", factor: float = 1.0,
                 original_max_position: int = 4096, attention_scale: float | None = None,
                 device: str | torch.device = "cuda", **kw) -> tuple[torch.Tensor, float]:
    """(turns, scale) of ``ops.rotary_embedding``: int64 [rot_dim / 2] on ``device``,
    2^64 times the turns per position, and the factor of queries and keys.

    ``scale`` is ``attention_scale``, or what the scaling is published with: 0.1
    ln(factor) + 1 for ``ramp``, sqrt(1 + ln(factor) / ln(original_max_position))
    for ``factors`` (where ``factor``, the context's extension, is above 1), 1
    otherwise. The keywords are those of ``rotary_frequencies``.
    """
    try:
        f = rotary_frequencies(rot_dim, scaling=scaling, factor=factor,
                               original_max_position=original_max_position, **kw)
        # A float times 2^64 is a whole number or rounds to one of 64 bits.
        turns = [round(math.ldexp(x / (2 * math.pi), 64)) % (1 << 64) for x in f]
    except OverflowError:
        raise ValueError("the frequencies must be finite, and 2^64 times them") from None
    signed = [t - (1 << 64) if t >= 1 << 63 else t for t in turns]
    if attention_scale is None:
        attention_scale = 1.0
        if scaling == "ramp" and factor > 1:
            attention_scale = 0.1 * math.log(factor) + 1.0
        elif scaling == "factors" and factor > 1:
            if original_max_position == 1:
                raise ValueError("scaling 'factors' needs original_max_position above 1 or an "
                                 "attention_scale")
            attention_scale = math.sqrt(1.0 + math.log(factor) / math.log(original_max_position))
    return torch.tensor(signed, dtype=torch.int64).to(device), float(attention_scale)
