"""Rotary frequencies, with the scalings that stretch them for long contexts.

The reference's rotary modules (``operators/core/rope/real.py``, paths relative to
``/root/reference/After-Revision-DROFELL``) keep sin / cos tables; here a pair's
frequency is all that is kept.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Tuple

KINDS = ("linear", "ntk", "wavelength", "yarn")


@dataclass
class RotaryScaling:
    """How frequencies change for contexts ``factor`` times the ``original_positions``:

    * ``linear``      every frequency divided by the factor;
    * ``ntk``         the base times factor^(d / (d - 2)): the fastest pair stays, the slowest is
                      divided by the factor;
    * ``wavelength``  pairs that turn more than ``high`` times within the original positions stay,
                      those below ``low`` turns are divided, those between are blended by turns;
    * ``yarn``        the same blend by the pair's index, between those of ``fast`` and of
                      ``slow`` turns, and the rotation scaled by ``magnitude``
                      (0.1 ln(factor) + 1 unless given).
    """

    kind: str
    factor: float
    original_positions: int = 4096
    low: float = 1.0
    high: float = 4.0
    fast: float = 32.0
    slow: float = 1.0
    magnitude: Optional[float] = None

    def __post_init__(self) -> None:
        if self.kind not in KINDS:
            raise ValueError(f"scaling {self.kind!r} is none of {KINDS}")
        if not (math.isfinite(self.factor) and self.factor >= 1):
            raise ValueError("the factor must be at least 1")
        if self.original_positions < 1:
            raise ValueError("original_positions must be at least 1")
        if not 0 < self.low < self.high or not 0 < self.slow < self.fast:
            raise ValueError("low must be below high, and slow below fast, both above 0")


def rotary_frequencies(rotary_dim: int, base: float,
                       scaling: Optional[RotaryScaling] = None) -> Tuple[List[float], float]:
    """Radians per position of each pair, and the rotation's magnitude."""
    half, kind = rotary_dim // 2, None if scaling is None else scaling.kind
    if kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs two pairs at least")
        base = base * scaling.factor ** (rotary_dim / (rotary_dim - 2))
    freq = [base ** (-2 * i / rotary_dim) for i in range(half)]
    if kind in (None, "ntk"):
        return freq, 1.0
    if kind == "linear":
        return [f / scaling.factor for f in freq], 1.0
    if kind == "wavelength":
        turns = [scaling.original_positions * f / (2 * math.pi) for f in freq]
        keep = [min(max((t - scaling.low) / (scaling.high - scaling.low), 0.0), 1.0) for t in turns]
        magnitude = 1.0
    else:
        # the index whose pair turns t times within the original positions
        first, last = (rotary_dim * math.log(scaling.original_positions / (2 * math.pi * t)) / (2 * math.log(base))
                       for t in (scaling.fast, scaling.slow))
        first, last = max(math.floor(first), 0), min(math.ceil(last), rotary_dim - 1)
        keep = [1 - min(max((i - first) / max(last - first, 0.001), 0.0), 1.0) for i in range(half)]
        magnitude = 0.1 * math.log(scaling.factor) + 1.0 if scaling.magnitude is None else scaling.magnitude
    return [f * k + f / scaling.factor * (1 - k) for f, k in zip(freq, keep)], magnitude
