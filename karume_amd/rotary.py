"""Frequencies of rotary positions, stretched for long contexts where asked.

A head's first R elements are R/2 pairs; pair j turns by position * f_j with f_j = base^(-2j/R).  A
model trained on short contexts serves longer ones with its frequencies lowered: all alike, by a
larger base, or the slow ones alone.  The result feeds GpuContext.rope_tables.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import numpy as np


def rope_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None,
                     factor: float = 1.0, trained: int = 0, slow: float = 1.0, fast: float = 32.0
                     ) -> Tuple[np.ndarray, float]:
    """(f64 frequencies [rotary_dim / 2], amplitude of the tables).

    ``scaling``, for a context ``factor`` times as long as the ``trained`` one:
      None          f_j
      "linear"      f_j / factor
      "base"        base * factor^(R / (R - 2)): the slowest pair stretched by factor, the fastest kept
      "wavelength"  pairs that turn fewer than ``slow`` times over the trained context are divided by
                    factor, those that turn more than ``fast`` times are kept, between them the
                    frequency is blended by its number of turns
      "ramp"        blended by the pair's index instead, between the indices whose pairs turn
                    ``fast`` and ``slow`` times (whole indices outwards); the tables' amplitude is
                    0.1 ln(factor) + 1
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} is not a positive even number")
    if not base > 1.0 or not math.isfinite(base):
        raise ValueError(f"base {base}")
    if not factor >= 1.0 or not math.isfinite(factor):
        raise ValueError(f"factor {factor} is below 1")
    pairs = rotary_dim // 2
    index = np.arange(pairs, dtype=np.float64)
    plain = float(base) ** -(index / pairs)
    if scaling is None:
        return plain, 1.0
    if scaling == "linear":
        return plain / factor, 1.0
    if scaling == "base":
        if pairs == 1:
            raise ValueError("one pair has no slower one to stretch")
        return (float(base) * factor ** (pairs / (pairs - 1))) ** -(index / pairs), 1.0
    if scaling not in ("wavelength", "ramp"):
        raise ValueError(f"scaling {scaling!r}")
    if trained < 1 or not 0.0 < slow < fast:
        raise ValueError(f"{scaling!r} needs the trained context and 0 < slow < fast")
    if scaling == "wavelength":
        turns = trained * plain / (2 * math.pi)
        keep = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
        return plain * keep + plain / factor * (1.0 - keep), 1.0

    def index_of(turned: float) -> float:
        return pairs * math.log(trained / (2 * math.pi * turned)) / math.log(base)

    first = max(math.floor(index_of(fast)), 0)
    last = min(math.ceil(index_of(slow)), rotary_dim - 1)
    stretched = np.clip((index - first) / max(last - first, 1e-3), 0.0, 1.0)
    return plain / factor * stretched + plain * (1.0 - stretched), 0.1 * math.log(factor) + 1.0
