"""Frequency factors of rotary embeddings for long contexts (``Compute.rope_at``).

Every scaling rule in use divides the angle of pair j, pos * theta^(-2j/rot), by a factor of its own
and may scale the rotated values by a magnitude: the functions below make the factors, in f64
rounded once to f32. Linear scaling is one factor for all pairs, which ``rope_at`` takes as its
``scale``; a GGUF file's ``rope_freqs.weight`` holds such factors as they are.
"""
from __future__ import annotations

import math
from typing import Tuple

import numpy as np


def _wavelengths(rotary_dim: int, theta: float) -> np.ndarray:
    """Positions per turn of each pair."""
    if rotary_dim < 2 or rotary_dim % 2 or not 0 < theta < math.inf:
        raise ValueError(f"Rotary dims {rotary_dim} / theta {theta} are invalid.")
    return 2 * math.pi * float(theta) ** (np.arange(0, rotary_dim, 2, dtype=np.float64) / rotary_dim)


def llama3_factors(rotary_dim: int, theta: float, factor: float, low: float, high: float, original: int) -> np.ndarray:
    """Llama 3's rule: pairs that turn more than ``high`` times within the ``original`` context keep
    their frequency, those below ``low`` turns are slowed by ``factor``, a ramp lies between."""
    if not (factor > 0 and high > low > 0 and original > 0):
        raise ValueError("Llama 3 scaling needs factor > 0, high > low > 0 and an original context.")
    turns = original / _wavelengths(rotary_dim, theta)
    keep = np.clip((turns - low) / (high - low), 0, 1)
    return (1 / ((1 - keep) / factor + keep)).astype(np.float32)


def yarn_factors(rotary_dim: int, theta: float, factor: float, original: int, fast: float = 32.0,
                 slow: float = 1.0) -> Tuple[np.ndarray, float]:
    """YaRN (Peng et al., 2023): a ramp over the pair index from the pair that turns ``fast`` times
    within the ``original`` context (kept) to the one that turns ``slow`` times (slowed by ``factor``).
    Returns the factors and the magnitude 0.1 ln(factor) + 1."""
    if not (factor >= 1 and fast > slow > 0 and original > 0 and theta > 1):
        raise ValueError("YaRN scaling needs factor >= 1, fast > slow > 0, an original context and theta > 1.")
    _wavelengths(rotary_dim, theta)
    pair = lambda turns: rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    first, last = max(0, math.floor(pair(fast))), min(rotary_dim - 1, math.ceil(pair(slow)))
    ramp = np.clip((np.arange(rotary_dim // 2) - first) / max(last - first, 1e-3), 0, 1)
    return (1 / (ramp / factor + (1 - ramp))).astype(np.float32), 0.1 * math.log(factor) + 1.0
