"""NumPy forms of the encoder-layer operators (tessery_b200/layers.py) in 64 bits: test
infrastructure only.  Written from the operators' formulas; loops where a loop is plainest."""

from __future__ import annotations

import math

import numpy as np
from numpy.typing import NDArray

_erf = np.vectorize(math.erf, otypes=[np.float64])


def rotary(x: NDArray, positions: NDArray, inv_freq: NDArray, *, amplitude: float = 1.0,
           interleaved: bool = False, inverse: bool = False, weight: NDArray | None = None,
           eps: float = 1e-6) -> NDArray:
    """x [tokens, heads, dim] as float values; weight as float values [dim] or None."""
    y = np.array(x, dtype=np.float64)
    if weight is not None:
        y = y / np.sqrt(np.mean(y * y, axis=-1, keepdims=True) + eps) * weight
    r = 2 * len(inv_freq)
    # The angle is by definition the float32 product of position and frequency.
    angle = (np.asarray(positions, np.float32)[:, None]
             * np.asarray(inv_freq, np.float32)).astype(np.float64)[:, None, :]
    cos, sin = amplitude * np.cos(angle), amplitude * np.sin(angle)
    if inverse:
        sin = -sin
    out = y.copy()
    for c in range(r // 2):
        i, j = (2 * c, 2 * c + 1) if interleaved else (c, c + r // 2)
        out[..., i] = y[..., i] * cos[..., c] - y[..., j] * sin[..., c]
        out[..., j] = y[..., j] * cos[..., c] + y[..., i] * sin[..., c]
    return out
