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


def open_keys(nq: int, nk: int, *, causal=False, window=(-1, -1), prefix=0, q_docs=None,
              k_docs=None) -> NDArray:
    """[nq, nk] truth values: the keys the rule leaves open to each query row."""
    pos = np.arange(nq)[:, None] + nk - nq
    j = np.arange(nk)[None, :]
    seen = np.ones((nq, nk), bool)
    if causal:
        seen &= j <= pos
    if window[0] >= 0:
        seen &= j >= pos - window[0]
    if window[1] >= 0:
        seen &= j <= pos + window[1]
    seen |= j < prefix
    if q_docs is not None:
        q_docs, k_docs = np.asarray(q_docs), np.asarray(k_docs)
        seen &= (q_docs[:, None] == k_docs[None, :]) & (q_docs[:, None] >= 0)
    return seen


def attention_scored(q: NDArray, k: NDArray, v: NDArray, *, scale=None, softcap=0.0, slopes=None,
                     table=None, **rule) -> tuple[NDArray, NDArray, float]:
    """One sequence: q [nq, heads, dim], k and v [nk, kv_heads, dim] as float values.  Returns
    the output, sum_j p_ij |v_j| (what the errors of the weights p are measured against) and the
    largest finite |score| plus |scale| sum |q||k| met.  A key that is not open is never read."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    nq, heads, dim = q.shape
    nk, group = k.shape[0], heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    seen = open_keys(nq, nk, **rule)
    pos = np.arange(nq)[:, None] + nk - nq
    dist = np.arange(nk)[None, :] - pos
    out, mass, biggest = np.zeros((nq, heads, dim)), np.zeros((nq, heads, dim)), 0.0
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        for i in range(nq):
            at = np.flatnonzero(seen[i])
            if not at.size:
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                z = scale * (kh[at] @ q[i, h])
                biggest = max(biggest, float(np.nanmax(
                    abs(scale) * (np.abs(kh[at]) @ np.abs(q[i, h])), initial=0.0)))
                if softcap:
                    z = softcap * np.tanh(z / softcap)
                if slopes is not None:
                    z = z - float(slopes[h]) * np.abs(dist[i, at])
                if table is not None:
                    reach = (table.shape[1] - 1) // 2
                    z = z + np.asarray(table[h], np.float64)[
                        np.clip(dist[i, at], -reach, reach) + reach]
                finite = np.abs(z[np.isfinite(z) & (np.abs(z) < 1e30)])
                biggest = max(biggest, float(finite.max(initial=0.0)))
                top = np.max(z)
                if top == -np.inf:
                    continue
                p = np.exp(z - top)
                p /= p.sum()
                at, p = at[p != 0], p[p != 0]
                out[i, h] = p @ vh[at]
                mass[i, h] = p @ np.abs(vh[at])
    return out, mass, biggest


def activate(y: NDArray, name: str) -> NDArray:
    if name == "none":
        return y
    if name == "relu":
        return np.maximum(y, 0.0)
    if name == "gelu":
        return y * 0.5 * (1.0 + _erf(y / math.sqrt(2.0)))
    if name == "gelu_tanh":
        return y * 0.5 * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y**3)))
    if name == "silu":
        return y / (1.0 + np.exp(-y))
    raise ValueError(name)


def linear_fused(x: NDArray, w: NDArray, *, bias=None, activation="none",
                 residual=None) -> NDArray:
    """act(x w^T + bias) + residual of float values."""
    y = np.asarray(x, np.float64) @ np.asarray(w, np.float64).T
    if bias is not None:
        y = y + bias
    y = activate(y, activation)
    return y if residual is None else y + residual
