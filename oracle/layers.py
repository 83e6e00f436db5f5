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


def rotary_axes(x: NDArray, positions: NDArray, pair_axes: NDArray, inv_freq: NDArray,
                **options) -> NDArray:
    """rotary, pair by pair: pair c alone turns, by the positions of its axis."""
    parts = []
    for a, c in zip(np.asarray(pair_axes), range(len(inv_freq)), strict=True):
        alone = np.zeros(len(inv_freq), np.float32)
        alone[c] = inv_freq[c]
        parts.append(rotary(x, np.asarray(positions)[a], alone, **options))
    # Where pair c stands in part c; a column of no pair is the same in all.
    out, half = parts[0].copy(), len(inv_freq)
    for c, part in enumerate(parts):
        for i in (2 * c, 2 * c + 1) if options.get("interleaved") else (c, c + half):
            out[..., i] = part[..., i]
    return out


def experts_route(logits: NDArray, top_k: int, *, scores="softmax", bias=None, groups=1,
                  top_groups=1, group_best=2, renormalise=True, scale=1.0, lengths=None, seq=0):
    """(experts, weights, offsets, order, places) of float logits, token by token."""
    logits = np.asarray(logits, np.float64)
    tokens, n = logits.shape
    bias = np.zeros(n) if bias is None else np.asarray(bias, np.float64)
    chosen, weights = np.full((tokens, top_k), -1), np.zeros((tokens, top_k))
    for t in range(tokens):
        if lengths is not None and t % seq >= lengths[t // seq]:
            continue
        row = logits[t]
        open_ = [e for e in range(n) if row[e] != -np.inf and bias[e] != -np.inf]
        if not open_:
            continue
        with np.errstate(over="ignore", invalid="ignore"):
            if scores == "softmax":
                s = np.exp(row - np.nanmax(row))
                s = s / s.sum()
            else:
                s = 1.0 / (1.0 + np.exp(-row))
        c = s + bias
        if groups > 1:
            per, sums = n // groups, []
            for g in range(groups):
                inside = sorted((c[e] for e in open_ if e // per == g and not np.isnan(c[e])),
                                reverse=True)
                sums.append(sum(inside[:group_best]) if inside else -np.inf)
            kept = sorted(range(groups), key=lambda g: (-sums[g], g))[:top_groups]
            open_ = [e for e in open_ if e // per in kept]
        order = sorted(open_, key=lambda e: (np.isnan(c[e]), 0 if np.isnan(c[e]) else -c[e], e))
        for j, e in enumerate(order[:top_k]):
            chosen[t, j], weights[t, j] = e, s[e]
        if renormalise and order:
            weights[t] /= weights[t].sum()
        weights[t] *= scale
    order, offsets, places = [], [0], np.full(tokens * top_k, -1)
    for e in range(n):
        for pair in np.flatnonzero(chosen.reshape(-1) == e):
            places[pair] = len(order)
            order.append(pair)
        offsets.append(len(order))
    order += [-1] * (tokens * top_k - len(order))
    return (chosen, weights, np.array(offsets), np.array(order, dtype=np.int64),
            places.reshape(tokens, top_k))


def experts_linear(x: NDArray, w: NDArray, offsets, *, order=None, top_k=1, gated=False,
                   activation="none", bias=None) -> tuple[NDArray, NDArray]:
    """(out, what its errors are measured against) [rows, n] of float values, row by row; rows of no
    expert are zeros.  The measure is |x| |w| + |bias| of a row, gated the product's two terms."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    rows = len(x) if order is None else len(x) * top_k
    n = w.shape[1] // (2 if gated else 1)
    out, mass = np.zeros((rows, n)), np.zeros((rows, n))
    for e in range(w.shape[0]):
        for r in range(offsets[e], offsets[e + 1]):
            xr = x[r if order is None else order[r] // top_k]
            y, m = w[e] @ xr, np.abs(w[e]) @ np.abs(xr)
            if bias is not None:
                y, m = y + bias[e], m + np.abs(bias[e])
            if gated:
                a = activate(y[:n], activation)
                out[r] = a * y[n:]
                mass[r] = np.abs(a) * m[n:] + m[:n] * np.abs(y[n:])
            else:
                out[r], mass[r] = activate(y, activation), m
    return out, mass


def norm(v: NDArray, *, kind, weight=None, bias=None, eps=1e-6, offset=0.0) -> NDArray:
    if kind == "layer":
        v = v - v.mean(axis=-1, keepdims=True)
    v = v / np.sqrt(np.mean(v * v, axis=-1, keepdims=True) + eps)
    v = v * (1.0 if weight is None else weight + offset)
    return v if bias is None else v + bias


def block_norm(x, y=None, *, after=None, before=None, x_scale=1.0, y_scale=1.0, gate=None,
               gate_row=None, places=None, weights=None) -> tuple[NDArray, NDArray]:
    """(out, h) of float values; gate_row: the row of gate of each row."""
    z = None if y is None else np.asarray(y, np.float64)
    if places is not None:
        joined = np.zeros((len(places), z.shape[1]))
        for t, row in enumerate(places):
            for j, place in enumerate(row):
                if place >= 0:
                    joined[t] += float(weights[t, j]) * z[place]
        z = joined
    if z is not None and after is not None:
        z = norm(z, **after)
    if z is not None and gate is not None:
        z = z * np.asarray(gate, np.float64)[gate_row]
    out = (0.0 if z is None else y_scale * z) + (
        0.0 if x is None else x_scale * np.asarray(x, np.float64))
    return out, out if before is None else norm(out, **before)
