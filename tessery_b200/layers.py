"""NumPy-in / NumPy-out operators for encoder layers with other options than the two built
in: the position rotation (layouts, part of the head, long-context frequencies, per-head
norms; positions on one axis or several), attention under a score rule (cap, distance bias,
window, prefix, documents), a linear layer with bias, activation and residual, the routing of
tokens to experts with the experts' products, and the norms after and before a block.

float32 arrays, or uint16 arrays holding bf16 bit patterns, as in attention.py.  The same
operators on device pointers are CudaRuntime.rotary_device, rotary_axes_device,
attention_scored_device, linear_fused_device, experts_route_device, experts_linear_device and
block_norm_device.
"""

from __future__ import annotations

import functools
import math
from collections.abc import Mapping, Sequence
from typing import Any, NamedTuple

import numpy as np
from numpy.typing import NDArray

from . import native
from .attention import _dtype_code, _upload, default_runtime
from .errors import InvalidInputError
from .runtime import CudaRuntime, _raise_for

_NP = {native.TX_F32: np.float32, native.TX_BF16: np.uint16}


def _out_code(name: str | None, default: int) -> int:
    code = default if name is None else {"float32": native.TX_F32,
                                         "bf16": native.TX_BF16}.get(name)
    if code is None:
        raise InvalidInputError()
    return code


def _read(rt: CudaRuntime, buffer, shape, code: int) -> NDArray:
    out = np.empty(shape, dtype=_NP[code])
    if out.size:
        _raise_for(rt._lib.tx_read(buffer.pointer, out.ctypes.data, out.nbytes))
    return out


def _int32(a) -> NDArray[np.int32]:
    """`a` as int32, refused where that changes a value: a document id or a position that wrapped
    would be another one."""
    a = np.asarray(a)
    with np.errstate(invalid="ignore"):
        held = np.ascontiguousarray(a, dtype=np.int32)
    if np.any(held != a):
        raise InvalidInputError()
    return held


def _values(a) -> NDArray[np.float32]:
    """`a` as float32; uint16 arrays, which hold bf16 patterns elsewhere here, are refused."""
    a = np.asarray(a)
    if a.dtype == np.uint16:
        raise InvalidInputError()
    return np.ascontiguousarray(a, dtype=np.float32)


def _one_at_a_time(operator):
    """Holds the runtime for a whole call.  The named workspaces that inputs and results go through
    are the runtime's: between an upload and the read-back another thread's call would overwrite
    them, or close one for a larger."""

    @functools.wraps(operator)
    def call(*args, runtime: CudaRuntime | None = None, **options):
        rt = runtime or default_runtime()
        with rt._lock:
            return operator(*args, runtime=rt, **options)

    return call


def rotary_frequencies(
    rot_dim: int,
    theta: float = 1e6,
    *,
    scaling: str = "none",
    factor: float = 1.0,
    original: int = 4096,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
) -> tuple[NDArray[np.float32], float]:
    """(inverse frequencies [rot_dim / 2], amplitude) for rotary / rotary_device.

    Column pair c turns by theta^(-2c / rot_dim) per position, rounded once from double.
    `scaling` stretches that for contexts `factor` times the `original` positions trained on:

    - "linear": every frequency divided by factor (position interpolation);
    - "ntk": theta multiplied by factor^(rot_dim / (rot_dim - 2)), which leaves the fastest
      pair as it is and divides the slowest by factor;
    - "yarn" (Peng et al., "YaRN: Efficient Context Window Extension of Large Language Models", 2023):
      pairs that turn more than beta_fast times over the original positions are left,
      those that turn less than beta_slow times divided by factor, with a linear ramp over the
      pair index between the two; the amplitude is 0.1 ln(factor) + 1.
    """
    if rot_dim < 2 or rot_dim % 2 or not theta > 0 or not factor >= 1 or original < 1:
        raise InvalidInputError()
    c = np.arange(rot_dim // 2, dtype=np.float64)
    amplitude = 1.0
    if scaling == "ntk":
        if rot_dim > 2:
            theta = theta * factor ** (rot_dim / (rot_dim - 2))
        freq = theta ** (-2.0 * c / rot_dim)
    elif scaling in ("none", "linear"):
        freq = theta ** (-2.0 * c / rot_dim) / (factor if scaling == "linear" else 1.0)
    elif scaling == "yarn":
        if not beta_fast > beta_slow > 0 or theta == 1.0:
            raise InvalidInputError()
        freq = theta ** (-2.0 * c / rot_dim)

        def pair_with(turns: float) -> float:  # the (real) pair index that turns so often
            return rot_dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(theta))

        low = max(math.floor(pair_with(beta_fast)), 0)
        high = min(math.ceil(pair_with(beta_slow)), rot_dim - 1)
        ramp = np.clip((c - low) / max(high - low, 1e-3), 0.0, 1.0)
        freq = freq * (1.0 - ramp) + freq / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    else:
        raise InvalidInputError()
    return freq.astype(np.float32), amplitude


@_one_at_a_time
def rotary(
    q: NDArray,
    k: NDArray | None = None,
    *,
    inv_freq: NDArray[np.float32],
    amplitude: float = 1.0,
    interleaved: bool = False,
    inverse: bool = False,
    positions: NDArray | None = None,
    cu_seqlens: NDArray | None = None,
    seq: int = 0,
    q_norm_weight: NDArray | None = None,
    k_norm_weight: NDArray | None = None,
    eps: float = 1e-6,
    out_dtype: str | None = None,
    runtime: CudaRuntime | None = None,
) -> tuple[NDArray, NDArray | None]:
    """Rotates q [tokens, heads, dim] and k [tokens, kv_heads, dim] by their positions
    (tx_rotary): the first 2 * len(inv_freq) columns of every head, half or interleaved
    layout.  Positions: `positions` [tokens], or the index inside each packed sequence
    (cu_seqlens), or token % seq.  Norm weights are bf16 bits [dim]."""
    rt = runtime or default_runtime()
    q = np.ascontiguousarray(q)
    k = None if k is None else np.ascontiguousarray(k)
    freq = np.ascontiguousarray(inv_freq, dtype=np.float32)
    if q.ndim != 3 or freq.ndim != 1 or not freq.size:
        raise InvalidInputError()
    tokens, heads, dim = q.shape
    code = _dtype_code(q)
    if k is not None and (k.ndim != 3 or k.shape[0] != tokens or k.shape[2] != dim
                          or _dtype_code(k) != code):
        raise InvalidInputError()
    out_code = _out_code(out_dtype, code)
    if not tokens:
        return (np.empty(q.shape, _NP[out_code]),
                None if k is None else np.empty(k.shape, _NP[out_code]))
    if sum(x is not None for x in (positions, cu_seqlens)) + bool(seq) != 1:
        raise InvalidInputError()
    pos_ptr = cu_ptr = None
    nseq = 0
    if positions is not None:
        pos = _int32(positions)
        if pos.shape != (tokens,) or pos.min() < 0 or pos.max() >= 1 << 24:
            raise InvalidInputError()
        pos_ptr = _upload(rt, "rotary_pos", pos)
    elif cu_seqlens is not None:
        cu = _int32(cu_seqlens)
        if cu.ndim != 1 or cu.size < 2 or cu[0] != 0 or cu[-1] != tokens or np.any(np.diff(cu) < 0):
            raise InvalidInputError()
        cu_ptr, nseq = _upload(rt, "rotary_cu", cu), cu.size - 1
    weights = []
    for name, w in (("rotary_qw", q_norm_weight), ("rotary_kw", k_norm_weight)):
        if w is not None:
            w = np.asarray(w)
            if w.shape != (dim,) or w.dtype.kind == "f":  # bit patterns, not values
                raise InvalidInputError()
            w = w.astype(np.uint16)
        weights.append(None if w is None else _upload(rt, name, w))
    size = 4 if out_code == native.TX_F32 else 2
    q_out = rt.workspace("rotary_q_out", q.size * size)
    k_out = None if k is None else rt.workspace("rotary_k_out", k.size * size)
    rt.rotary_device(
        _upload(rt, "rotary_q", q), None if k is None else _upload(rt, "rotary_k", k),
        q_out.device_ptr, None if k_out is None else k_out.device_ptr, tokens=tokens, heads=heads,
        kv_heads=0 if k is None else k.shape[1], dim=dim,
        inv_freq=_upload(rt, "rotary_freq", freq), rot_dim=2 * freq.size, interleaved=interleaved,
        inverse=inverse, amplitude=amplitude, positions=pos_ptr, cu_seqlens=cu_ptr, nseq=nseq,
        seq=seq, q_norm_weight=weights[0], k_norm_weight=weights[1], eps=eps, in_dtype=code,
        out_dtype=out_code,
    )
    rt.sync()
    return (_read(rt, q_out, q.shape, out_code),
            None if k is None else _read(rt, k_out, k.shape, out_code))


@_one_at_a_time
def attention_scored(
    q: NDArray,
    k: NDArray,
    v: NDArray,
    *,
    cu_q: NDArray | None = None,
    cu_k: NDArray | None = None,
    q_lengths: NDArray | None = None,
    k_lengths: NDArray | None = None,
    scale: float | None = None,
    causal: bool = True,
    window: tuple[int, int] = (-1, -1),
    softcap: float = 0.0,
    slopes: NDArray | None = None,
    distance_bias: NDArray | None = None,
    prefix: NDArray | None = None,
    q_docs: NDArray | None = None,
    k_docs: NDArray | None = None,
    out_dtype: str | None = None,
    runtime: CudaRuntime | None = None,
) -> NDArray:
    """Attention under a score rule (tx_attention_scored).

    Packed: q [Tq, H, d] with cu_q, k/v [Tk, Hkv, d] with cu_k (cu_k None: cu_q's).
    Padded: q [B, Lq, H, d], k/v [B, Lk, Hkv, d] with lengths (None: all rows valid).
    A sequence's queries are its last positions.  slopes [H]; distance_bias [H, 2R + 1];
    prefix [B]; q_docs / k_docs int32 per row in q's / k's row layout (q_docs alone serves
    both where the rows are the same).  Returns q's layout in q's dtype or `out_dtype`."""
    rt = runtime or default_runtime()
    q, k, v = (np.ascontiguousarray(a) for a in (q, k, v))
    code = _dtype_code(q)
    if _dtype_code(k) != code or _dtype_code(v) != code or k.shape != v.shape:
        raise InvalidInputError()
    out_code = _out_code(out_dtype, code)
    packed = cu_q is not None
    if q.ndim != (3 if packed else 4) or k.ndim != q.ndim or k.shape[-1] != q.shape[-1]:
        raise InvalidInputError()
    heads, dim = q.shape[-2:]
    if slopes is not None and np.shape(slopes) != (heads,):
        raise InvalidInputError()
    if distance_bias is not None and (np.ndim(distance_bias) != 2 or distance_bias.shape[0] != heads
                                      or distance_bias.shape[1] % 2 == 0):
        raise InvalidInputError()
    if q_docs is not None and k_docs is None:
        k_docs = q_docs
    kw: dict = {}

    def layout(side: str, x: NDArray, cu, lengths) -> int:
        """Uploads one side's layout; returns its number of sequences."""
        if packed:
            cu = _int32(cu)
            if (lengths is not None or cu.ndim != 1 or cu.size < 2 or cu[0] != 0
                    or cu[-1] != x.shape[0] or np.any(np.diff(cu) < 0)):
                raise InvalidInputError()
            kw["cu_" + side] = _upload(rt, "scored_cu_" + side, cu)
            kw["rows_" + side], kw["max_" + side] = x.shape[0], int(np.diff(cu).max())
            return cu.size - 1
        if cu is not None:
            raise InvalidInputError()
        if lengths is not None:
            n = _int32(lengths)
            if n.shape != x.shape[:1] or np.any(n < 0) or np.any(n > x.shape[1]):
                raise InvalidInputError()
            kw[side + "_lengths"] = _upload(rt, f"scored_{side}_lengths", n) if n.size else None
        kw["rows_" + side], kw["max_" + side] = x.shape[0] * x.shape[1], x.shape[1]
        return x.shape[0]

    nseq = layout("q", q, cu_q, q_lengths)
    if layout("k", k, cu_q if packed and cu_k is None else cu_k, k_lengths) != nseq:
        raise InvalidInputError()
    if prefix is not None and np.shape(prefix) != (nseq,):
        raise InvalidInputError()
    for name, docs, x in (("q_docs", q_docs, q), ("k_docs", k_docs, k)):
        if docs is not None:
            docs = _int32(docs)
            if docs.shape != x.shape[:-2]:
                raise InvalidInputError()
            kw[name] = _upload(rt, "scored_" + name, docs) if docs.size else None
    if not q.size:
        return np.empty(q.shape, _NP[out_code])
    for name, a in (("slopes", slopes), ("distance_bias", distance_bias)):
        if a is not None:
            kw[name] = _upload(rt, "scored_" + name, np.ascontiguousarray(a, dtype=np.float32))
    if prefix is not None:
        kw["prefix"] = _upload(rt, "scored_prefix", _int32(prefix))
    if not k.size:  # nothing to attend: every row is empty
        return np.zeros(q.shape, _NP[out_code])
    out = rt.workspace("scored_out", q.size * (4 if out_code == native.TX_F32 else 2))
    rt.attention_scored_device(
        _upload(rt, "scored_q", q), _upload(rt, "scored_k", k), _upload(rt, "scored_v", v),
        out.device_ptr, nseq=nseq, heads=heads, kv_heads=k.shape[-2], dim=dim, in_dtype=code,
        out_dtype=out_code, scale=scale, causal=causal, window=window, softcap=softcap,
        reach=0 if distance_bias is None else distance_bias.shape[1] // 2, **kw)
    rt.sync()
    return _read(rt, out, q.shape, out_code)


@_one_at_a_time
def linear_fused(
    x: NDArray,
    w: NDArray,
    *,
    bias: NDArray | None = None,
    activation: str = "none",
    residual: NDArray | None = None,
    out_dtype: str = "bf16",
    runtime: CudaRuntime | None = None,
) -> NDArray:
    """act(x w^T + bias) + residual (tx_linear_fused): x [m, k] and w [n, k] bf16 bits, bias
    [n], residual [m, n] float32 or bf16 bits; activation none, relu, gelu, gelu_tanh, silu."""
    rt = runtime or default_runtime()
    x, w = np.asarray(x), np.asarray(w)
    if (x.ndim != 2 or w.ndim != 2 or x.shape[1] != w.shape[1] or x.dtype != np.uint16
            or w.dtype != np.uint16 or not w.size):
        raise InvalidInputError()
    (m, k), n = x.shape, w.shape[0]
    out_code = _out_code(out_dtype, native.TX_BF16)
    res_code = native.TX_F32
    if bias is not None and np.shape(bias) != (n,):
        raise InvalidInputError()
    if residual is not None:
        residual = np.ascontiguousarray(residual)
        res_code = _dtype_code(residual)
        if residual.shape != (m, n):
            raise InvalidInputError()
    if activation not in native.ACTIVATIONS:
        raise InvalidInputError()
    if not m:
        return np.empty((m, n), _NP[out_code])
    ld = -(-k // 8) * 8  # rows on 16-byte boundaries

    def rows(name: str, a: NDArray) -> int:
        padded = np.zeros((a.shape[0], ld), np.uint16)
        padded[:, :k] = a
        return _upload(rt, name, padded)

    out = rt.workspace("linear_out", m * n * (4 if out_code == native.TX_F32 else 2))
    rt.linear_fused_device(
        rows("linear_x", x), rows("linear_w", w), out.device_ptr, m=m, n=n, k=k, ldx=ld, ldw=ld,
        bias=None if bias is None else _upload(rt, "linear_bias",
                                               np.ascontiguousarray(bias, np.float32)),
        activation=activation,
        residual=None if residual is None else _upload(rt, "linear_residual", residual),
        residual_dtype=res_code, out_dtype=out_code)
    rt.sync()
    return _read(rt, out, (m, n), out_code)


def rotary_pair_axes(sections: Sequence[int], *, cycle: bool = False) -> NDArray[np.int32]:
    """The axis of each rotated pair for rotary_axes: sections[a] pairs for axis a, one section
    behind the other, or with `cycle` the axes in turn, each until it has had its pairs."""
    sections = [int(n) for n in sections]
    if not sections or min(sections) < 0 or not sum(sections):
        raise InvalidInputError()
    if not cycle:
        return np.repeat(np.arange(len(sections)), sections).astype(np.int32)
    # Pair i of an axis comes in turn i; within a turn the axes stand in their order.
    turn = np.concatenate([np.arange(n) for n in sections])
    axis = np.repeat(np.arange(len(sections)), sections)
    return axis[np.lexsort((axis, turn))].astype(np.int32)


@_one_at_a_time
def rotary_axes(
    q: NDArray,
    k: NDArray | None = None,
    *,
    positions: NDArray,
    pair_axes: NDArray,
    inv_freq: NDArray[np.float32],
    amplitude: float = 1.0,
    interleaved: bool = False,
    inverse: bool = False,
    q_norm_weight: NDArray | None = None,
    k_norm_weight: NDArray | None = None,
    eps: float = 1e-6,
    out_dtype: str | None = None,
    runtime: CudaRuntime | None = None,
) -> tuple[NDArray, NDArray | None]:
    """`rotary` for tokens that stand on several axes (tx_rotary_axes): positions [axes, tokens],
    of which pair c of the rotated columns turns by those of axis pair_axes[c]."""
    rt = runtime or default_runtime()
    q = np.ascontiguousarray(q)
    k = None if k is None else np.ascontiguousarray(k)
    freq = np.ascontiguousarray(inv_freq, dtype=np.float32)
    if q.ndim != 3 or freq.ndim != 1 or not freq.size:
        raise InvalidInputError()
    tokens, heads, dim = q.shape
    code = _dtype_code(q)
    if k is not None and (k.ndim != 3 or k.shape[0] != tokens or k.shape[2] != dim
                          or _dtype_code(k) != code):
        raise InvalidInputError()
    out_code = _out_code(out_dtype, code)
    pos, axis = _int32(positions), _int32(pair_axes)
    if pos.ndim != 2 or pos.shape[1] != tokens or not pos.shape[0] or axis.shape != freq.shape:
        raise InvalidInputError()
    if axis.min() < 0 or axis.max() >= pos.shape[0]:
        raise InvalidInputError()
    if tokens and max(-int(pos.min()), int(pos.max())) >= 1 << 24:
        raise InvalidInputError()
    if not tokens:
        return (np.empty(q.shape, _NP[out_code]),
                None if k is None else np.empty(k.shape, _NP[out_code]))
    weights = []
    for name, w in (("rotary_qw", q_norm_weight), ("rotary_kw", k_norm_weight)):
        if w is not None:
            w = np.asarray(w)
            if w.shape != (dim,) or w.dtype.kind == "f":  # bit patterns, not values
                raise InvalidInputError()
            w = w.astype(np.uint16)
        weights.append(None if w is None else _upload(rt, name, w))
    size = 4 if out_code == native.TX_F32 else 2
    q_out = rt.workspace("rotary_q_out", q.size * size)
    k_out = None if k is None else rt.workspace("rotary_k_out", k.size * size)
    rt.rotary_axes_device(
        _upload(rt, "rotary_q", q), None if k is None else _upload(rt, "rotary_k", k),
        q_out.device_ptr, None if k_out is None else k_out.device_ptr, tokens=tokens, heads=heads,
        kv_heads=0 if k is None else k.shape[1], dim=dim,
        inv_freq=_upload(rt, "rotary_freq", freq), rot_dim=2 * freq.size,
        pair_axes=_upload(rt, "rotary_pair_axes", axis), positions=_upload(rt, "rotary_pos", pos),
        axes=pos.shape[0], interleaved=interleaved, inverse=inverse, amplitude=amplitude,
        q_norm_weight=weights[0], k_norm_weight=weights[1], eps=eps, in_dtype=code,
        out_dtype=out_code)
    rt.sync()
    return (_read(rt, q_out, q.shape, out_code),
            None if k is None else _read(rt, k_out, k.shape, out_code))


class Routes(NamedTuple):
    """What experts_route returns: experts and weights [tokens, top_k], and the plan of the rows by
    expert (offsets [experts + 1], order [tokens * top_k] with -1 behind the last row, places
    [tokens, top_k])."""

    experts: NDArray[np.int32]
    weights: NDArray[np.float32]
    offsets: NDArray[np.int32]
    order: NDArray[np.int32]
    places: NDArray[np.int32]


@_one_at_a_time
def experts_route(
    logits: NDArray,
    top_k: int,
    *,
    bias: NDArray | None = None,
    scores: str = "softmax",
    groups: int = 1,
    top_groups: int = 1,
    group_best: int = 2,
    renormalise: bool = True,
    scale: float = 1.0,
    lengths: NDArray | None = None,
    seq: int = 0,
    runtime: CudaRuntime | None = None,
) -> Routes:
    """Routing of tokens to experts (tx_experts_route): logits [tokens, experts]; `lengths` are the
    valid rows of each sequence of `seq` rows."""
    rt = runtime or default_runtime()
    logits = np.ascontiguousarray(logits)
    if logits.ndim != 2 or not logits.shape[1]:
        raise InvalidInputError()
    code, (tokens, experts) = _dtype_code(logits), logits.shape
    if top_k > experts:  # before memory for as many is taken
        raise InvalidInputError()
    bias = None if bias is None else _values(bias)
    if bias is not None and bias.shape != (experts,):
        raise InvalidInputError()
    if lengths is not None:
        if seq < 1:
            raise InvalidInputError()
        lengths = _int32(lengths)
        if lengths.shape != (-(-tokens // seq),) or np.any(lengths < 0) or np.any(lengths > seq):
            raise InvalidInputError()
    pairs = tokens * top_k
    room = rt.workspace("route_out", 4 * max(1, 4 * pairs + experts + 1))
    if tokens and top_k > 0:
        room.write(np.full(4 * pairs + experts + 1, -1, np.int32))
    at = [room.device_ptr + 4 * pairs * i for i in range(5)]
    # A refusal is the device call's, an empty batch among them.
    rt.experts_route_device(
        _upload(rt, "route_logits", logits) if tokens else at[0], at[0], at[1], tokens=tokens,
        num_experts=experts, top_k=top_k, logits_dtype=code,
        bias=None if bias is None else _upload(rt, "route_bias", bias),
        scores=scores, groups=groups, top_groups=top_groups, group_best=group_best,
        renormalise=renormalise, scale=scale, seq=seq,
        lengths=None if lengths is None or not tokens else _upload(rt, "route_lengths", lengths),
        order=at[2], places=at[3], offsets=at[4])
    rt.sync()
    out = _read(rt, room, (4 * pairs + experts + 1,), native.TX_F32).view(np.int32)
    chosen, weights, order, places = (out[pairs * i:pairs * (i + 1)] for i in range(4))
    shape = (tokens, top_k)
    return Routes(chosen.reshape(shape), weights.view(np.float32).reshape(shape), out[4 * pairs:],
                  order, places.reshape(shape))


def _plan_offsets(offsets: NDArray, rows: int) -> NDArray[np.int32]:
    offsets = _int32(offsets)
    if (offsets.ndim != 1 or offsets.size < 2 or offsets[0] != 0 or np.any(np.diff(offsets) < 0)
            or offsets[-1] > rows):
        raise InvalidInputError()
    return offsets


@_one_at_a_time
def experts_linear(
    x: NDArray,
    w: NDArray,
    offsets: NDArray,
    *,
    order: NDArray | None = None,
    top_k: int = 1,
    gated: bool = False,
    activation: str = "none",
    bias: NDArray | None = None,
    out_dtype: str = "bf16",
    runtime: CudaRuntime | None = None,
) -> NDArray:
    """The experts' products (tx_experts_linear) over rows that experts_route planned.  With order
    [tokens * top_k]: x [tokens, k] bf16 bits, one row for each entry; without: x [rows, k], by
    expert.  w [experts, n, k] bf16 bits, gated [experts, 2 n, k], bias [experts, n or 2 n].
    Returns [rows, n], rows that no expert has being zeros."""
    rt = runtime or default_runtime()
    x, w = np.asarray(x), np.asarray(w)
    if (x.ndim != 2 or w.ndim != 3 or x.shape[1] != w.shape[2] or x.dtype != np.uint16
            or w.dtype != np.uint16 or not w.size or (gated and w.shape[1] % 2) or top_k < 1):
        raise InvalidInputError()
    experts, wide, k = w.shape
    n = wide // 2 if gated else wide
    rows = len(x)
    if order is not None:
        rows, order = len(x) * top_k, _int32(order)
    elif rows % top_k:
        raise InvalidInputError()
    offsets = _plan_offsets(offsets, rows)
    if offsets.size != experts + 1 or activation not in native.ACTIVATIONS:
        raise InvalidInputError()
    bias = None if bias is None else _values(bias)
    if bias is not None and bias.shape != (experts, wide):
        raise InvalidInputError()
    if order is not None:
        used = order[:offsets[-1]]
        if order.shape != (rows,) or np.any(used < 0) or np.any(used >= rows):
            raise InvalidInputError()
    out_code = _out_code(out_dtype, native.TX_BF16)
    if not offsets[-1]:
        return np.zeros((rows, n), _NP[out_code])
    ld = -(-k // 8) * 8  # rows on 16-byte boundaries

    def padded(name: str, a: NDArray) -> int:
        b = np.zeros((*a.shape[:-1], ld), np.uint16)
        b[..., :k] = a
        return _upload(rt, name, b)

    out = rt.workspace("experts_out", rows * n * (4 if out_code == native.TX_F32 else 2))
    rt.experts_linear_device(
        padded("experts_x", x), padded("experts_w", w), out.device_ptr,
        offsets=_upload(rt, "experts_offsets", offsets), tokens=rows // top_k, top_k=top_k,
        num_experts=experts, n=n, k=k, gated=gated, activation=activation, ldx=ld, ldw=ld,
        order=None if order is None else _upload(rt, "experts_order", order),
        bias=None if bias is None else _upload(rt, "experts_bias", bias),
        out_dtype=out_code)
    rt.sync()
    got = _read(rt, out, (rows, n), out_code)
    got[offsets[-1]:] = 0
    return got


@_one_at_a_time
def block_norm(
    x: NDArray | None,
    y: NDArray | None = None,
    *,
    after: Mapping[str, Any] | None = None,
    before: Mapping[str, Any] | None = None,
    x_scale: float = 1.0,
    y_scale: float = 1.0,
    gate: NDArray | None = None,
    cu_seqlens: NDArray | None = None,
    seq: int = 0,
    places: NDArray | None = None,
    weights: NDArray | None = None,
    out_dtype: str = "float32",
    h_dtype: str = "bf16",
    runtime: CudaRuntime | None = None,
) -> tuple[NDArray, NDArray]:
    """The rows between two blocks (tx_block_norm): (out, h), out = x_scale x + y_scale gate *
    after(y) and h = before(out).  Norms are mappings with `kind` ("rms" or "layer") and, where
    wanted, `weight` and `bias` [cols], `eps`, `offset`.  gate [gate rows, cols].  With places and
    weights [rows, top_k] from experts_route, y [.., cols] holds the experts' rows."""
    rt = runtime or default_runtime()
    x, y, gate = (None if a is None else np.ascontiguousarray(a) for a in (x, y, gate))
    if any(a is not None and a.ndim != 2 for a in (x, y, gate)):
        raise InvalidInputError()
    if x is None and y is None or places is not None and np.ndim(places) != 2:
        raise InvalidInputError()
    rows, cols = x.shape if x is not None else y.shape
    if x is None and places is not None:
        rows = np.shape(places)[0]
    if not cols or any(a is not None and a.shape[1] != cols for a in (x, y, gate)):
        raise InvalidInputError()
    kw: dict = {}
    if places is not None:
        places = _int32(places)
        weights = None if weights is None else _values(weights)
        if (y is None or places.ndim != 2 or places.shape[0] != rows or np.shape(weights) != places.shape
                or not places.shape[1] or np.any(places >= len(y))):
            raise InvalidInputError()
        kw.update(top_k=places.shape[1], y_rows=len(y))
    elif weights is not None or (y is not None and len(y) != rows):
        raise InvalidInputError()
    if gate is not None:
        if rows and not len(gate):
            raise InvalidInputError()
        kw.update(gate_rows=len(gate), gate_dtype=_dtype_code(gate), seq=seq)
    if cu_seqlens is not None:
        cu = _int32(cu_seqlens)
        if (gate is None or seq or cu.shape != (len(gate) + 1,) or cu[0] != 0 or cu[-1] != rows
                or np.any(np.diff(cu) < 0)):
            raise InvalidInputError()
    norms = []
    for norm in (after, before):
        if norm is not None:
            norm = dict(norm)
            for name in ("weight", "bias"):
                if norm.get(name) is not None:
                    a = norm[name] = np.ascontiguousarray(norm[name])
                    if a.shape != (cols,) or norm.setdefault("dtype", _dtype_code(a)) != _dtype_code(a):
                        raise InvalidInputError()
        norms.append(norm)
    codes = [_out_code(out_dtype, native.TX_F32), _out_code(h_dtype, native.TX_BF16)]
    if not rows:
        return tuple(np.empty((0, cols), _NP[c]) for c in codes)
    for name, a in (("x", x), ("y", y)):
        if a is not None:
            kw[name + "_dtype"] = _dtype_code(a)
    at = {name: _upload(rt, "norm_" + name, a)
          for name, a in (("x", x), ("y", y), ("gate", gate), ("places", places),
                          ("weights", weights),
                          ("cu_seqlens", None if cu_seqlens is None else cu))
          if a is not None and a.size}
    for which, norm in zip(("after", "before"), norms, strict=True):
        if norm is not None:
            for name in ("weight", "bias"):
                if norm.get(name) is not None:
                    norm[name] = _upload(rt, f"norm_{which}_{name}", norm[name])
    if y is not None and not y.size:  # no expert has a row
        at["y"] = rt.workspace("norm_y", 256).device_ptr
    outs = [rt.workspace("norm_" + name, rows * cols * (4 if c == native.TX_F32 else 2))
            for name, c in zip(("out", "h"), codes, strict=True)]
    rt.block_norm_device(at.pop("x", None), at.pop("y", None), rows=rows, cols=cols,
                         out=outs[0].device_ptr, h=outs[1].device_ptr, out_dtype=codes[0],
                         h_dtype=codes[1], after=norms[0], before=norms[1], x_scale=x_scale,
                         y_scale=y_scale, **at, **kw)
    rt.sync()
    return tuple(_read(rt, b, (rows, cols), c) for b, c in zip(outs, codes, strict=True))
