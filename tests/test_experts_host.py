"""Host-side parts of the operators for layers of experts (no GPU): what is refused before any call
of the library, on device addresses (a stand-in records what reaches it) and on arrays (a runtime
that keeps its buffers in host memory)."""

import numpy as np
import pytest
from test_layers_counts import Runtime
from test_layers_threads import HostRuntime

from tessery_b200 import InvalidInputError, native
from tessery_b200.layers import (
    block_norm,
    experts_linear,
    experts_route,
    rotary_axes,
    rotary_pair_axes,
)

ROUTE = dict(tokens=4, num_experts=8, top_k=2, ld=8, groups=2, top_groups=1, seq=0)
PRODUCT = dict(tokens=4, top_k=2, num_experts=8, n=16, k=32, offsets=4096)
NORM = dict(rows=4, cols=16, out=4096, h=8192)
ROTARY = dict(tokens=4, heads=2, kv_heads=1, dim=32, inv_freq=4096, pair_axes=4096, positions=4096,
              axes=2)


def route(rt, **kw):
    rt.experts_route_device(4096, 8192, 8192, **{**ROUTE, **kw})


def product(rt, **kw):
    rt.experts_linear_device(4096, 4096, 8192, **{**PRODUCT, **kw})


def norm(rt, **kw):
    rt.block_norm_device(4096, 4096, **{**NORM, **kw})


def axes(rt, **kw):
    rt.rotary_axes_device(4096, 8192, 4096, 8192, **{**ROTARY, **kw})


def refused(call, **kw):
    rt = Runtime()
    call(rt)
    assert len(rt._lib.calls) == 1
    with pytest.raises(InvalidInputError):
        call(rt, **kw)
    assert len(rt._lib.calls) == 1


COUNTS = [(route, n) for n in ("tokens", "num_experts", "top_k", "groups", "top_groups", "group_best",
                               "seq")] + [
    (product, n) for n in ("tokens", "top_k", "num_experts", "n", "k")] + [
    (norm, n) for n in ("rows", "cols", "gate_rows", "seq", "top_k", "y_rows")] + [
    (axes, n) for n in ("tokens", "heads", "kv_heads", "dim", "rot_dim", "axes")]


@pytest.mark.parametrize("call,name", COUNTS)
@pytest.mark.parametrize("value", [-1, -2**31, 2**31, 2**32 + 4, 2**70])
def test_counts(call, name, value):
    refused(call, **{name: value})


@pytest.mark.parametrize("call,name", [(route, "ld"), (axes, "axis_stride")] + [
    (product, n) for n in ("ldx", "ldw", "expert_stride", "ldo")] + [
    (norm, n) for n in ("ldx", "ldy", "ldo", "ldh", "ldg")])
@pytest.mark.parametrize("value", [-8, 2**64])
def test_strides(call, name, value):
    refused(call, **{name: value})


@pytest.mark.parametrize("call,kw", [
    (route, dict(scores="other")), (route, dict(scale=1e39)), (product, dict(activation="other")),
    (product, dict(tokens=2**16, top_k=2**15)), (norm, dict(x_scale=1e39)),
    (norm, dict(after={})), (norm, dict(after=dict(kind="other"))),
    (norm, dict(before=dict(kind="rms", scale=2.0))), (norm, dict(before=dict(kind="rms", eps=1e39)))])
def test_options(call, kw):
    refused(call, **kw)


def test_packed_structures_have_the_sizes_of_the_header():
    assert native.TX_ROUTE.size == 104 and native.TX_BLOCK_NORM.size == 232


def test_missing_context_is_refused():
    lib = native.load()
    assert lib.tx_experts_route(None, b"", 1, 1, 1, None) == native.TX_EINVAL
    assert lib.tx_experts_linear(None, None, 8, 1, None, 8, 8, None, None, 0, 1, None, None, 1, 1, 1, 1, 1,
                                 0, 0, None) == native.TX_EINVAL
    assert lib.tx_block_norm(None, b"", 1, 1, None) == native.TX_EINVAL
    assert lib.tx_rotary_axes(None, b"", b"", 0, 0, 1, 8, 8, 0, 0, None, 1, 1, None, None, 1.0, 0.0,
                              None) == native.TX_EINVAL


def test_pair_axes():
    np.testing.assert_array_equal(rotary_pair_axes((3, 1, 2)), [0, 0, 0, 1, 2, 2])
    np.testing.assert_array_equal(rotary_pair_axes((3, 1, 2), cycle=True), [0, 1, 2, 0, 2, 0])
    np.testing.assert_array_equal(rotary_pair_axes((0, 2)), [1, 1])
    for bad in ((), (0, 0), (3, -1)):
        with pytest.raises(InvalidInputError):
            rotary_pair_axes(bad)


class Host(HostRuntime):
    """Takes the calls and does nothing: the arrays' checks come before them."""

    def experts_route_device(self, *a, **kw):
        pass

    experts_linear_device = block_norm_device = rotary_axes_device = experts_route_device


X = np.ones((6, 16), np.uint16)
W = np.ones((3, 8, 16), np.uint16)
BAD = [2**32, 0.5, np.nan, -2**40]


@pytest.mark.parametrize("kw", [
    dict(offsets=[0, 2, 4]), dict(offsets=[0, 2, 1, 4]), dict(offsets=[1, 2, 3, 4]),
    dict(offsets=[0, 2, 4, 7]), *[dict(offsets=[0, 2, b, 6]) for b in BAD],
    dict(order=[0, 1, 2]), dict(order=[0, 1, 2, 3, 4, 6]), dict(order=[0, 1, 2, 3, 4, -1]),
    dict(top_k=0), dict(top_k=4), dict(bias=np.ones((3, 7))), dict(activation="other"),
    dict(out_dtype="fp8"), dict(w=W.astype(np.float32)), dict(w=W[0]), dict(w=W[:, :, :8]),
    dict(w=W[:, :7], gated=True), dict(x=X.astype(np.float32)), dict(x=X[0])])
def test_experts_linear_arrays(kw):
    ok = dict(x=X, w=W, offsets=[0, 2, 4, 6], runtime=Host())
    assert experts_linear(**ok).shape == (6, 8)
    with pytest.raises(InvalidInputError):
        experts_linear(**{**ok, **kw})


@pytest.mark.parametrize("kw", [
    dict(bias=np.ones(7)), dict(lengths=[2, 2]), dict(lengths=[2, 2], seq=2),
    dict(lengths=[2, 2, 3], seq=2), dict(lengths=[2, -1, 2], seq=2),
    *[dict(lengths=[2, b, 2], seq=2) for b in BAD], dict(logits=np.ones(8, np.float32)),
    dict(logits=np.ones((6, 8), np.int64))])
def test_experts_route_arrays(kw):
    ok = dict(logits=np.ones((6, 8), np.float32), top_k=2, runtime=Host())
    experts_route(**ok)
    experts_route(**ok, lengths=[2, 0, 1], seq=2)
    with pytest.raises(InvalidInputError):
        experts_route(**{**ok, **kw})


F = np.ones((6, 16), np.float32)


@pytest.mark.parametrize("kw", [
    dict(x=None, y=None), dict(y=F[:5]), dict(y=F[:, :8]), dict(x=F[0]), dict(weights=np.ones((6, 2))),
    dict(places=np.zeros((6, 2), int)), dict(places=np.zeros(6, int), weights=np.ones(6)),
    dict(places=np.full((6, 2), 6), weights=np.ones((6, 2))),
    dict(places=np.zeros((5, 2), int), weights=np.ones((5, 2))), dict(gate=F[:, :8]),
    dict(gate=F[:2], cu_seqlens=[0, 3]), dict(gate=F[:2], cu_seqlens=[0, 3, 5]),
    dict(gate=F[:2], cu_seqlens=[0, 7, 6]), dict(cu_seqlens=[0, 6]),
    *[dict(gate=F[:2], cu_seqlens=[0, b, 6]) for b in BAD],
    dict(after=dict(kind="rms", weight=F[0, :8])),
    dict(after=dict(kind="layer", weight=F[0], bias=F[0].astype(np.uint16))), dict(out_dtype="fp8")])
def test_block_norm_arrays(kw):
    ok = dict(x=F, y=F, runtime=Host())
    block_norm(**ok, after=dict(kind="rms", weight=F[0]), gate=F[:2], cu_seqlens=[0, 3, 6])
    with pytest.raises(InvalidInputError):
        block_norm(**{**ok, **kw})


@pytest.mark.parametrize("kw", [
    dict(positions=np.zeros(6, int)), dict(positions=np.zeros((2, 5), int)),
    dict(positions=np.full((2, 6), 1 << 24)), dict(positions=np.full((2, 6), -(1 << 24))),
    *[dict(positions=np.full((2, 6), b)) for b in BAD], dict(pair_axes=[0, 1, 2, 0]),
    dict(pair_axes=[0, -1, 0, 0]), dict(pair_axes=[0, 1]), dict(inv_freq=np.ones((2, 2)))])
def test_rotary_axes_arrays(kw):
    ok = dict(q=np.ones((6, 2, 8), np.float32), positions=np.zeros((2, 6), int),
              pair_axes=[0, 1, 0, 1], inv_freq=np.ones(4), runtime=Host())
    rotary_axes(**ok)
    with pytest.raises(InvalidInputError):
        rotary_axes(**{**ok, **kw})
