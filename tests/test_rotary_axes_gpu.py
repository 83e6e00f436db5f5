"""The rotation by positions on several axes (layers.rotary_axes / rotary_axes_device) on a B200
against its formula in 64 bits, with the tolerances of the rotation on one axis: 1.2e-5 of a value up to
5 (two hardware sines and cosines of 2^-20.4 and a few roundings), bf16 2^-8 of the value more."""

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200 import InvalidInputError, TX_F32
from tessery_b200.layers import rotary, rotary_axes, rotary_frequencies, rotary_pair_axes
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu


def make(rng, shape, dtype):
    x = rng.standard_normal(shape).astype(np.float32).clip(-5, 5)
    return (to_bf16_bits(x), from_bf16_bits(to_bf16_bits(x))) if dtype == "bf16" else (x, x)


def check(got, want):
    b16 = got.dtype == np.uint16
    g = from_bf16_bits(got) if b16 else got
    big = max(1.0, float(np.abs(want).max()) / 5)
    np.testing.assert_array_less(np.abs(g - want), 1.2e-5 * big + (2.0**-8 * np.abs(want) if b16 else 0))


@pytest.mark.parametrize("heads,kv_heads,dim,sections", [
    (16, 8, 128, (16, 24, 24)), (12, 12, 64, (16, 16)), (2, 2, 32, (8, 8)), (9, 3, 80, (8, 16, 16)),
    (4, 1, 256, (32, 32, 32, 32)), (6, 2, 96, (5, 7)), (3, 1, 33, (4, 0, 3)), (1, 1, 2, (1,)),
    (2, 1, 255, (100, 27))])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("cycle", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sections(runtime, heads, kv_heads, dim, sections, interleaved, cycle, dtype):
    rng = np.random.default_rng(dim)
    tokens, pairs = 23, sum(sections)
    q, qf = make(rng, (tokens, heads, dim), dtype)
    k, kf = make(rng, (tokens, kv_heads, dim), dtype)
    w = to_bf16_bits(1 + 0.1 * rng.standard_normal(dim).astype(np.float32)) if cycle else None
    wf = None if w is None else from_bf16_bits(w)
    freq = rotary_frequencies(2 * pairs, 10000.0)[0]
    pos = rng.integers(-500, 30000, (len(sections), tokens))
    axes = rotary_pair_axes(sections, cycle=cycle)
    for out in ("float32", "bf16"):
        got = rotary_axes(q, k, positions=pos, pair_axes=axes, inv_freq=freq, interleaved=interleaved,
                          q_norm_weight=w, k_norm_weight=w, out_dtype=out, runtime=runtime)
        assert runtime.last_kernel() == "rotary_axes"
        for g, x in zip(got, (qf, kf), strict=True):
            check(g, oracle.rotary_axes(x, pos, axes, freq, interleaved=interleaved, weight=wf))


@pytest.mark.parametrize("tokens", [1, 8, 1184, 3001])
def test_equal_axes_are_the_plain_rotation(runtime, tokens):
    rng = np.random.default_rng(tokens)
    q, _ = make(rng, (tokens, 4, 64), "bf16")
    k, _ = make(rng, (tokens, 2, 64), "bf16")
    freq = rotary_frequencies(64)[0]
    pos = rng.integers(0, 1 << 20, tokens)
    axes = rotary_pair_axes((12, 10, 10), cycle=True)
    want = rotary(q, k, inv_freq=freq, positions=pos, runtime=runtime)
    got = rotary_axes(q, k, inv_freq=freq, positions=np.stack([pos] * 3), pair_axes=axes,
                      runtime=runtime)
    for g, w in zip(got, want, strict=True):
        np.testing.assert_array_equal(g, w)
    alone, none = rotary_axes(q, inv_freq=freq, positions=np.stack([pos] * 3), pair_axes=axes,
                              runtime=runtime)
    np.testing.assert_array_equal(alone, want[0])
    assert none is None


def test_inverse_and_amplitude(runtime):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((30, 2, 32)).astype(np.float32)
    freq = rotary_frequencies(32, 100.0)[0]
    kw = dict(positions=rng.integers(-1000, 1000, (2, 30)), pair_axes=rotary_pair_axes((8, 8)),
              inv_freq=freq, runtime=runtime)
    turned = rotary_axes(x, amplitude=2.0, **kw)[0]
    back = rotary_axes(turned, amplitude=0.5, inverse=True, **kw)[0]
    np.testing.assert_allclose(back, x, atol=4e-5)


def test_axis_that_is_not_there(runtime):
    b = runtime.buffer(4096)
    b.write(np.zeros(1024, np.float32))
    axes = runtime.buffer(256)
    kw = dict(tokens=3, heads=1, dim=8, inv_freq=b.device_ptr, pair_axes=axes.device_ptr,
              positions=b.device_ptr + 1024, axes=2, in_dtype=TX_F32, out_dtype=TX_F32)
    runtime.rotary_axes_device(b.device_ptr, None, b.device_ptr, None, **kw)
    runtime.sync()
    for bad in (2, -1, 2**31 - 1):
        axes.write(np.array([0, 1, bad, 0], np.int32))
        runtime.rotary_axes_device(b.device_ptr, None, b.device_ptr, None, **kw)
        with pytest.raises(InvalidInputError):
            runtime.sync()
    axes.close()
    b.close()


def test_refusals(runtime):
    b = runtime.buffer(8192)
    p = b.device_ptr
    ok = dict(tokens=4, heads=2, dim=32, inv_freq=p + 4096, pair_axes=p + 5120, positions=p + 6144,
              axes=2, in_dtype=TX_F32, out_dtype=TX_F32)
    call = runtime.rotary_axes_device
    call(p, None, p, None, **ok)
    call(p, None, p, None, **{**ok, "axis_stride": 16})
    for kw in (dict(axes=0), dict(axis_stride=3), dict(pair_axes=p + 2), dict(positions=p + 1),
               dict(pair_axes=None), dict(positions=None), dict(rot_dim=3), dict(rot_dim=34),
               dict(dim=257), dict(amplitude=np.inf), dict(eps=-1.0), dict(in_dtype=2),
               dict(q_out_strides=(32, 32)), dict(inv_freq=None)):
        before = runtime.launch_count()
        with pytest.raises(InvalidInputError):
            call(p, None, p, None, **{**ok, **kw})
        assert runtime.launch_count() == before
    runtime.sync()
    b.close()
