"""The linear layer with bias, activation and residual (layers.linear_fused /
linear_fused_device) on a B200 against the formula in 64 bits, and its refusals.

Tolerance, per element, with A = sum |x w| + |bias|: the products of bf16 values are exact in
fp32 and the sum of k of them in fp32 is off by at most k 2^-23 A in the worst order; tensor-core
accumulation adds 16 products at a time and cuts rather than rounds, so k / 16 + 16 additions of
2^-23 each bound it, and the plain sums over lanes are shorter still: (k / 16 + 16) 2^-23 A.  No
activation here is steeper than 1.13, nor off by more than 2^-20 of its value plus 2^-21 of |y|
(the erf form cancels for negative y).  bf16 output: 2^-8 of the value."""

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200 import InvalidInputError, TX_BF16, TX_F32
from tessery_b200.layers import linear_fused
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def bf16(rng, shape, scale=1.0):
    bits = to_bf16_bits((scale * rng.standard_normal(shape)).astype(np.float32))
    return bits, from_bf16_bits(bits)


def check(got, xf, wf, bias, act, residual):
    b16 = got.dtype == np.uint16
    g = from_bf16_bits(got) if b16 else got
    want = oracle.linear_fused(xf, wf, bias=bias, activation=act, residual=residual)
    mass = np.abs(xf.astype(np.float64)) @ np.abs(wf.astype(np.float64)).T
    if bias is not None:
        mass = mass + np.abs(bias)
    tol = 1.13 * (xf.shape[1] / 16 + 16) * 2.0**-23 * mass + 2.0**-20 * mass
    if residual is not None:
        tol = tol + 2.0**-23 * np.abs(residual)
    if b16:
        tol = tol + 2.0**-8 * np.abs(want)
    np.testing.assert_array_less(np.abs(g - want), tol + 1e-30)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 7, 8, 9, 33, 128, 129, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (7, 9), (64, 64), (65, 63), (128, 1000), (1000, 257),
                                 (384, 384), (33, 2049)])
def test_sizes(runtime, m, n, k):
    rng = np.random.default_rng(m * 1000 + n + k)
    x, xf = bf16(rng, (m, k))
    w, wf = bf16(rng, (n, k), k**-0.5)
    bias = rng.standard_normal(n).astype(np.float32)
    act = ACTS[(m + n + k) % 5]
    check(linear_fused(x, w, bias=bias, activation=act, out_dtype="float32", runtime=runtime),
          xf, wf, bias, act, None)
    assert runtime.last_kernel() == "linear_fused"
    check(linear_fused(x, w, activation=act, runtime=runtime), xf, wf, None, act, None)


@pytest.mark.parametrize("m", [1, 6, 200])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("res", ["none", "f32", "bf16"])
@pytest.mark.parametrize("out", ["float32", "bf16"])
def test_epilogues(runtime, m, act, res, out):
    rng = np.random.default_rng(m)
    n, k = 136, 200
    x, xf = bf16(rng, (m, k), 3.0)
    w, wf = bf16(rng, (n, k), k**-0.5)
    bias = rng.standard_normal(n).astype(np.float32)
    r = rf = None
    if res != "none":
        r, rf = bf16(rng, (m, n))
        r = rf if res == "f32" else r
    got = linear_fused(x, w, bias=bias, activation=act, residual=r, out_dtype=out, runtime=runtime)
    check(got, xf, wf, bias, act, rf)


def test_wide_tiles(runtime):
    """Enough rows for every tile width, with ragged last tiles, several tiles per CTA."""
    rng = np.random.default_rng(0)
    for m, n, k in ((19000, 200, 72), (9700, 300, 136), (3000, 1100, 520)):
        x, xf = bf16(rng, (m, k))
        w, wf = bf16(rng, (n, k), k**-0.5)
        r = rng.standard_normal((m, n)).astype(np.float32)
        check(linear_fused(x, w, residual=r, out_dtype="float32", runtime=runtime), xf, wf, None,
              "none", r)


@pytest.mark.parametrize("m,n,k", [(14000, 256, 72), (20000, 264, 600), (700, 1000, 1400)])
@pytest.mark.parametrize("out", ["float32", "bf16"])
def test_several_tiles_in_turn(runtime, m, n, k, out):
    """CTAs that send several tiles through the same staging buffers; sums in several parts."""
    rng = np.random.default_rng(m)
    x, xf = bf16(rng, (m, k))
    w, wf = bf16(rng, (n, k), k**-0.5)
    bias = rng.standard_normal(n).astype(np.float32)
    check(linear_fused(x, w, bias=bias, activation="gelu", out_dtype=out, runtime=runtime), xf, wf,
          bias, "gelu", None)
    r, rf = bf16(rng, (m, n))
    r = rf if out == "float32" else r
    check(linear_fused(x, w, residual=r, out_dtype=out, runtime=runtime), xf, wf, None, "none", rf)


@pytest.mark.parametrize("m,n,k", [(9, 4096, 513), (40, 65, 4097), (130, 343, 1024), (773, 117, 3754),
                                   (16, 1024, 4096), (20, 1, 9000)])
@pytest.mark.parametrize("out", ["float32", "bf16"])
def test_few_tiles_of_long_k(runtime, m, n, k, out):
    """k cut into parts that CTAs of their own sum: right, the same every time, and the counters as
    they were before."""
    rng = np.random.default_rng(m + k)
    x, xf = bf16(rng, (m, k))
    w, wf = bf16(rng, (n, k), k**-0.5)
    bias = rng.standard_normal(n).astype(np.float32)
    r, rf = bf16(rng, (m, n))
    got = [linear_fused(x, w, bias=bias, activation="silu", residual=r, out_dtype=out,
                        runtime=runtime) for _ in range(3)]
    check(got[0], xf, wf, bias, "silu", rf)
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


@pytest.mark.parametrize("m", [2, 40])
@pytest.mark.parametrize("act", ACTS)
def test_infinite_sums_stay_infinite(runtime, m, act):
    rng = np.random.default_rng(m)
    x, xf = bf16(rng, (m, 64))
    w, wf = bf16(rng, (40, 64), 0.1)
    bias = np.zeros(40, np.float32)
    bias[7] = np.inf
    got = linear_fused(x, w, bias=bias, activation=act, out_dtype="float32", runtime=runtime)
    assert np.isposinf(got[:, 7]).all()
    rest = np.arange(40) != 7
    check(got[:, rest], xf, wf[rest], None, act, None)


@pytest.mark.parametrize("k", [72, 600])
@pytest.mark.parametrize("out", ["float32", "bf16"])
def test_widest_tiles(runtime, k, out):
    """Enough tiles of 128 x 256 for several per CTA, the last of each row ragged; sums in one part
    and in two."""
    rng = np.random.default_rng(k)
    m, n = 9400, 1530
    x, xf = bf16(rng, (m, k))
    w, wf = bf16(rng, (n, k), k**-0.5)
    bias = rng.standard_normal(n).astype(np.float32)
    r, rf = bf16(rng, (m, n))
    r = rf if out == "float32" else r
    check(linear_fused(x, w, bias=bias, activation="relu", residual=r, out_dtype=out,
                       runtime=runtime), xf, wf, bias, "relu", rf)


@pytest.mark.parametrize("m", [3, 150])
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("out", [TX_F32, TX_BF16])
def test_strides_and_in_place_residual(runtime, m, odd, out):
    """Row strides of every operand, values past k and n that must not be read or written, the
    residual updated in place; an odd output stride takes the vector stores away."""
    rng = np.random.default_rng(m + odd)
    n, k, ldx, ldw, ldo = 100, 70, 80, 96, 108 + odd
    x, xf = bf16(rng, (m, ldx))
    w, wf = bf16(rng, (n, ldw), 0.1)
    x[:, k:], w[:, k:] = 0x7FC0, 0x7F80  # NaN, Inf
    dt = np.float32 if out == TX_F32 else np.uint16
    y = rng.standard_normal((m, ldo)).astype(np.float32)
    y0 = y if out == TX_F32 else to_bf16_bits(y)
    yf = y if out == TX_F32 else from_bf16_bits(y0)
    bx, bw, by = (runtime.buffer(a.nbytes, np.ascontiguousarray(a)) for a in (x, w, y0))
    runtime.linear_fused_device(bx.device_ptr, bw.device_ptr, by.device_ptr, m=m, n=n, k=k,
                                ldx=ldx, ldw=ldw, ldr=ldo, ldo=ldo, residual=by.device_ptr,
                                residual_dtype=out, out_dtype=out, activation="silu")
    runtime.sync()
    got = runtime.read(by, (m, ldo), dt)
    np.testing.assert_array_equal(got[:, n:], y0[:, n:])
    check(np.ascontiguousarray(got[:, :n]), xf[:, :k], wf[:, :k], None, "silu", yf[:, :n])
    for b in (bx, bw, by):
        b.close()


def test_values_that_are_not_finite_stay_in_their_row_and_column(runtime):
    for m in (4, 140):
        x, w = np.full((m, 64), 0x3F80, np.uint16), np.full((40, 64), 0x3F80, np.uint16)
        x[1, 5], w[7, 9] = 0x7FC0, 0x7F80
        got = linear_fused(x, w, out_dtype="float32", runtime=runtime)
        assert np.isnan(got[1]).all() and np.all(got[0, :7] == 64) and np.isinf(got[0, 7])
        assert np.all(got[2:, 8:] == 64)


def test_activations_far_out(runtime):
    """Values where an exponential over- or underflows."""
    v = np.array([-200, -90, -30, -10, -5.5, -1, -0.0, 0.0, 1, 5.5, 30, 90, 200], np.float32)
    for m in (1, 16):
        x = np.zeros((m, 8), np.uint16)
        x[:, 0] = 0x3F80
        w = np.zeros((v.size, 8), np.uint16)
        w[:, 0] = to_bf16_bits(v)
        for act in ACTS:
            got = linear_fused(x, w, activation=act, out_dtype="float32", runtime=runtime)
            want = oracle.activate(from_bf16_bits(w[:, 0]).astype(np.float64), act)
            assert np.isfinite(got).all()
            np.testing.assert_allclose(got, np.broadcast_to(want, got.shape), rtol=2e-6,
                                       atol=2.0**-21 * 6)


def test_refusals(runtime):
    x, w = np.zeros((4, 16), np.uint16), np.zeros((8, 16), np.uint16)
    assert linear_fused(x[:0], w, runtime=runtime).shape == (0, 8)
    for kw in (dict(bias=np.zeros(7)), dict(residual=np.zeros((4, 7), np.float32)),
               dict(residual=np.zeros((4, 8))), dict(activation="tanh"), dict(out_dtype="f16")):
        with pytest.raises(InvalidInputError):
            linear_fused(x, w, runtime=runtime, **kw)
    for a, b in ((x, w[:, :8]), (x.astype(np.float32), w), (x, w[:0]), (x[0], w)):
        with pytest.raises(InvalidInputError):
            linear_fused(a, b, runtime=runtime)
    b = runtime.buffer(4096)
    p = b.device_ptr
    ok = dict(m=4, n=8, k=16)
    runtime.linear_fused_device(p, p, p + 2048, **ok)
    for kw in (dict(ldx=12), dict(ldw=20), dict(ldx=8), dict(ldo=7), dict(n=0), dict(k=0),
               dict(m=-1), dict(out_dtype=3), dict(residual=p, residual_dtype=7),
               dict(residual=p, ldr=4), dict(residual=p + 2048, residual_dtype=TX_F32),
               dict(activation="elu"), dict(ldo=-8)):
        with pytest.raises(InvalidInputError):
            runtime.linear_fused_device(p, p, p + 2048, **{**ok, **kw})
    for args in ((p + 2, p, p), (p, p + 8, p), (p, p, p + 1), (None, p, p), (p, None, p),
                 (p, p, None)):
        with pytest.raises(InvalidInputError):
            runtime.linear_fused_device(*args, **ok)
    runtime.sync()
    b.close()


def test_wait_limit_is_reported_and_the_runtime_goes_on(runtime):
    rng = np.random.default_rng(3)
    x, xf = bf16(rng, (300, 512))
    w, wf = bf16(rng, (300, 512), 0.05)
    runtime.set_wait_limit(1)
    try:
        from tessery_b200 import DeviceTimeoutError

        with pytest.raises(DeviceTimeoutError):
            linear_fused(x, w, runtime=runtime)
    finally:
        runtime.set_wait_limit(0)
    check(linear_fused(x, w, runtime=runtime), xf, wf, None, "none", None)
