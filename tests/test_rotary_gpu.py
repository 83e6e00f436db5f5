"""The position rotation (layers.rotary / rotary_device) on a B200 against its formula in 64
bits, and its refusals.

Tolerances.  fp32: a result is x C - y S with |C|, |S| <= amplitude known to about 2^-20.4
absolute (the hardware sine and cosine after a reduction to [-pi, pi], 2^-21 each), so it is
off by at most (|x| + |y|) amplitude 2^-20.4 plus a few roundings of 2^-24; behind a norm the
row's scale adds about 2^-22.  With |x| <= 5 (and norm weights near 1) that is below 1e-5, and
the gate is 1.2e-5 times the amplitude and the row's largest value over 5 where that is more.
bf16 out: half an ulp of bf16, 2^-8 of the value (2^-9 relative to the next power of two,
doubled for a value that the fp32 error pushes across), plus the fp32 gate."""

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200 import InvalidInputError, TX_BF16, TX_F32
from tessery_b200.layers import rotary, rotary_frequencies
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu


def check(got, want, amplitude, bf16):
    big = max(1.0, float(np.abs(want).max()) / 5)
    tol = 1.2e-5 * amplitude * big + (np.abs(want) * 2.0**-8 if bf16 else 0.0)
    np.testing.assert_array_less(np.abs(got - want), tol + 1e-30)


def make(rng, shape, dtype):
    x = rng.standard_normal(shape).astype(np.float32).clip(-5, 5)
    return (to_bf16_bits(x), from_bf16_bits(to_bf16_bits(x))) if dtype == "bf16" else (x, x)


CASES = [  # heads, kv_heads, dim, rot
    (16, 8, 128, 128), (12, 12, 32, 16), (12, 12, 64, 64), (9, 3, 80, 40), (8, 1, 256, 64),
    (3, 1, 96, 24), (5, 2, 33, 32), (1, 1, 2, 2), (4, 4, 255, 254), (2, 2, 48, 48), (3, 3, 24, 8),
    (7, 1, 16, 16),
]


@pytest.mark.parametrize("heads,kv_heads,dim,rot", CASES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
def test_rotary_packed(runtime, heads, kv_heads, dim, rot, interleaved, dtype, norm):
    rng = np.random.default_rng(dim * 7 + rot)
    cu = np.array([0, 0, 1, 1, 38, 41, 41], np.int32)  # empty sequences among them
    q, qf = make(rng, (41, heads, dim), dtype)
    k, kf = make(rng, (41, kv_heads, dim), dtype)
    w = to_bf16_bits(1 + 0.1 * rng.standard_normal(dim).astype(np.float32)) if norm else None
    freq, amp = rotary_frequencies(rot, 10000.0, scaling="yarn", factor=4.0, original=2048)
    assert amp > 1
    pos = np.concatenate([np.arange(n) for n in np.diff(cu)])
    for out in ("float32", "bf16"):
        gq, gk = rotary(q, k, inv_freq=freq, amplitude=amp, interleaved=interleaved,
                        cu_seqlens=cu, q_norm_weight=w, k_norm_weight=w, out_dtype=out,
                        runtime=runtime)
        assert runtime.last_kernel() == "rotary"
        wf = None if w is None else from_bf16_bits(w)
        for got, x in ((gq, qf), (gk, kf)):
            want = oracle.rotary(x, pos, freq, amplitude=amp, interleaved=interleaved, weight=wf)
            check(from_bf16_bits(got) if out == "bf16" else got, want, amp, out == "bf16")


@pytest.mark.parametrize("tokens", [1, 7, 300, 2500])
def test_rotary_positions_far_and_padded(runtime, tokens):
    rng = np.random.default_rng(tokens)
    q, qf = make(rng, (tokens, 4, 64), "bf16")
    freq, _ = rotary_frequencies(64, 1e6)
    far = rng.integers(0, 1 << 24, size=tokens)
    got, none = rotary(q, inv_freq=freq, positions=far, out_dtype="float32", runtime=runtime)
    assert none is None
    check(got, oracle.rotary(qf, far, freq), 1.0, False)
    got, _ = rotary(q, inv_freq=freq, seq=37, out_dtype="float32", runtime=runtime)
    check(got, oracle.rotary(qf, np.arange(tokens) % 37, freq), 1.0, False)


@pytest.mark.parametrize("nseq", [1, 31, 33, 1025, 3000])
def test_rotary_many_sequences(runtime, nseq):
    rng = np.random.default_rng(nseq)
    lens = rng.integers(0, 4, size=nseq)
    lens[-1] = 3
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    q, qf = make(rng, (int(cu[-1]), 2, 32), "f32")
    freq, _ = rotary_frequencies(32, 100.0)
    got, _ = rotary(q, inv_freq=freq, cu_seqlens=cu, runtime=runtime)
    pos = np.concatenate([np.arange(n) for n in lens])
    check(got, oracle.rotary(qf, pos, freq), 1.0, False)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_inverse_returns(runtime, interleaved):
    """Turning and turning back gives the input: also the rotation's gradient, since the
    rotation is orthogonal."""
    rng = np.random.default_rng(5)
    q, _ = make(rng, (50, 3, 64), "f32")
    freq, _ = rotary_frequencies(64, 1e4)
    turned, _ = rotary(q, inv_freq=freq, seq=50, interleaved=interleaved, runtime=runtime)
    back, _ = rotary(turned, inv_freq=freq, seq=50, interleaved=interleaved, inverse=True,
                     runtime=runtime)
    np.testing.assert_allclose(back, q, atol=4e-5, rtol=0)  # two rotations' gates


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset", [0, 1])
def test_rotary_strided_in_place(runtime, dtype, offset):
    """q and k as columns of fused rows, turned in place: the v columns stay untouched.  An
    offset of one element takes the vectors' alignment away."""
    rng = np.random.default_rng(8)
    heads, kv_heads, dim, tokens = 4, 2, 64, 37
    width = (heads + 2 * kv_heads) * dim + offset
    x, xf = make(rng, (tokens, width), dtype)
    esz = x.itemsize
    buf = runtime.buffer(x.nbytes, x)
    freq, _ = rotary_frequencies(dim, 1e4)
    fb = runtime.buffer(freq.nbytes, freq)
    w = to_bf16_bits(np.ones(dim, np.float32) * 1.5)
    wb = runtime.buffer(w.nbytes, w)
    code = TX_F32 if dtype == "f32" else TX_BF16
    at = buf.device_ptr + offset * esz
    qs = (width, dim)
    runtime.rotary_device(at, at + heads * dim * esz, at, at + heads * dim * esz, tokens=tokens,
                          heads=heads, kv_heads=kv_heads, dim=dim, inv_freq=fb.device_ptr,
                          seq=tokens, q_norm_weight=wb.device_ptr, in_dtype=code, out_dtype=code,
                          q_strides=qs, k_strides=qs, q_out_strides=qs, k_out_strides=qs)
    runtime.sync()
    got = runtime.read(buf, x.shape, x.dtype)
    for b in (buf, fb, wb):
        b.close()
    np.testing.assert_array_equal(got[:, :offset], x[:, :offset])
    np.testing.assert_array_equal(got[:, offset + (heads + kv_heads) * dim:],
                                  x[:, offset + (heads + kv_heads) * dim:])
    gf = from_bf16_bits(got) if dtype == "bf16" else got
    cut = lambda a, h0, n: a[:, offset + h0 * dim:offset + (h0 + n) * dim].reshape(tokens, n, dim)
    pos = np.arange(tokens)
    check(cut(gf, 0, heads), oracle.rotary(cut(xf, 0, heads), pos, freq,
                                           weight=np.full(dim, 1.5)), 1.0, dtype == "bf16")
    check(cut(gf, heads, kv_heads), oracle.rotary(cut(xf, heads, kv_heads), pos, freq), 1.0,
          dtype == "bf16")


def test_rotary_nonfinite_values_stay_in_their_head(runtime):
    q = np.ones((3, 2, 32), np.float32)
    q[1, 0, 3] = np.nan
    q[2, 1, 0] = np.inf
    freq, _ = rotary_frequencies(32, 1e4)
    got, _ = rotary(q, inv_freq=freq, seq=3, q_norm_weight=to_bf16_bits(np.ones(32, np.float32)),
                    runtime=runtime)
    assert np.isnan(got[1, 0]).all() and np.isfinite(got[0]).all()
    assert np.isfinite(got[1, 1]).all() and np.isfinite(got[2, 0]).all()


def test_rotary_agrees_with_the_fused_prologue(runtime):
    """The half layout over the whole head, unscaled and normed, is qk_norm_rope's result."""
    from tessery_b200 import qk_norm_rope

    rng = np.random.default_rng(11)
    q, _ = make(rng, (100, 16, 128), "bf16")
    k, _ = make(rng, (100, 8, 128), "bf16")
    w = to_bf16_bits(1 + 0.02 * rng.standard_normal(128).astype(np.float32))
    want = qk_norm_rope(q, k, w, w, seq=100, out_dtype="float32", runtime=runtime)
    got = rotary(q, k, inv_freq=rotary_frequencies(128, 1e6)[0], seq=100, q_norm_weight=w,
                 k_norm_weight=w, out_dtype="float32", runtime=runtime)
    for a, b in zip(got, want):
        np.testing.assert_allclose(a, b, atol=2.4e-5, rtol=0)


def test_rotary_refusals(runtime):
    q = np.zeros((4, 2, 32), np.float32)
    freq, _ = rotary_frequencies(32)
    rotary(q, inv_freq=freq, seq=4, runtime=runtime)
    empty, _ = rotary(q[:0], inv_freq=freq, seq=4, runtime=runtime)
    assert empty.shape == (0, 2, 32)
    bad = [
        dict(), dict(seq=4, positions=np.arange(4)), dict(positions=np.arange(3)),
        dict(positions=np.array([0, 1, -1, 2])), dict(positions=np.array([0, 1, 1 << 24, 2])),
        dict(cu_seqlens=np.array([0, 3])), dict(cu_seqlens=np.array([0, 3, 2, 4])),
        dict(seq=4, q_norm_weight=np.zeros(31, np.uint16)), dict(seq=4, amplitude=np.inf),
        dict(seq=4, eps=-1.0), dict(seq=4, out_dtype="float64"),
    ]
    for kw in bad:
        with pytest.raises(InvalidInputError):
            rotary(q, inv_freq=freq, runtime=runtime, **kw)
    with pytest.raises(InvalidInputError):
        rotary(q, inv_freq=np.zeros(17, np.float32), seq=4, runtime=runtime)  # rot_dim > dim
    with pytest.raises(InvalidInputError):
        rotary(q.astype(np.float64), inv_freq=freq, seq=4, runtime=runtime)
    with pytest.raises(InvalidInputError):
        rotary(q, q[:, :, :16], inv_freq=freq, seq=4, runtime=runtime)
    b = runtime.buffer(4096)
    p = b.device_ptr
    f = runtime.buffer(64, np.zeros(16, np.float32))
    ok = dict(tokens=4, heads=2, dim=32, inv_freq=f.device_ptr, seq=4, in_dtype=TX_F32,
              out_dtype=TX_F32)
    runtime.rotary_device(p, None, p, None, **ok)
    for kw in (dict(rot_dim=31), dict(rot_dim=34), dict(dim=257), dict(heads=0),
               dict(out_dtype=TX_BF16), dict(q_out_strides=(128, 32)), dict(in_dtype=9),
               dict(q_strides=(64, 16), q_out_strides=(64, 16)), dict(inv_freq=None),
               dict(q_strides=(-64, 32))):
        with pytest.raises(InvalidInputError):
            runtime.rotary_device(p, None, p, None, **{**ok, **kw})
    with pytest.raises(InvalidInputError):
        runtime.rotary_device(p, p, p, None, kv_heads=2, **ok)
    runtime.sync()
    b.close()
    f.close()
