"""The norms after and before a block with its gate and residual (layers.block_norm /
block_norm_device) on a B200 against the formulas in 64 bits.

Tolerance.  A row's sums have at most 32 terms in a thread and 11 steps over threads, each off by 2^-24 of
the whole: 43 x 2^-24 = 2^-18.6, of which half goes into a norm's factor and, for LayerNorm, once more
through the mean; rsqrt adds 2^-22 and the products a few 2^-24.  A joined sum of up to 9 rows adds 9 x
2^-24 of its terms.  The gate is 2^-17 of the largest magnitude in the row's sum out, and for h, which
divides by out's root mean square, of h's largest times one plus that magnitude over the root mean
square.  bf16: 2^-8 of the value."""

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200 import InvalidInputError, TX_BF16, TX_F32
from tessery_b200.layers import block_norm
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def values(rng, shape, dtype="f32", scale=1.0, middle=0.0):
    x = (middle + scale * rng.standard_normal(shape)).astype(np.float32)
    return (to_bf16_bits(x), from_bf16_bits(to_bf16_bits(x))) if dtype == "bf16" else (x, x)


def norm_of(rng, cols, kind, dtype, offset=0.0, bias=False):
    w, wf = values(rng, cols, dtype, 0.2, 1.0 - offset)
    norm, exact = dict(kind=kind, weight=w, offset=offset), dict(kind=kind, weight=wf, offset=offset)
    if bias:
        norm["bias"], exact["bias"] = values(rng, cols, dtype, 0.3)
    return norm, exact


def check(got, x, y, **kw):
    """got: (out, h) of block_norm, bf16 as bits."""
    with np.errstate(invalid="ignore", divide="ignore"):
        out, h = oracle.block_norm(x, y, **kw)
    terms = np.abs(out)
    if x is not None:
        terms = np.maximum(terms, np.abs(kw.get("x_scale", 1.0) * x))
    if y is not None:
        rest = {k: v for k, v in kw.items() if k not in ("before", "x_scale")}
        z = np.abs(oracle.block_norm(None, y, **rest)[0])
        if kw.get("after"):
            # A LayerNorm's parts before they cancel in its bias, the joined sum before its norm.
            z = np.maximum(z, np.abs(kw.get("y_scale", 1.0)) * np.max(z, axis=-1, keepdims=True))
        if kw.get("places") is not None and not kw.get("after"):
            a = {**rest, "weights": np.abs(kw["weights"])}
            z = np.maximum(z, np.abs(oracle.block_norm(None, np.abs(y), **a)[0]))
        terms = np.maximum(terms, z)
    big = np.max(terms, axis=-1, keepdims=True)
    rms = np.sqrt(np.mean(out * out, axis=-1, keepdims=True) + 1e-6)
    tol = {0: 2.0**-17 * big, 1: 2.0**-17 * big if kw.get("before") is None else
           2.0**-17 * np.max(np.abs(h), axis=-1, keepdims=True) * (1 + big / rms)}
    for i, (g, want) in enumerate(zip(got, (out, h), strict=True)):
        b16 = g.dtype == np.uint16
        g = from_bf16_bits(g) if b16 else g
        limit = tol[i] + (2.0**-8 if b16 else 0.0) * np.abs(want) + 1e-30
        np.testing.assert_array_less(np.abs(g - want), limit)


COLS = [1, 2, 7, 8, 31, 32, 100, 255, 256, 264, 384, 511, 512, 520, 768, 1000, 1023, 1024, 1032, 2048,
        2049, 4096, 4104, 5000, 8192, 16383, 16384]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("after,before", [("rms", "rms"), ("layer", "layer"), (None, "layer"),
                                          ("rms", None), (None, None)])
def test_sizes(runtime, cols, after, before):
    rng = np.random.default_rng(cols)
    rows = 19 if cols < 3000 else 3
    i = COLS.index(cols)
    x, xf = values(rng, (rows, cols), "bf16" if i % 2 else "f32")
    y, yf = values(rng, (rows, cols), "f32" if i % 3 else "bf16", 2.0, 0.3)
    kw, exact = {}, {}
    for name, kind in (("after", after), ("before", before)):
        if kind:
            kw[name], exact[name] = norm_of(rng, cols, kind, "bf16" if i % 4 < 2 else "f32",
                                            offset=float(i % 2), bias=kind == "layer")
    kw.update(x_scale=0.5, y_scale=1.25)
    exact.update(x_scale=0.5, y_scale=1.25)
    for out, h in (("float32", "bf16"), ("bf16", "float32")):
        check(block_norm(x, y, out_dtype=out, h_dtype=h, runtime=runtime, **kw), xf, yf, **exact)
    assert runtime.last_kernel() == "block_norm"


@pytest.mark.parametrize("cols", [48, 50, 1024, 2000])
@pytest.mark.parametrize("top_k", [1, 2, 8, 9])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_joined_rows(runtime, cols, top_k, dtype):
    rng = np.random.default_rng(cols + top_k)
    rows = 50
    y, yf = values(rng, (rows * top_k, cols), dtype)
    places = rng.permutation(rows * top_k).reshape(rows, top_k).astype(np.int32)
    places[rng.random(places.shape) < 0.2] = -1
    places[7] = -1  # a row without any
    places[9] = 5  # and one with the same row again and again
    unread = np.setdiff1d(np.arange(rows * top_k), places)
    if unread.size:
        y = y.copy()
        y[unread] = np.nan if dtype == "f32" else 0x7FC0  # rows of nobody may hold anything
    weights = rng.random((rows, top_k)).astype(np.float32)
    weights[places < 0] = np.nan
    x, xf = values(rng, (rows, cols))
    for after in (None, "rms"):
        kw, exact = {}, {}
        if after:
            kw["after"], exact["after"] = norm_of(rng, cols, after, "bf16")
        kw["before"], exact["before"] = norm_of(rng, cols, "layer", "f32", bias=True)
        for b in (kw, exact):
            b.update(places=places, weights=np.where(places < 0, 0, weights).astype(np.float32))
        got = block_norm(x, y, runtime=runtime, **{**kw, "weights": weights})
        check(got, xf, yf, **exact)
        check(block_norm(None, y, runtime=runtime, **kw), None, yf, **exact)


@pytest.mark.parametrize("rows,cols", [(9000, 72), (9000, 50), (5000, 264), (3000, 600), (2500, 1024),
                                       (2500, 1030), (700, 4096), (400, 9000), (3000, 383),
                                       (1500, 2001), (500, 5001)])
def test_many_rows(runtime, rows, cols):
    """More rows than are in work at once, plain and joined."""
    rng = np.random.default_rng(rows)
    x, xf = values(rng, (rows, cols))
    n, ne = norm_of(rng, cols, "layer", "f32", bias=True)
    for top_k in (0, 2):
        y, yf = values(rng, (rows * max(1, top_k), cols), "bf16")
        kw = {}
        if top_k:
            kw = dict(places=rng.permutation(rows * top_k).reshape(rows, top_k),
                      weights=rng.random((rows, top_k)).astype(np.float32))
        gate, gf = values(rng, (7, cols))
        seq = -(-rows // 7)
        check(block_norm(x, y, after=n, before=n, gate=gate, seq=seq, runtime=runtime, **kw), xf, yf,
              after=ne, before=ne, gate=gf, gate_row=np.arange(rows) // seq, **kw)


@pytest.mark.parametrize("gate_dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [40, 41, 1500])
def test_gates(runtime, cols, gate_dtype):
    rng = np.random.default_rng(cols)
    rows = 60
    x, xf = values(rng, (rows, cols))
    y, yf = values(rng, (rows, cols), "bf16")
    cu = np.array([0, 0, 13, 13, 59, 60, 60], np.int32)
    for gates, where, row in ((1, {}, np.zeros(rows, int)), (rows, dict(seq=1), np.arange(rows)),
                              (3, dict(seq=25), np.arange(rows) // 25),
                              (6, dict(cu_seqlens=cu), np.repeat(np.arange(6), np.diff(cu)))):
        gate, gf = values(rng, (gates, cols), gate_dtype)
        n, ne = norm_of(rng, cols, "rms", "bf16")
        check(block_norm(x, y, after=n, before=n, gate=gate, runtime=runtime, **where), xf, yf,
              after=ne, before=ne, gate=gf, gate_row=row)


def test_one_side_alone(runtime):
    """A plain norm of x, a norm of y alone, and norms without weights."""
    rng = np.random.default_rng(2)
    x, xf = values(rng, (9, 300))
    y, yf = values(rng, (9, 300), "bf16")
    for kind in ("rms", "layer"):
        plain = dict(kind=kind, eps=1e-3)
        check(block_norm(x, before=plain, runtime=runtime), xf, None, before=plain)
        check(block_norm(None, y, after=plain, runtime=runtime), None, yf, after=plain)
    zeros = block_norm(np.zeros((4, 16), np.float32), before=dict(kind="layer"), runtime=runtime)
    assert not zeros[0].any() and not zeros[1].any()
    out, h = block_norm(np.empty((0, 16), np.float32), runtime=runtime)
    assert out.shape == h.shape == (0, 16)


@pytest.mark.parametrize("cols,ld,start", [(64, 72, 0), (64, 67, 0), (64, 72, 3), (61, 64, 0),
                                           (1024, 1040, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_in_place_and_columns_behind(runtime, cols, ld, start, dtype):
    g = torch.Generator(device="cuda").manual_seed(cols + ld)
    code = TX_BF16 if dtype == torch.bfloat16 else TX_F32
    x, y, h = (torch.randn(30, ld + start, generator=g, device="cuda").to(dtype) for _ in range(3))
    w = torch.rand(cols + start, generator=g, device="cuda").to(dtype)
    before = [t.clone() for t in (x, y, h)]
    norm = dict(kind="rms", weight=w[start:].data_ptr(), dtype=code)
    torch.cuda.synchronize()
    at = [t[:, start:].data_ptr() for t in (x, y, h)]
    runtime.block_norm_device(at[0], at[1], rows=30, cols=cols, out=at[0], h=at[2], x_dtype=code,
                              y_dtype=code, out_dtype=code, h_dtype=code, after=norm, before=norm,
                              ldx=ld + start, ldy=ld + start, ldo=ld + start, ldh=ld + start)
    runtime.sync()
    wf = w[start:].double().cpu().numpy()

    def part(t):
        return t[:, start:start + cols].double().cpu().numpy()

    exact = dict(kind="rms", weight=wf)
    out, want = oracle.block_norm(part(before[0]), part(before[1]), after=exact, before=exact)
    loose = 2.0**-8 if code == TX_BF16 else 0.0
    np.testing.assert_allclose(part(x), out, rtol=loose, atol=2.0**-16 * np.abs(out).max())
    np.testing.assert_allclose(part(h), want, rtol=loose, atol=2.0**-15 * np.abs(want).max())
    assert torch.equal(y, before[1])
    for t, was in ((x, before[0]), (h, before[2])):
        t[:, start:start + cols] = was[:, start:start + cols]
        assert torch.equal(t, was)


def test_places_outside_y(runtime):
    y = torch.ones(4, 16, device="cuda")
    out = torch.zeros(2, 16, device="cuda")
    w = torch.ones(2, 2, device="cuda")
    for bad in (4, 2**31 - 1):
        places = torch.tensor([[0, bad], [1, 2]], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        runtime.block_norm_device(None, y.data_ptr(), rows=2, cols=16, out=out.data_ptr(),
                                  y_dtype=TX_F32, places=places.data_ptr(), weights=w.data_ptr(),
                                  top_k=2, y_rows=4)
        with pytest.raises(InvalidInputError):
            runtime.sync()
    assert (out[1] == 2).all()


def test_infinities_and_nan_stay_in_their_rows(runtime):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((40, 128)).astype(np.float32)
    x[3, 5], x[8, 0] = np.nan, np.inf
    n = dict(kind="layer")
    out, h = block_norm(x, before=n, h_dtype="float32", runtime=runtime)
    np.testing.assert_array_equal(out, x)
    bad = np.zeros(40, bool)
    bad[[3, 8]] = True
    assert np.isnan(h[bad]).all() and np.isfinite(h[~bad]).all()


def test_refusals(runtime):
    b = runtime.buffer(1 << 16)
    p = b.device_ptr
    f32 = dict(x_dtype=TX_F32, y_dtype=TX_F32, out_dtype=TX_F32, h_dtype=TX_F32)
    ok = dict(rows=4, cols=16, out=p + 1024, h=p + 2048, **f32)
    call = runtime.block_norm_device
    call(p, p + 512, **ok)
    norm = dict(kind="rms", weight=p)
    call(p, p + 512, after=norm, before=norm, **ok)
    join = dict(places=p + 4096, weights=p + 8192, top_k=2, y_rows=8)
    call(p, p + 512, **join, **ok)
    gate = dict(gate=p + 16384, gate_rows=1)
    call(p, p + 512, **gate, **ok)
    call(p, p + 512, **{**ok, "out": p})  # in place
    for kw in (dict(cols=0), dict(cols=16385), dict(out=None, h=None), dict(out=p + 2048),
               dict(x_dtype=2), dict(h_dtype=7), dict(ldx=15), dict(ldy=15), dict(ldo=15), dict(ldh=15),
               dict(x_scale=np.inf), dict(y_scale=np.nan), dict(out=p, out_dtype=TX_BF16),
               dict(out=p, ldo=24), dict(h=p + 2049), dict(after={**norm, "kind": "other"}),
               dict(after={**norm, "size": 3}), dict(after={**norm, "eps": -1.0}),
               dict(after={**norm, "eps": np.nan}), dict(before={**norm, "weight": p + 2}),
               dict(before={**norm, "dtype": 2}), dict(before={**norm, "offset": np.inf}),
               {**join, "top_k": 0}, {**join, "top_k": 33}, {**join, "weights": None}, {**join, "places": p + 2},
               {**join, "out": p + 512}, {**gate, "gate_rows": 2}, {**gate, "gate_rows": 0},
               {**gate, "gate_rows": 3, "seq": 1}, {**gate, "ldg": 8}, {**gate, "gate_dtype": 2},
               {**gate, "cu_seqlens": p, "seq": 4}, {**gate, "cu_seqlens": p + 1},
               {**gate, "gate": p + 2}):
        before = runtime.launch_count()
        with pytest.raises(InvalidInputError):
            call(p, p + 512, **{**ok, **kw})
        assert runtime.launch_count() == before
    with pytest.raises(InvalidInputError):
        call(None, None, **ok)
    with pytest.raises(InvalidInputError):
        call(p, None, **join, **ok)
    runtime.sync()
    b.close()
