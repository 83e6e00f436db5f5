"""Attention under a score rule (layers.attention_scored / attention_scored_device) on a B200
against the formula in 64 bits, one query row at a time, and its refusals.

Tolerances, per element, with A = sum_j p_j |v_j| from the oracle and Z the largest |score| (or
scale sum |q||k|) plus the cap:
- An error dz of a score moves the output by at most 2 dz A.  fp32 route: split TF32 products are
  off by 2^-21 of sum |q||k| at worst (lo parts truncated to 2^-11, lo.lo dropped), the cap,
  bias, scaling to log2 units and exp2 by a few 2^-23 of Z; dz <= 2^-20 (Z + 1) covers them.
  P.V in split TF32 and the sums add 2^-20 A.  Gate: (2 (Z + 1) + 1) 2^-20 A.
- Few-rows route: fp32 as above.  bf16: P is rounded to TF32, 2^-11 of each weight, and scores are
  off by 2^-19 (Z + 1) (16 more additions in the tensor core, cut rather than rounded): gate
  (2^-11 + (2 (Z + 1) + 1) 2^-19) A.
- Tensor-memory route: bf16 inputs are exact, dz <= 2^-19 (Z + 1) (hardware exp2 and reciprocal);
  P is rounded to bf16, 2^-8 of each weight: 2^-8 A.  Gate: (2^-8 + 2^-18 (Z + 1)) A.
- bf16 output: 2^-8 of the value more.  A term of 1e-30 admits exact zeros."""

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200 import InvalidInputError, TX_BF16, TX_F32
from tessery_b200.layers import attention_scored
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu


def make(rng, shape, dtype, scale=1.0):
    x = (scale * rng.standard_normal(shape)).astype(np.float32)
    return (to_bf16_bits(x), from_bf16_bits(to_bf16_bits(x))) if dtype == "bf16" else (x, x)


def gate(want, mass, big, cap, route, bf16, dtype="bf16"):
    z = big + cap + 1
    if route == "scored_f32" or (route == "scored_few" and dtype == "f32"):
        rel = (2 * z + 1) * 2.0**-20
    elif route == "scored_few":
        rel = 2.0**-11 + (2 * z + 1) * 2.0**-19
    else:
        rel = 2.0**-8 + z * 2.0**-18
    return rel * mass + (np.abs(want) * 2.0**-8 if bf16 else 0.0) + 1e-30


def run_packed(runtime, lens_q, lens_k, heads, kv_heads, dim, dtype, *, out=None, seed=0,
               route=None, docs=None, prefix=None, qk_scale=1.0, touch=None, **rule):
    """Runs a packed batch and checks every sequence against the oracle."""
    rng = np.random.default_rng(seed)
    cu_q = np.concatenate([[0], np.cumsum(lens_q)]).astype(np.int32)
    cu_k = np.concatenate([[0], np.cumsum(lens_k)]).astype(np.int32)
    q, qf = make(rng, (cu_q[-1], heads, dim), dtype, qk_scale)
    k, kf = make(rng, (cu_k[-1], kv_heads, dim), dtype, qk_scale)
    v, vf = make(rng, (cu_k[-1], kv_heads, dim), dtype)
    if touch is not None:  # values written into k and v: (row, what)
        kf, vf = kf.copy(), vf.copy()
        for r, what in touch:
            kf[r], vf[r] = what, what
        k, v = (to_bf16_bits(kf), to_bf16_bits(vf)) if dtype == "bf16" else (kf, vf)
    q_docs = k_docs = None
    if docs is not None:
        k_docs = np.asarray(docs(rng, int(cu_k[-1])), np.int32)
        q_docs = np.concatenate([k_docs[b - n:b] for n, b in zip(lens_q, cu_k[1:])])
    got = attention_scored(q, k, v, cu_q=cu_q, cu_k=cu_k, out_dtype=out, prefix=prefix,
                           q_docs=q_docs, k_docs=k_docs, runtime=runtime, **rule)
    took = runtime.last_kernel()
    if route:
        assert took == route
    bf16 = got.dtype == np.uint16
    gf = from_bf16_bits(got) if bf16 else got
    rule = dict(rule)
    table = rule.pop("distance_bias", None)
    rule.setdefault("causal", True)
    for s in range(len(lens_q)):
        a, b = slice(cu_q[s], cu_q[s + 1]), slice(cu_k[s], cu_k[s + 1])
        want, mass, big = oracle.attention_scored(
            qf[a], kf[b], vf[b], table=table, prefix=0 if prefix is None else int(prefix[s]),
            q_docs=None if docs is None else q_docs[a], k_docs=None if docs is None else k_docs[b],
            **rule)
        tol = gate(want, mass, big, rule.get("softcap", 0.0), took, bf16, dtype)
        bad = ~(np.abs(gf[a] - want) <= tol) & ~(np.isnan(want) & np.isnan(gf[a])) \
            & ~(np.isinf(want) & (want == gf[a]))
        assert not bad.any(), (s, np.argwhere(bad)[:4], gf[a][bad][:4], want[bad][:4])
    return gf


LENS = [1, 0, 2, 127, 128, 129, 300, 17]
SHAPES = [(4, 2, 128), (3, 3, 64), (6, 2, 32), (2, 1, 96), (9, 3, 80), (8, 1, 40), (1, 1, 8),
          (12, 4, 72)]


def slopes_of(heads):
    return (2.0 ** (-8.0 * (1 + np.arange(heads)) / heads)).astype(np.float32)


def table_of(heads, reach, seed=3):
    return np.random.default_rng(seed).standard_normal((heads, 2 * reach + 1)).astype(np.float32)


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
def test_ragged(runtime, heads, kv_heads, dim, dtype, causal):
    run_packed(runtime, LENS, LENS, heads, kv_heads, dim, dtype, causal=causal,
               route="scored_tc" if dtype == "bf16" else "scored_f32")


@pytest.mark.parametrize("dtype,dim,route", [("bf16", 20, "scored_f32"), ("bf16", 160, "scored_f32"),
                                             ("f32", 33, "scored_f32"), ("f32", 256, "scored_f32"),
                                             ("f32", 1, "scored_f32")])
def test_other_head_dims(runtime, dtype, dim, route):
    run_packed(runtime, [5, 130, 1], [5, 130, 1], 4, 2, dim, dtype, route=route, softcap=20.0)


RULES = {
    "cap": dict(softcap=5.0),
    "cap_large": dict(softcap=50.0, qk_scale=3.0),
    "slopes": dict(slopes=True),
    "slopes_both_ways": dict(slopes=True, causal=False),
    "table": dict(table=40),
    "table_cap": dict(table=3, softcap=8.0, causal=False),
    "table_one": dict(table=0, causal=False),
    "window": dict(window=(5, -1)),
    "window_zero": dict(window=(0, 0), causal=False),
    "window_both": dict(window=(130, 7), causal=False),
    "window_right": dict(window=(-1, 20), causal=False),
    "window_prefix": dict(window=(3, -1), prefix=True),
    "prefix": dict(prefix=True),
    "prefix_cap_slopes": dict(prefix=True, softcap=15.0, slopes=True),
    "large_scores": dict(qk_scale=4.0),
}


@pytest.mark.parametrize("name", sorted(RULES))
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(4, 2, 128), (3, 1, 64)])
def test_rules(runtime, name, dtype, shape):
    rule = dict(RULES[name])
    heads, kv_heads, dim = shape
    if rule.pop("slopes", False):
        rule["slopes"] = slopes_of(heads)
    if "table" in rule:
        rule["distance_bias"] = table_of(heads, rule.pop("table"))
    if rule.pop("prefix", False):
        rule["prefix"] = np.array([0, 0, 1, 60, 128, 500, 133, 17], np.int32)
    run_packed(runtime, LENS, LENS, heads, kv_heads, dim, dtype, **rule)


DOCS = {
    "runs": lambda rng, n: np.repeat(np.arange(n), 37)[:n],
    "mixed": lambda rng, n: rng.integers(-1, 4, size=n),
    "backwards": lambda rng, n: 1000 - np.repeat(np.arange(n), 50)[:n],
    "padding_runs": lambda rng, n: np.where(np.repeat(rng.random(n) < 0.4, 20)[:n], -1,
                                            np.repeat(np.arange(n), 33)[:n]),
    "none": lambda rng, n: np.full(n, -5),
    "one": lambda rng, n: np.full(n, 2**31 - 1),
}


@pytest.mark.parametrize("name", sorted(DOCS))
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rule", [dict(causal=False), dict(window=(9, -1), softcap=9.0)])
def test_documents(runtime, name, dtype, rule):
    got = run_packed(runtime, [300, 1, 129], [300, 1, 129], 4, 2, 64, dtype, docs=DOCS[name], **rule)
    if name == "none":
        assert not got.any()


def test_documents_skip_many_tiles(runtime):
    """A long row whose documents are short: most key tiles are never visited."""
    docs = lambda rng, n: np.repeat(np.arange(n), 70)[:n]
    run_packed(runtime, [2500], [2500], 2, 1, 64, "bf16", docs=docs, causal=False)
    run_packed(runtime, [2500], [2500], 2, 1, 32, "f32", docs=docs, causal=False)


def few_rows_route(rows, dim, dtype, cap=False):
    """The kernel that takes `rows` query rows per kv head, 16-byte rows of k and v."""
    if dtype == "f32":
        return "scored_few" if rows <= 16 else "scored_f32"
    if dim <= 128:
        return "scored_few" if rows <= 8 and (dim <= 64 or cap) else "scored_tc"
    return "scored_few" if rows <= 16 else "scored_f32"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 2, 5, 17])
@pytest.mark.parametrize("shape", [(16, 8, 128), (8, 1, 64), (3, 3, 32), (6, 2, 80)])
def test_new_tokens_against_kept_keys(runtime, dtype, new, shape):
    """Few query rows, long keys: the key range is split and joined."""
    lens_k = [1, 5, 700, 3000, 129, 2049]
    lens_q = [min(new, n) for n in lens_k]
    rows = new * (shape[0] // shape[1])
    run_packed(runtime, lens_q, lens_k, *shape, dtype,
               route=few_rows_route(rows, shape[2], dtype))
    run_packed(runtime, lens_q, lens_k, *shape, dtype,
               route=few_rows_route(rows, shape[2], dtype, cap=True), softcap=10.0,
               window=(900, -1), prefix=np.array([1, 0, 3, 200, 0, 5], np.int32))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 8), (10, 2, 40), (3, 1, 72), (16, 1, 256),
                                                (7, 7, 136), (9, 3, 24)])
def test_few_rows_of_any_group_and_dim(runtime, heads, kv_heads, dim, dtype):
    """Groups that are no power of two, head_dims between the compiled ones, every rule."""
    lens_k = [300, 1, 17, 1000]
    kw = dict(route=few_rows_route(heads // kv_heads, dim, dtype))
    run_packed(runtime, [1] * 4, lens_k, heads, kv_heads, dim, dtype, out="float32", **kw)
    run_packed(runtime, [1] * 4, lens_k, heads, kv_heads, dim, dtype, slopes=slopes_of(heads),
               softcap=9.0, window=(200, -1), route="scored_few")
    run_packed(runtime, [1] * 4, lens_k, heads, kv_heads, dim, dtype,
               distance_bias=table_of(heads, 20), docs=lambda rng, n: rng.integers(-1, 3, size=n),
               **kw)
    run_packed(runtime, [1] * 4, lens_k, heads, kv_heads, dim, dtype, window=(30, 0),
               prefix=np.array([40, 0, 17, 5], np.int32), qk_scale=3.0, **kw)


@pytest.mark.parametrize("new,heads,kv_heads,dim", [(0, 3, 1, 80), (1, 8, 1, 128)])
def test_fp32_sums_over_many_keys(runtime, new, heads, kv_heads, dim):
    """Sums over many keys round to nearest: n / 8 partial sums, each off by 2^-24 / sqrt(3) of the
    sum so far in the mean square, are off by sqrt(2200 / 8) 2^-24 / sqrt(3) = 5.7e-7 of it at most,
    taken over the whole result.  Sums that cut bits off always towards zero are off by 2e-6."""
    rng = np.random.default_rng(3)
    n = 2200
    q = rng.standard_normal((new or n, heads, dim)).astype(np.float32)
    k, v = (rng.standard_normal((n, kv_heads, dim)).astype(np.float32) for _ in range(2))
    got = attention_scored(q, k, v, cu_q=[0, len(q)], cu_k=[0, n], causal=False, runtime=runtime)
    rows = slice(0, None, 97)
    want = oracle.attention_scored(q[rows], k, v)[0]
    assert np.linalg.norm(got[rows] - want) < 6e-7 * np.linalg.norm(want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_more_queries_than_keys_leaves_rows_empty(runtime, dtype):
    """nq > nk: causal rows at negative positions see nothing and are zeros."""
    got = run_packed(runtime, [10, 4, 3], [3, 4, 0], 2, 1, 64, dtype)
    assert not got[:7].any() and got[7:10].any() and not got[14:].any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_padded_layout_and_padding_values(runtime, dtype):
    """Padded rows of k and v hold NaN and Inf; query rows past a length give zeros."""
    rng = np.random.default_rng(4)
    b, lq, lk, heads, kv_heads, dim = 4, 150, 150, 4, 2, 64
    n = np.array([150, 0, 1, 97], np.int32)
    q, qf = make(rng, (b, lq, heads, dim), dtype)
    k, kf = make(rng, (b, lk, kv_heads, dim), dtype)
    v, vf = make(rng, (b, lk, kv_heads, dim), dtype)
    for s in range(b):
        for x in (kf, vf):
            x[s, n[s]:] = np.nan
            x[s, n[s] + 1::2] = np.inf
    if dtype == "bf16":
        k, v = to_bf16_bits(kf), to_bf16_bits(vf)
    got = attention_scored(q, k, v, q_lengths=n, k_lengths=n, causal=False, runtime=runtime)
    gf = from_bf16_bits(got) if dtype == "bf16" else got
    for s in range(b):
        assert not gf[s, n[s]:].any()
        want, mass, big = oracle.attention_scored(qf[s, :n[s]], kf[s, :n[s]], vf[s, :n[s]])
        tol = gate(want, mass, big, 0.0, runtime.last_kernel(), dtype == "bf16")
        assert np.all(np.abs(gf[s, :n[s]] - want) <= tol)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("dim", [64, 128])
def test_nonfinite_values_behind_the_mask(runtime, dtype, value, dim):
    """Rows that a rule closes the key to never feel its NaN or Inf: later positions, other
    documents, outside the window."""
    run_packed(runtime, [260, 40], [260, 40], 2, 1, dim, dtype, touch=[(130, value), (255, value)])
    run_packed(runtime, [260], [260], 2, 1, dim, dtype, causal=False,
               docs=lambda rng, n: np.repeat(np.arange(n), 45)[:n],
               touch=[(3, value), (100, value)])
    run_packed(runtime, [260], [260], 2, 1, dim, dtype, window=(20, -1), softcap=10.0,
               touch=[(0, value), (140, value)])
    run_packed(runtime, [1, 1], [900, 901], 2, 1, dim, dtype, window=(50, -1),
               touch=[(3, value), (400, value), (845, value)])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_bias_at_the_ends_of_its_type(runtime, dtype):
    """-inf in the table closes a key (a row closed everywhere is zeros); the lowest finite value
    does not: rows that see nothing else weigh their keys evenly."""
    low = np.finfo(np.float32).min
    t = np.zeros((2, 2 * 3 + 1), np.float32)
    t[0, :] = -np.inf
    t[1, :3] = low
    got = run_packed(runtime, [140], [140], 2, 1, 64, dtype, distance_bias=t)
    assert not got[:, 0].any()
    t[1] = low
    run_packed(runtime, [140], [140], 2, 1, 64, dtype, distance_bias=t, causal=False)


def test_empty_rows_of_both_routes_are_zeros_with_bad_keys(runtime):
    for dtype in ("bf16", "f32"):
        got = run_packed(runtime, [64], [64], 2, 1, 64, dtype, docs=lambda rng, n: np.full(n, -1),
                         touch=[(i, np.nan) for i in range(64)])
        assert not got.any()


@pytest.mark.parametrize("out", ["float32", "bf16"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_output_types(runtime, dtype, out):
    run_packed(runtime, [200, 3], [200, 3], 4, 2, 64, dtype, out=out, softcap=30.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strided_heads_of_a_fused_row(runtime, dtype):
    """q, k, v as columns of fused rows; one element of offset moves bf16 to the other route."""
    rng = np.random.default_rng(2)
    heads, kv_heads, dim, n = 4, 2, 64, 200
    width = (heads + 2 * kv_heads) * dim + 8
    code = TX_BF16 if dtype == "bf16" else TX_F32
    for offset in (0, 1):
        x, xf = make(rng, (n, width), dtype)
        buf = runtime.buffer(x.nbytes, x)
        out = runtime.buffer(n * heads * dim * 4)
        cu = runtime.buffer(8, np.array([0, n], np.int32))
        at = buf.device_ptr + offset * x.itemsize
        st = (width, dim)
        runtime.attention_scored_device(
            at, at + heads * dim * x.itemsize, at + (heads + kv_heads) * dim * x.itemsize,
            out.device_ptr, nseq=1, rows_q=n, rows_k=n, max_q=n, max_k=n, heads=heads,
            kv_heads=kv_heads, dim=dim, cu_q=cu.device_ptr, cu_k=cu.device_ptr, in_dtype=code,
            out_dtype=TX_F32, q_strides=st, k_strides=st, v_strides=st)
        runtime.sync()
        took = runtime.last_kernel()
        assert took == ("scored_tc" if dtype == "bf16" and not offset else "scored_f32")
        got = runtime.read(out, (n, heads, dim))
        cut = lambda h0, m: xf[:, offset + h0 * dim:offset + (h0 + m) * dim].reshape(n, m, dim)
        want, mass, big = oracle.attention_scored(
            cut(0, heads), cut(heads, kv_heads), cut(heads + kv_heads, kv_heads), causal=True)
        assert np.all(np.abs(got - want) <= gate(want, mass, big, 0.0, took, False))
        for b in (buf, out, cu):
            b.close()


def test_agrees_with_the_attention_without_a_rule(runtime):
    from tessery_b200 import attention

    rng = np.random.default_rng(9)
    cu = np.array([0, 40, 300], np.int32)
    q, _ = make(rng, (300, 4, 128), "bf16")
    k, kf = make(rng, (300, 2, 128), "bf16")
    v, vf = make(rng, (300, 2, 128), "bf16")
    want = attention(q, k, v, cu_seqlens=cu, causal=True, runtime=runtime)
    got = attention_scored(q, k, v, cu_q=cu, out_dtype="float32", runtime=runtime)
    np.testing.assert_allclose(got, want, atol=2 * 2.0**-8 * np.abs(vf).max(), rtol=0)


def test_same_result_every_time(runtime):
    rng = np.random.default_rng(1)
    for dtype in ("bf16", "f32"):
        q, _ = make(rng, (3, 2, 4, 64), dtype)
        k, _ = make(rng, (3, 2000, 2, 64), dtype)
        first = attention_scored(q, k, k, runtime=runtime)
        for _ in range(5):
            np.testing.assert_array_equal(attention_scored(q, k, k, runtime=runtime), first)


def test_device_lengths_out_of_range_are_reported(runtime):
    """Offsets in device memory that leave the rows: cut to fit, reported, and the runtime goes
    on."""
    x = runtime.buffer(64 * 64 * 4, np.ones((64, 64), np.float32))
    out = runtime.buffer(64 * 64 * 4)
    for cu in ([0, 90], [0, -3], [70, 80], [0, 40]):  # the last: longer than max_q
        b = runtime.buffer(8, np.array(cu, np.int32))
        runtime.attention_scored_device(
            x.device_ptr, x.device_ptr, x.device_ptr, out.device_ptr, nseq=1, rows_q=64, rows_k=64,
            max_q=32, max_k=64, heads=1, kv_heads=1, dim=64, cu_q=b.device_ptr, cu_k=b.device_ptr,
            in_dtype=TX_F32, out_dtype=TX_F32)
        with pytest.raises(InvalidInputError):
            runtime.sync()
        b.close()
    x.close()
    out.close()
    run_packed(runtime, [5], [5], 1, 1, 64, "f32")


def test_refusals(runtime):
    q = np.zeros((8, 2, 32), np.float32)
    cu = np.array([0, 8], np.int32)
    attention_scored(q, q, q, cu_q=cu, runtime=runtime)
    assert attention_scored(q[:0], q, q, cu_q=np.array([0, 0]), cu_k=cu, runtime=runtime).shape \
        == (0, 2, 32)
    assert not attention_scored(q, q[:0], q[:0], cu_q=cu, cu_k=np.array([0, 0]),
                                runtime=runtime).any()
    bad = [
        dict(cu_q=np.array([0, 7])), dict(cu_q=np.array([0, 9, 8])), dict(cu_q=np.array([8])),
        dict(), dict(cu_q=cu, q_lengths=[8]), dict(cu_q=cu, cu_k=np.array([0, 4, 8])),
        dict(cu_q=cu, softcap=-1.0), dict(cu_q=cu, softcap=np.inf), dict(cu_q=cu, scale=np.nan),
        dict(cu_q=cu, slopes=np.zeros(3)), dict(cu_q=cu, distance_bias=np.zeros((2, 4))),
        dict(cu_q=cu, slopes=np.zeros(2), distance_bias=np.zeros((2, 5))),
        dict(cu_q=cu, prefix=np.zeros(2)), dict(cu_q=cu, q_docs=np.zeros(7)),
        dict(cu_q=cu, out_dtype="int8"),
    ]
    for kw in bad:
        with pytest.raises(InvalidInputError):
            attention_scored(q, q, q, runtime=runtime, **kw)
    with pytest.raises(InvalidInputError):
        attention_scored(q, q[:, :1], q, cu_q=cu, runtime=runtime)
    with pytest.raises(InvalidInputError):
        attention_scored(np.zeros((8, 3, 32), np.float32), q, q, cu_q=cu, runtime=runtime)
    with pytest.raises(InvalidInputError):
        attention_scored(q.astype(np.float64), q, q, cu_q=cu, runtime=runtime)
    b = runtime.buffer(8 * 2 * 32 * 4)
    p = b.device_ptr
    ok = dict(nseq=1, rows_q=8, rows_k=8, max_q=8, max_k=8, heads=2, kv_heads=2, dim=32,
              in_dtype=TX_F32, out_dtype=TX_F32)
    runtime.attention_scored_device(p, p, p, p, **ok)
    for kw in (dict(dim=257), dict(dim=0), dict(kv_heads=0), dict(nseq=2), dict(reach=1 << 21,
               distance_bias=p), dict(q_docs=p), dict(in_dtype=5), dict(nseq=-1),
               dict(q_strides=(-64, 32))):
        with pytest.raises(InvalidInputError):
            runtime.attention_scored_device(p, p, p, p, **{**ok, **kw})
    with pytest.raises(InvalidInputError):
        runtime.attention_scored_device(p + 2, p, p, p, **ok)
    with pytest.raises(InvalidInputError):
        runtime.attention_scored_device(p, None, p, p, **ok)
    runtime.sync()
    b.close()


def test_wait_limit_is_reported_and_the_runtime_goes_on(runtime):
    """Waits that run out end the kernel with a status; a split call after it joins its parts as
    ever (the arrival counters have returned to zero)."""
    from tessery_b200 import DeviceTimeoutError

    runtime.set_wait_limit(1)
    try:
        for lens_q, lens_k in (([300], [300]), ([9, 9], [3000, 900])):
            with pytest.raises(DeviceTimeoutError):
                run_packed(runtime, lens_q, lens_k, 4, 2, 128, "bf16")
    finally:
        runtime.set_wait_limit(0)
    run_packed(runtime, [9, 9], [3000, 900], 4, 2, 128, "bf16", route="scored_tc")
