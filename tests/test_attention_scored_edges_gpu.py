"""Attention under a score rule at the ends of its arguments: queries before the first key with
windows of any reach, infinite and largest finite values, caps of any size, distance tables with
special values and of every place they are kept in.  Against the formula in 64 bits.

Tolerances, per element, from each row's own scores: A = sum_j p_j |v_j|, Z = the largest
scale sum |q||k| over finite products of the row, or the largest finite |score| if that is more (a
cap adds nothing: a capped score is off relative to itself).  As in test_attention_scored_gpu,
a score is off by at most 2^-20 (Z + 1) in the fp32 kernels and 2^-19 (Z + 1) in the bf16 ones,
which moves the output by twice that times A, and P.V adds 2^-20 A in fp32, 2^-16 A where P is held
in two bf16 parts (2^-17 each) and 2^-8 A where it is rounded to bf16 once."""

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200.layers import attention_scored
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu

LARGE = 2**31 - 1


def exact(q, k, v, *, softcap=0.0, slopes=None, table=None, **rule):
    """One sequence in 64 bits: the output, A and Z per row [nq, heads, dim] / [nq, heads, 1]."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    (nq, heads, dim), nk = q.shape, k.shape[0]
    group, scale = heads // k.shape[1], dim**-0.5
    seen = oracle.open_keys(nq, nk, **rule)
    dist = np.arange(nk)[None] - (np.arange(nq)[:, None] + nk - nq)
    out, mass, size = np.zeros((nq, heads, dim)), np.zeros((nq, heads, dim)), np.zeros((nq, heads, 1))
    with np.errstate(invalid="ignore", over="ignore"):
        for h in range(heads):
            for i in range(nq):
                at = np.flatnonzero(seen[i])
                if not at.size:
                    continue
                kh, vh = k[at, h // group], v[at, h // group]
                products = scale * kh * q[i, h]
                z = products.sum(-1)
                size[i, h] = np.where(np.isfinite(products), np.abs(products), 0).sum(-1).max()
                if softcap:
                    z = softcap * np.tanh(z / softcap)
                if slopes is not None:
                    z = z - float(slopes[h]) * np.abs(dist[i, at])
                if table is not None:
                    reach = table.shape[1] // 2
                    z = z + np.asarray(table[h], np.float64)[
                        np.clip(dist[i, at], -reach, reach) + reach]
                common = np.abs(z[np.abs(z) < 1e30])
                size[i, h] = max(size[i, h, 0], common.max(initial=0.0))
                if np.max(z) == -np.inf:
                    continue
                p = np.exp(z - np.max(z))
                p /= p.sum()
                used = p != 0
                out[i, h], mass[i, h] = p[used] @ vh[used], p[used] @ np.abs(vh[used])
    return out, mass, size


def relative(took, dtype, size):
    f32 = took == "scored_f32" or dtype == "f32"
    scores = 2 * (size + 1) * (2.0**-20 if f32 else 2.0**-19)
    return scores + (2.0**-20 if f32 else 2.0**-16 if took == "scored_few" else 2.0**-8)


def check(runtime, q, k, v, dtype, *, route=None, distance_bias=None, **rule):
    """Runs one sequence of float values with fp32 output and compares every element."""
    if dtype == "bf16":
        held = [to_bf16_bits(x) for x in (q, k, v)]
        q, k, v = (from_bf16_bits(x) for x in held)
    else:
        held = [np.asarray(x, np.float32) for x in (q, k, v)]
    host = dict(rule)
    if "prefix" in host:
        host["prefix"] = np.array([host["prefix"]])
    got = attention_scored(*held, cu_q=np.array([0, len(q)]), cu_k=np.array([0, len(k)]),
                           distance_bias=distance_bias, out_dtype="float32", runtime=runtime, **host)
    took = runtime.last_kernel()
    if route:
        assert took == route
    rule.setdefault("causal", True)
    want, mass, size = exact(q, k, v, table=distance_bias, **rule)
    finite = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[np.isinf(want)], want[np.isinf(want)])
    with np.errstate(invalid="ignore"):
        bad = finite & ~(np.abs(got - want) <= relative(took, dtype, size) * mass + 1e-30)
    assert not bad.any(), (took, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])
    return got


def normal(seed, nq, nk, heads, kv_heads, dim):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((nq, heads, dim)).astype(np.float32),
            *(rng.standard_normal((nk, kv_heads, dim)).astype(np.float32) for _ in range(2)))


# ROUTES: (kernel, dtype, query rows, heads, kv_heads, dim)
ROUTES = [("scored_tc", "bf16", 40, 2, 1, 64), ("scored_tc", "bf16", 40, 4, 2, 128),
          ("scored_f32", "f32", 40, 2, 1, 64), ("scored_f32", "bf16", 40, 2, 1, 160),
          ("scored_few", "bf16", 6, 1, 1, 64), ("scored_few", "f32", 6, 2, 1, 64),
          ("scored_few", "bf16", 5, 3, 1, 136)]


@pytest.mark.parametrize("kernel,dtype,nq,heads,kv_heads,dim", ROUTES)
@pytest.mark.parametrize("rule", [
    dict(causal=False, window=(LARGE, -1)), dict(causal=False, window=(LARGE, LARGE)),
    dict(causal=False, window=(LARGE - 1, 0)), dict(window=(LARGE, LARGE)),
    dict(causal=False, window=(2, 3)), dict(causal=False, window=(-1, 1)),
    dict(causal=False, window=(0, 4), prefix=2), dict(causal=False, slopes=True),
    dict(causal=False, table=True), dict(causal=False, docs=True),
    dict(causal=False, docs=True, window=(LARGE, 2), slopes=True)])
def test_queries_before_the_first_key(runtime, kernel, dtype, nq, heads, kv_heads, dim, rule):
    """More query rows than keys: the first ones stand at negative positions."""
    rule = dict(rule)
    if rule.pop("slopes", False):
        rule["slopes"] = (0.5 ** np.arange(1, heads + 1)).astype(np.float32)
    if rule.pop("table", False):
        rule["distance_bias"] = np.random.default_rng(1).standard_normal(
            (heads, 2 * 4 + 1)).astype(np.float32)
    for nk in (3, 1):
        q, k, v = normal(nk, nq, nk, heads, kv_heads, dim)
        if rule.pop("docs", False) or "k_docs" in rule:
            rule["k_docs"] = np.arange(nk, dtype=np.int32) % 2
            rule["q_docs"] = (np.arange(nq, dtype=np.int32) % 3) - 1
        check(runtime, q, k, v, dtype, route=kernel, **rule)


@pytest.mark.parametrize("kernel,dtype,nq,heads,kv_heads,dim", ROUTES)
def test_infinite_values_that_a_row_sees(runtime, kernel, dtype, nq, heads, kv_heads, dim):
    """An infinite value of v makes its column infinite, two of both signs make it NaN, and the
    other columns are as ever, whether or not a key near it is closed."""
    q, k, v = normal(3, nq, 300, heads, kv_heads, dim)
    v[20, :, 1], v[20, :, 2], v[150, :, 4] = np.inf, -np.inf, np.inf
    v[20, :, 5], v[21, :, 5], v[77, :, 7] = np.inf, -np.inf, np.nan
    check(runtime, q, k, v, dtype, route=kernel, causal=False)
    check(runtime, q, k, v, dtype, route=kernel)
    check(runtime, q, k, v, dtype, route=kernel, window=(200, -1), prefix=30)


@pytest.mark.parametrize("kernel,dtype,nq,heads,kv_heads,dim", ROUTES)
def test_infinite_scores(runtime, kernel, dtype, nq, heads, kv_heads, dim):
    """A score of -inf weighs nothing and leaves its row as it is; one of +inf makes the row NaN; a cap
    makes both finite."""
    q, k, v = normal(4, nq, 200, heads, kv_heads, dim)
    q[..., 3] = np.abs(q[..., 3]) + 0.5
    k[17, :, 3] = -np.inf
    check(runtime, q, k, v, dtype, route=kernel, causal=False)
    q[2, :, 3] *= -1  # this row's score is +inf
    check(runtime, q, k, v, dtype, route=kernel, causal=False)
    check(runtime, q, k, v, dtype, causal=False, softcap=4.0)
    k[17] = 0.0
    k[17, :, 3] = 1.0
    k[..., 5] = np.abs(k[..., 5]) + 0.5
    q[..., 5] = 0.25
    q[3, :, 5], q[4, :, 5] = -np.inf, np.inf  # every score of these rows
    got = check(runtime, q, k, v, dtype, route=kernel, causal=False)
    assert not got[3].any() and np.isnan(got[4]).all()
    check(runtime, q, k, v, dtype, causal=False, softcap=4.0)


@pytest.mark.parametrize("kernel,nq,dim", [("scored_f32", 40, 64), ("scored_few", 6, 64),
                                           ("scored_few", 6, 160)])
def test_largest_finite_values(runtime, kernel, nq, dim):
    """fp32 values whose upper TF32 part would be infinite."""
    big = np.finfo(np.float32).max
    q, k, v = normal(5, nq, 100, 2, 1, dim)
    q[..., 1] = 2.0**-126
    k[::7, :, 1] = big
    k[3::7, :, 1] = -big
    v[:, :, 0] = np.abs(v[:, :, 0])
    v[11, :, 0], v[50, :, 3] = big, -big
    check(runtime, q, k, v, "f32", route=kernel, causal=False)
    check(runtime, q, k, v, "f32", route=kernel, causal=False, softcap=10.0)


@pytest.mark.parametrize("kernel,dtype,nq,heads,kv_heads,dim", ROUTES)
@pytest.mark.parametrize("cap", [1e-9, 1e-3, 0.5, 30.0, 1e4, 1e6, 1e30])
def test_caps_of_any_size(runtime, kernel, dtype, nq, heads, kv_heads, dim, cap):
    """A capped score is off relative to itself, not to the cap; rows whose scores reach the cap do not
    touch the others."""
    q, k, v = normal(6, nq, 150, heads, kv_heads, dim)
    q[1] = 0.0
    q[2] *= 3.0
    check(runtime, q, k, v, dtype, causal=False, softcap=cap)
    if 1 < cap < 1e10:
        q[3] *= cap  # scores that reach the cap, in the same warps
        check(runtime, q, k, v, dtype, causal=False, softcap=cap)
    check(runtime, 0 * q, k, v, dtype, causal=False, softcap=cap)


@pytest.mark.parametrize("kernel,dtype,nq,heads,kv_heads,dim", ROUTES)
@pytest.mark.parametrize("reach", [3, 1500])
def test_special_values_of_a_table(runtime, kernel, dtype, nq, heads, kv_heads, dim, reach):
    """NaN reaches the rows that see it and no others; the largest finite value takes all the weight;
    -inf closes a key."""
    big = np.finfo(np.float32).max
    q, k, v = normal(7, nq, 140, heads, kv_heads, dim)
    for what in (np.nan, big, -big, -np.inf, np.inf):
        t = np.zeros((heads, 2 * reach + 1), np.float32)
        t[:, reach - 2] = what  # two keys before the query
        check(runtime, q, k, v, dtype, distance_bias=t, causal=False)
        t[:] = 0.0
        t[:, 0] = what  # and everything farther to the left
        check(runtime, q, k, v, dtype, distance_bias=t)
    t[:] = np.linspace(-2, 2, 2 * reach + 1)
    check(runtime, q, k, v, dtype, distance_bias=t, causal=False, softcap=5.0)


@pytest.mark.parametrize("heads,kv_heads,dim,reach", [
    (4, 2, 128, 700), (2, 1, 64, 1700), (4, 1, 128, 300), (4, 1, 64, 800), (8, 1, 128, 40),
    (8, 1, 64, 900), (3, 3, 128, 1500), (1, 1, 64, 3500), (4, 1, 96, 255), (2, 1, 80, 671),
    (2, 1, 128, 672)])
@pytest.mark.parametrize("rule", [dict(causal=False), dict(window=(1100, 5), causal=False, prefix=9),
                                  dict(softcap=6.0)])
def test_tables_of_every_length(runtime, heads, kv_heads, dim, reach, rule):
    """Tables that fit on chip whole and tables of which each warp keeps the part it needs, for packs
    of one, two and four heads."""
    q, k, v = normal(reach, 70, 1900, heads, kv_heads, dim)
    t = np.random.default_rng(reach).standard_normal((heads, 2 * reach + 1)).astype(np.float32)
    check(runtime, q, k, v, "bf16", route="scored_tc", distance_bias=t, **rule)


@pytest.mark.parametrize("heads,kv_heads,dim,rule", [
    (1, 1, 64, {}), (8, 1, 64, {}), (4, 1, 32, {}), (2, 1, 128, dict(softcap=20.0)),
    (8, 1, 128, dict(softcap=20.0)), (16, 1, 256, {}), (3, 1, 136, {})])
def test_few_rows_hold_the_weights_in_two_parts(runtime, heads, kv_heads, dim, rule):
    q, k, v = normal(8, 1, 1500, heads, kv_heads, dim)
    check(runtime, q, k, v, "bf16", route="scored_few", **rule)
