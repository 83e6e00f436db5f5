"""The experts' products on a B200 where a result is small beside its sums, and for fp32 results of
long sums, against the formula in 64 bits."""

import math

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200 import TX_F32, InvalidInputError
from tessery_b200.layers import experts_linear
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

ERFC = np.vectorize(math.erfc)
FORMULA = {
    "gelu": lambda y: 0.5 * y * ERFC(-y / math.sqrt(2)),
    "gelu_tanh": lambda y: y / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y**3))),
    "silu": lambda y: y / (1 + np.exp(-y)),
}


@pytest.mark.parametrize("out", ["bf16", "float32"])
@pytest.mark.parametrize("act", list(FORMULA))
def test_gates_far_below_zero(runtime, act, out):
    """Gates from -8 (tanh: -6) to 8 that are exact, each a bias with rows of zeros, and up halves to
    4096.  bf16 results within half a step (2^-8 of the value), fp32 ones within 2^-17: the argument
    of the exponential, at most 32, comes out of at most six roundings of 2^-24, and the polynomials,
    the hardware's exponential and reciprocal (2^-22) and the product add less than 2^-18."""
    rng = np.random.default_rng(7)
    n = 640
    x = np.zeros((3, 8), np.uint16)
    w = np.zeros((2, 2 * n, 8), np.uint16)
    bias = np.empty((2, 2 * n), np.float32)
    bias[:, :n] = np.linspace(-6 if act == "gelu_tanh" else -8, 8, 2 * n).reshape(2, n)
    bias[:, n:] = rng.choice([-1, 1], (2, n)) * 2.0 ** rng.uniform(-4, 12, (2, n))
    got = experts_linear(x, w, [0, 1, 3], gated=True, activation=act, bias=bias, out_dtype=out,
                         runtime=runtime)
    got = from_bf16_bits(got) if out == "bf16" else got
    b = bias.astype(np.float64)[[0, 1, 1]]
    want = FORMULA[act](b[:, :n]) * b[:, n:]
    rel = 2.0**-8 + 2.0**-17 if out == "bf16" else 2.0**-17
    np.testing.assert_array_less(np.abs(got - want), rel * np.abs(want) + 1e-30)


@pytest.mark.parametrize("gated,n,k,out", [(False, 129, 72, "bf16"), (False, 160, 200, "float32"),
                                           (False, 255, 40, "bf16"), (False, 520, 1100, "float32"),
                                           (True, 65, 72, "bf16"), (True, 130, 700, "float32"),
                                           (True, 257, 200, "bf16")])
def test_widest_tiles_of_gathered_rows(runtime, gated, n, k, out):
    """Rows of tokens in any order, enough that tiles are 256 columns wide: last columns and rows of
    every kind, experts without rows, with one and with several tiles.  Tolerance as in
    test_experts_linear_gpu.py."""
    rng = np.random.default_rng(n)
    counts = np.array([0, 4000, 1, 127, 128, 129, 0, 6001, 5, 300, 0])
    rows, experts, top_k = int(counts.sum()), len(counts), 3
    offsets = np.r_[0, np.cumsum(counts)]
    tokens = -(-rows // top_k) + 50
    order = np.full(tokens * top_k, -1)
    order[:rows] = rng.permutation(tokens * top_k)[:rows]
    wide = 2 * n if gated else n
    x = to_bf16_bits(rng.standard_normal((tokens, k)).astype(np.float32))
    w = to_bf16_bits((k**-0.5 * rng.standard_normal((experts, wide, k))).astype(np.float32))
    bias = rng.standard_normal((experts, wide)).astype(np.float32)
    kw = dict(gated=gated, activation="silu" if gated else "relu", bias=bias)
    got = experts_linear(x, w, offsets, order=order, top_k=top_k, out_dtype=out, runtime=runtime, **kw)
    assert not got[rows:].any()
    for _ in range(2):
        again = experts_linear(x, w, offsets, order=order, top_k=top_k, out_dtype=out, runtime=runtime,
                               **kw)
        assert np.array_equal(got, again)
    some = np.unique(np.r_[offsets[1:] - 1, offsets[:-1], rng.integers(0, rows, 200)]).clip(0, rows - 1)
    small = np.searchsorted(np.searchsorted(offsets, some, side="right") - 1, np.arange(experts + 1))
    want, mass = oracle.experts_linear(from_bf16_bits(x)[order[some] // top_k], from_bf16_bits(w), small,
                                       **kw)
    got = from_bf16_bits(got) if out == "bf16" else got
    tol = 1.13 * (k / 16 + 16) * 2.0**-23 * 1.001 * mass + 2.0**-20 * mass
    tol = tol + (2.0**-8 * np.abs(want) if out == "bf16" else 0)
    np.testing.assert_array_less(np.abs(got[some] - want), tol + 1e-30)


def test_negative_entries_of_a_plan_of_many_choices(runtime):
    """Of 1000 choices a token, 2^32 - 1 is one of token 4294967, which is there: the library's own
    call takes a number of rows of x apart from that of the plan."""
    x = torch.ones(4_300_000, 8, device="cuda").bfloat16()
    w = torch.ones(1, 8, 8, device="cuda").bfloat16()
    out = torch.zeros(6, 8, device="cuda")
    offsets = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    for entries, bad in (([0, 1, 2, 4000, 4, 5], False), ([0, 1, 2, -1, 4, 5], True)):
        order = torch.tensor(entries, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        rc = runtime._lib.tx_experts_linear(
            runtime._pointer, x.data_ptr(), 8, len(x), w.data_ptr(), 8, 64, None, out.data_ptr(), TX_F32,
            8, offsets.data_ptr(), order.data_ptr(), 6, 1, 1000, 8, 8, 0, 0, None)
        assert rc == 0
        if bad:
            with pytest.raises(InvalidInputError):
                runtime.sync()
        else:
            runtime.sync()
        assert (out == 8).all()


def parts_bound(k):
    """What an fp32 result may be off by, relative to the sum of its terms' magnitudes: in parts of 512
    columns each of 32 additions of 16 products cuts less than a step of 2^-23 off, each part is added
    with a rounding, and 16 more for the 16 products' own alignment, as in test_experts_linear_gpu.py."""
    return (512 / 16 + -(-k // 512) + 16) * 2.0**-23


@pytest.mark.parametrize("rows,experts,n,k,gather", [
    (3, 2, 16, 16384, True), (40, 3, 130, 20000, False), (300, 2, 260, 16392, True),
    (4000, 2, 512, 16384, False), (4000, 2, 300, 16384, True)])
@pytest.mark.parametrize("gated", [False, True])
def test_long_sums_of_one_sign(runtime, rows, experts, n, k, gather, gated):
    """Where every addition cuts off in the same direction: a single accumulator over k would be off by
    more than twice the bound (test_experts_sums.py)."""
    rng = np.random.default_rng(rows + k)
    wide = 2 * n if gated else n
    x = to_bf16_bits(rng.uniform(0.5, 1, (rows, k)).astype(np.float32))
    w = to_bf16_bits((rng.uniform(0.5, 1, (experts, wide, k)) / k).astype(np.float32))
    offsets = np.linspace(0, rows, experts + 1).astype(int)
    order = rng.permutation(rows) if gather else None
    got = experts_linear(x, w, offsets, order=order, gated=gated, out_dtype="float32", runtime=runtime)
    some = np.unique(np.r_[offsets[1:] - 1, offsets[:-1], rng.integers(0, rows, 60)])
    some = some[some < rows]
    small = np.searchsorted(np.searchsorted(offsets, some, side="right") - 1, np.arange(experts + 1))
    want, _ = oracle.experts_linear(from_bf16_bits(x)[order[some] if gather else some],
                                    from_bf16_bits(w), small, gated=gated)
    rel = np.abs(got[some] - want) / want
    # Gated, both sums' errors are in the product, and its rounding.
    bound = parts_bound(k) * (2.001 if gated else 1) + 2.0**-23
    print(f"worst {rel.max() * 2**23:.1f}, bound {bound * 2**23:.1f} of 2^-23")
    assert rel.max() <= bound


@pytest.mark.parametrize("gated", [False, True])
def test_bf16_results_of_very_long_sums(runtime, gated):
    """2^21 columns of one sign: half a step of bf16 and no more (a single accumulator cuts off about
    2^-23 at each of 131072 additions, 1 % in all)."""
    rng = np.random.default_rng(21)
    rows, n, k = 2, 8, 1 << 21
    wide = 2 * n if gated else n
    x = to_bf16_bits(rng.uniform(0.5, 1, (rows, k)).astype(np.float32))
    w = to_bf16_bits((rng.uniform(0.5, 1, (1, wide, k)) / k).astype(np.float32))
    got = from_bf16_bits(experts_linear(x, w, [0, rows], gated=gated, runtime=runtime))
    want, _ = oracle.experts_linear(from_bf16_bits(x), from_bf16_bits(w), [0, rows], gated=gated)
    # The parts' own: 4096 of them added with a rounding each (2^-12 at worst; 2^-18 in the mean).
    np.testing.assert_array_less(np.abs(got - want), (2.0**-8 + 2.0**-12 * (1 + gated)) * want)
