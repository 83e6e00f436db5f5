"""The experts' products on a B200 where a result is small beside its sums, and for fp32 results of
long sums, against the formula in 64 bits."""

import math

import numpy as np
import pytest

from tessery_b200.layers import experts_linear
from tessery_b200.workloads import from_bf16_bits

pytestmark = pytest.mark.gpu

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
