"""GELU in the linear layer's epilogue, on sums that are exact (one column of x is one, the rest
zero), so that the activation's own error is what is measured.

Bounds, y the sum.  fp32 results are y (1 - Q) or y Q, Q = erfc(|y| / sqrt 2) / 2 at most 1/2 and off by
2^-21 of itself near zero (a fit of 2^-24, the hardware exponential's 2^-22, eight roundings of 2^-25
on the average): 2^-22 |y|, with the two roundings behind it below 2^-21 |y|.  On the negative side the
factor vanishes and the exponent t = y^2 / 2 log2 e, rounded twice by 2^-24 of it, moves Q by ln 2 times
that: 46 ln 2 x 2^-23 down to y = -8, with the rest below 2^-16 of the value.  bf16 results: 2^-8 of the
value and 2^-19 |y|."""

import math

import numpy as np
import pytest

from tessery_b200.layers import linear_fused
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu


def gelu(y):
    return np.array([0.5 * t * math.erfc(-t / math.sqrt(2.0)) for t in y.ravel()]).reshape(y.shape)


@pytest.mark.parametrize("m", [1, 3, 40])
@pytest.mark.parametrize("n", [700, 20000])
@pytest.mark.parametrize("k", [8, 600])
@pytest.mark.parametrize("out", ["float32", "bf16"])
def test_gelu(runtime, m, n, k, out):
    x = np.zeros((m, k), np.uint16)
    x[:, k - 3] = 0x3F80  # 1
    w = np.zeros((n, k), np.uint16)
    w[:, k - 3] = to_bf16_bits(np.linspace(-9, 9, n).astype(np.float32))
    y = from_bf16_bits(w[:, k - 3]).astype(np.float64)
    got = linear_fused(x, w, activation="gelu", out_dtype=out, runtime=runtime)
    want = np.broadcast_to(gelu(y), (m, n))
    if out == "bf16":
        tol = 2.0**-8 * np.abs(want) + 2.0**-19 * np.abs(y)
        got = from_bf16_bits(got)
    else:
        tol = np.where(y > -8, np.minimum(2.0**-21 * np.abs(y), 2.0**-16 * np.abs(want)),
                       2.0**-21 * np.abs(y))
    bad = ~(np.abs(got - want) <= tol + 1e-30)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])
