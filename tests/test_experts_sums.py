"""The bound on the experts' fp32 results of long sums tells a sum in parts from a single accumulator
(no GPU: the tensor core's additions, which cut off instead of rounding, restated in 64 bits)."""

import numpy as np
import pytest

BITS = 24  # of the accumulator


def cut(v):
    """v >= 0 without the bits behind the first 24."""
    step = 2.0 ** (np.floor(np.log2(v)) - (BITS - 1))
    return np.floor(v / step) * step


def accumulate(products):
    """Sixteen products at once, their sum exact, added to an accumulator that is cut."""
    acc = np.zeros(products.shape[0])
    for i in range(0, products.shape[1], 16):
        acc = cut(acc + products[:, i:i + 16].sum(1))
    return acc


@pytest.mark.parametrize("k", [16384, 20000])
def test_the_bound_separates_parts_from_one_accumulator(k):
    bound = (512 / 16 + -(-k // 512) + 16) * 2.0**-23  # parts_bound of test_experts_linear_edges_gpu.py
    rng = np.random.default_rng(k)
    products = rng.uniform(0.5, 1, (40, k)) * rng.uniform(0.5, 1, (40, k)) / k
    want = products.sum(1)
    one = (want - accumulate(products)) / want
    parts = np.zeros(40, np.float32)
    for i in range(0, k, 512):
        parts += accumulate(products[:, i:i + 512]).astype(np.float32)
    assert one.min() > 2 * bound
    assert np.abs((want - parts) / want).max() < bound / 2
