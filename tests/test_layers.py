"""Host-side parts of the encoder-layer operators (no GPU)."""

import numpy as np
import pytest

from tessery_b200 import InvalidInputError
from tessery_b200.layers import rotary_frequencies


def test_frequencies_plain_and_linear():
    f, amp = rotary_frequencies(128, 1e6)
    np.testing.assert_array_equal(f, (1e6 ** (-np.arange(64) / 64)).astype(np.float32))
    assert amp == 1.0
    g, amp = rotary_frequencies(128, 1e6, scaling="linear", factor=4.0)
    np.testing.assert_allclose(g, f / 4, rtol=1e-7)
    assert amp == 1.0


def test_frequencies_ntk_keeps_the_fastest_and_divides_the_slowest():
    f, _ = rotary_frequencies(64, 1e4)
    g, _ = rotary_frequencies(64, 1e4, scaling="ntk", factor=8.0)
    assert g[0] == f[0] == 1.0
    np.testing.assert_allclose(g[-1], f[-1] / 8, rtol=1e-6)
    assert np.all(np.diff(g / f) < 0)


def test_frequencies_yarn_by_parts():
    f, _ = rotary_frequencies(128, 1e4)
    g, amp = rotary_frequencies(128, 1e4, scaling="yarn", factor=16.0, original=4096)
    assert amp == pytest.approx(0.1 * np.log(16) + 1)
    turns = f.astype(np.float64) * 4096 / (2 * np.pi)
    np.testing.assert_array_equal(g[turns > 34], f[turns > 34])
    slow = turns < 0.9
    np.testing.assert_allclose(g[slow], f[slow] / 16, rtol=1e-6)
    assert np.all(np.diff(g / f) <= 1e-7)
    same, amp = rotary_frequencies(128, 1e4, scaling="yarn", factor=1.0)
    np.testing.assert_array_equal(same, f)
    assert amp == 1.0


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=8, theta=0.0),
                                dict(rot_dim=8, factor=0.5), dict(rot_dim=8, scaling="other"),
                                dict(rot_dim=8, scaling="yarn", beta_fast=1.0),
                                dict(rot_dim=8, original=0)])
def test_frequencies_refusals(kw):
    with pytest.raises(InvalidInputError):
        rotary_frequencies(**kw)
