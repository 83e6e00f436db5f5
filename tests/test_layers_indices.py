"""Index arrays of the encoder-layer operators that int32 cannot hold (no GPU)."""

import numpy as np
import pytest
from test_layers_threads import HostRuntime

from tessery_b200 import InvalidInputError
from tessery_b200.layers import attention_scored, rotary

X = np.ones((4, 2, 8), np.float32)
FREQ = np.ones(4, np.float32)
PADDED = X[None]
BAD = [2**32, 2**32 + 1, -(2**32), 0.5, np.nan, np.inf, 2**63]


def array(good, at, value):
    """`good` with one entry replaced, in a type that holds it."""
    a = np.array(good, dtype=np.uint64 if value == 2**63 else np.float64
                 if isinstance(value, float) else np.int64)
    a[at] = value
    return a


@pytest.mark.parametrize("value", BAD)
@pytest.mark.parametrize("name,good", [("positions", [0, 1, 2, 3]), ("cu_seqlens", [0, 2, 4])])
def test_rotary(name, good, value):
    rotary(X, X, inv_freq=FREQ, runtime=HostRuntime(), **{name: np.array(good, np.int64)})
    with pytest.raises(InvalidInputError):
        rotary(X, X, inv_freq=FREQ, runtime=HostRuntime(), **{name: array(good, 1, value)})


@pytest.mark.parametrize("value", BAD)
@pytest.mark.parametrize("name,good", [("cu_q", [0, 2, 4]), ("cu_k", [0, 2, 4]), ("prefix", [1, 1]),
                                       ("q_docs", [0, 0, 1, 1]), ("k_docs", [0, 0, 1, 1])])
def test_attention_packed(name, good, value):
    ok = dict(cu_q=np.array([0, 2, 4]), cu_k=np.array([0, 2, 4]), runtime=HostRuntime())
    if name.endswith("docs"):
        ok.update(q_docs=np.array(good), k_docs=np.array(good))
    attention_scored(X, X, X, **{**ok, name: np.array(good, np.int64)})
    attention_scored(X, X, X, **{**ok, name: np.array(good, np.float64)})
    with pytest.raises(InvalidInputError):
        attention_scored(X, X, X, **{**ok, name: array(good, 1, value)})


@pytest.mark.parametrize("value", BAD)
@pytest.mark.parametrize("name", ["q_lengths", "k_lengths"])
def test_attention_padded(name, value):
    attention_scored(PADDED, PADDED, PADDED, runtime=HostRuntime(), **{name: [3]})
    with pytest.raises(InvalidInputError):
        attention_scored(PADDED, PADDED, PADDED, runtime=HostRuntime(), **{name: array([3], 0, value)})


def test_norm_weights_are_bit_patterns():
    rotary(X, X, inv_freq=FREQ, seq=4, q_norm_weight=np.full(8, 0x3F80), runtime=HostRuntime())
    with pytest.raises(InvalidInputError):
        rotary(X, X, inv_freq=FREQ, seq=4, q_norm_weight=np.ones(8, np.float32),
               runtime=HostRuntime())
