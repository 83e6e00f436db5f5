"""Calls of the operators for layers of experts on arrays that are refused before any memory is taken
for them (no GPU: a runtime that keeps its buffers in host memory)."""

import numpy as np
import pytest
from test_experts_host import Host

from tessery_b200 import InvalidInputError
from tessery_b200.layers import block_norm, experts_linear, experts_route

F = np.ones((6, 16), np.float32)


@pytest.mark.parametrize("seq", [0, 3])
def test_a_gate_without_rows(seq):
    """It would be as if there were no gate."""
    block_norm(F, F, gate=F[:2], seq=3, runtime=Host())
    with pytest.raises(InvalidInputError):
        block_norm(F, F, gate=F[:0], seq=seq, runtime=Host())


class NoMemory(Host):
    """Host, of which a call may not take more than a few rows' memory before it is refused."""

    def workspace(self, name, size):
        assert size < 1 << 20
        return super().workspace(name, size)


@pytest.mark.parametrize("top_k", [17, 2**20, 2**45, 2**70])
def test_more_choices_than_experts(top_k):
    """Before room for as many is taken on the device, and filled on the host."""
    with pytest.raises(InvalidInputError):
        experts_route(F, top_k, runtime=NoMemory())
    with pytest.raises(InvalidInputError):
        experts_route(F[:0], top_k, runtime=NoMemory())


@pytest.mark.parametrize("call", [
    lambda a: experts_route(F, 2, bias=a(16), runtime=Host()),
    lambda a: experts_linear(F.astype(np.uint16), np.ones((3, 8, 16), np.uint16), [0, 2, 4, 6],
                             bias=a(3, 8), runtime=Host()),
    lambda a: block_norm(F, F, places=np.zeros((6, 2), int), weights=a(6, 2), runtime=Host())])
def test_bf16_patterns_where_values_are_wanted(call):
    """As numbers the patterns would be other values."""
    call(lambda *shape: np.ones(shape))
    call(lambda *shape: np.ones(shape, int))
    with pytest.raises(InvalidInputError):
        call(lambda *shape: np.full(shape, 0x3F80, np.uint16))
