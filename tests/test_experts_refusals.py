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
