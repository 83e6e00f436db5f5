"""What the encoder-layer operators refuse on device pointers (needs a B200): a refused call queues
nothing."""

import numpy as np
import pytest

from tessery_b200 import InvalidInputError, TX_F32

pytestmark = pytest.mark.gpu


@pytest.fixture
def block(runtime):
    b = runtime.buffer(8192)
    yield b.device_ptr
    b.close()


def refused(runtime, call, *args, **kw):
    before = runtime.launch_count()
    with pytest.raises(InvalidInputError):
        call(*args, **kw)
    assert runtime.launch_count() == before
    runtime.sync()


@pytest.mark.parametrize("name", ["positions", "cu_seqlens", "inv_freq"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_rotary_misaligned_words(runtime, block, name, off):
    ok = dict(tokens=4, heads=2, dim=32, inv_freq=block + 4096, in_dtype=TX_F32, out_dtype=TX_F32)
    where = {"positions": dict(positions=block + 5120), "cu_seqlens": dict(
        cu_seqlens=block + 5120, nseq=1), "inv_freq": dict(seq=4)}[name]
    runtime.rotary_device(block, None, block, None, **ok, **where)
    bad = {**ok, **where}
    bad[name] += off
    refused(runtime, runtime.rotary_device, block, None, block, None, **bad)


@pytest.mark.parametrize("name", ["cu_q", "cu_k", "q_lengths", "k_lengths", "slopes", "distance_bias",
                                  "prefix", "q_docs", "k_docs"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_attention_misaligned_words(runtime, block, name, off):
    ok = dict(nseq=1, rows_q=8, rows_k=8, max_q=8, max_k=8, heads=2, kv_heads=2, dim=32,
              in_dtype=TX_F32, out_dtype=TX_F32)
    at = block + 6144  # zeros: no rows, no prefix, document 0
    if name.endswith("docs"):
        ok.update(q_docs=at, k_docs=at)
    elif name.startswith("cu"):
        ok.update(cu_q=at, cu_k=at)
    else:
        ok[name] = at
    runtime.attention_scored_device(block, block, block, block + 2048, **ok)
    ok[name] += off
    refused(runtime, runtime.attention_scored_device, block, block, block, block + 2048, **ok)
