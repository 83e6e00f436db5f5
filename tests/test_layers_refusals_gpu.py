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


@pytest.mark.parametrize("tokens,heads,strides,fits", [
    (4, 2, (64, 32), True), (4, 2, (32, 32), False), (4, 2, (32, 128), True),
    (4, 2, (32, 127), False), (4, 2, (63, 32), False), (4, 3, (64, 96), False),
    (2, 2, (64, 96), True), (3, 2, (64, 96), True), (4, 2, (96, 64), True), (2, 2, (65, 40), False),
    (1, 2, (0, 32), True), (4, 1, (32, 0), True), (4, 2, (0, 32), False), (4, 2, (64, 31), False),
    (2, 40, (32, 64), True), (3, 40, (32, 64), False)])
def test_rotary_output_strides(runtime, tokens, heads, strides, fits):
    """Exactly the strides under which no two output heads share an element are taken: compared with
    the elements counted one by one."""
    dim = 32
    at = [t * strides[0] + h * strides[1] for t in range(tokens) for h in range(heads)]
    elements = [a + c for a in at for c in range(dim)]
    assert fits == (len(set(elements)) == len(elements))
    x = np.random.default_rng(0).standard_normal((tokens, heads, dim)).astype(np.float32)
    buf, out = runtime.buffer(x.nbytes, x), runtime.buffer(4 * (max(elements) + 1))
    freq = runtime.buffer(256)  # zeros: the rotation leaves the values as they are
    kw = dict(tokens=tokens, heads=heads, dim=dim, inv_freq=freq.device_ptr, seq=tokens,
              in_dtype=TX_F32, out_dtype=TX_F32, q_out_strides=strides)
    if fits:
        runtime.rotary_device(buf.device_ptr, None, out.device_ptr, None, **kw)
        runtime.sync()
        got = runtime.read(out, (max(elements) + 1,))
        np.testing.assert_allclose(got[elements], x.ravel(), rtol=1e-6, atol=1e-6)
    else:
        refused(runtime, runtime.rotary_device, buf.device_ptr, None, out.device_ptr, None, **kw)
    for b in (buf, out, freq):
        b.close()


def test_rotary_one_output_for_both(runtime, block):
    kw = dict(tokens=2, heads=1, kv_heads=1, dim=32, inv_freq=block + 4096, seq=2, in_dtype=TX_F32,
              out_dtype=TX_F32)
    runtime.rotary_device(block, block + 512, block + 1024, block + 2048, **kw)
    refused(runtime, runtime.rotary_device, block, block + 512, block + 1024, block + 1024, **kw)
