"""The encoder-layer operators in CUDA graphs and on several streams (needs a B200).  A call that cuts its range over CTAs has
scratch; a graph has to keep its own, whatever calls come after the capture."""

import numpy as np
import pytest

from tessery_b200 import TX_F32

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def attention(rt, keys, seqs=2):
    """Few query rows over `keys` keys: the call, an input and the output."""
    g = torch.Generator(device="cuda").manual_seed(keys)
    q = torch.randn(seqs, 2, 4, 64, generator=g, device="cuda").bfloat16()
    k = torch.randn(seqs, keys, 2, 64, generator=g, device="cuda").bfloat16()
    out = torch.zeros(seqs, 2, 4, 64, device="cuda")

    def call(stream):
        rt.attention_scored_device(q.data_ptr(), k.data_ptr(), k.data_ptr(), out.data_ptr(),
                                   nseq=seqs, rows_q=2 * seqs, rows_k=seqs * keys, max_q=2,
                                   max_k=keys, heads=4, kv_heads=2, dim=64, out_dtype=TX_F32,
                                   stream=stream)

    return call, q, out


def linear(rt, k, m=16, n=200):
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    w = torch.randn(n, k, generator=g, device="cuda").bfloat16()
    out = torch.zeros(m, n, device="cuda")

    def call(stream):
        rt.linear_fused_device(x.data_ptr(), w.data_ptr(), out.data_ptr(), m=m, n=n, k=k,
                               out_dtype=TX_F32, activation="silu", stream=stream)

    return call, x, out


@pytest.mark.parametrize("make,small,large", [(attention, 3000, 200000), (linear, 4096, 16384)])
def test_split_calls_in_a_graph(runtime, make, small, large):
    call, x, out = make(runtime, small)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        call(stream.cuda_stream)
        runtime.sync(stream.cuda_stream)
        first = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(torch.cuda.current_stream().cuda_stream)
            call(torch.cuda.current_stream().cuda_stream)
        out.zero_()
        graph.replay()
        assert torch.equal(out, first)
        # A call that needs more scratch than any before it, and one on the runtime's own stream.
        bigger, _, other = make(runtime, large, 16)
        torch.cuda.synchronize()
        bigger(stream.cuda_stream)
        runtime.sync(stream.cuda_stream)
        want = other.clone()
        x.neg_()  # other inputs for the graph
        call(stream.cuda_stream)
        second = out.clone()
        out.zero_()
        bigger(stream.cuda_stream)
        graph.replay()
        bigger(stream.cuda_stream)
        graph.replay()
        runtime.sync(stream.cuda_stream)
        assert torch.equal(out, second) and not torch.equal(second, first)
        assert torch.equal(other, want)
    call(0)
    runtime.sync()
    assert torch.equal(out, second)
    assert np.isfinite(out.cpu().numpy()).all()
    del graph
    torch.cuda.synchronize()


@pytest.mark.parametrize("make,size", [(attention, 3000), (linear, 4096)])
def test_split_calls_on_two_streams(runtime, make, size):
    """Calls in turn on two streams and the runtime's own share the scratch one after another."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    calls = [make(runtime, size + 512 * i) for i in range(3)]
    torch.cuda.synchronize()
    want = []
    for call, _, out in calls:
        call(streams[0].cuda_stream)
        runtime.sync(streams[0].cuda_stream)
        want.append(out.clone())
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for (call, _, _), stream in zip(calls, (*streams, None), strict=True):
            call(stream.cuda_stream if stream else 0)
    for s in (*(s.cuda_stream for s in streams), 0):
        runtime.sync(s)
    torch.cuda.synchronize()
    for (_, _, out), w in zip(calls, want, strict=True):
        assert torch.equal(out, w)
