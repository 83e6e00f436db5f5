"""The operators for layers of experts on two streams at once, and a wait that runs out in the widest
tiles of gathered rows (on a B200)."""

import pytest

from tessery_b200 import DeviceTimeoutError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def layer(runtime, seed, tokens, experts, top_k, n, k):
    """(queue on a stream, results): a routing with its plan, gated products of gathered rows, products
    of rows by expert, and the rows joined."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = tokens * top_k

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def ints(*shape):
        return torch.zeros(*shape, dtype=torch.int32, device="cuda")

    logits, x = normal(tokens, experts), normal(tokens, k).bfloat16()
    up = normal(experts, 2 * n, k).mul(k**-0.5).bfloat16()
    down = normal(experts, k, n).mul(n**-0.5).bfloat16()
    ids, weights, order, places = ints(tokens, top_k), normal(tokens, top_k), ints(rows), ints(rows)
    offsets, u, d = ints(experts + 1), normal(rows, n).bfloat16(), normal(rows, k).bfloat16()
    out, h = normal(tokens, k), normal(tokens, k).bfloat16()
    residual = normal(tokens, k)

    def queue(stream):
        s = stream.cuda_stream
        runtime.experts_route_device(
            logits.data_ptr(), ids.data_ptr(), weights.data_ptr(), tokens=tokens, num_experts=experts,
            top_k=top_k, offsets=offsets.data_ptr(), order=order.data_ptr(), places=places.data_ptr(),
            stream=s)
        runtime.experts_linear_device(
            x.data_ptr(), up.data_ptr(), u.data_ptr(), offsets=offsets.data_ptr(),
            order=order.data_ptr(), tokens=tokens, top_k=top_k, num_experts=experts, n=n, k=k,
            gated=True, activation="silu", stream=s)
        runtime.experts_linear_device(
            u.data_ptr(), down.data_ptr(), d.data_ptr(), offsets=offsets.data_ptr(), tokens=tokens,
            top_k=top_k, num_experts=experts, n=k, k=n, stream=s)
        runtime.block_norm_device(
            residual.data_ptr(), d.data_ptr(), rows=tokens, cols=k, out=out.data_ptr(), h=h.data_ptr(),
            places=places.data_ptr(), weights=weights.data_ptr(), top_k=top_k, y_rows=rows,
            before=dict(kind="rms"), stream=s)

    return queue, (ids, weights, order, places, offsets, u, d, out, h)


@pytest.mark.parametrize("sizes", [((6000, 16, 4, 256, 256), (3000, 64, 8, 192, 136)),
                                   ((9, 8, 2, 64, 64), (5000, 8, 2, 512, 256))])
def test_two_streams_at_once(runtime, sizes):
    """Two layers, one on each stream, queued in turn without waiting: each is, bit by bit, what it is
    alone.  (Routings of many tokens share the runtime's scratch.)"""
    layers = [layer(runtime, i, *s) for i, s in enumerate(sizes)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    want = []
    for (queue, results), stream in zip(layers, streams, strict=True):
        queue(stream)
        runtime.sync(stream.cuda_stream)
        want.append([r.clone() for r in results])
        for r in results:
            r.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for (queue, _), stream in zip(layers, streams, strict=True):
            queue(stream)
    for stream in streams:
        runtime.sync(stream.cuda_stream)
    for (_, results), wanted in zip(layers, want, strict=True):
        for a, b in zip(results, wanted, strict=True):
            assert torch.equal(a, b)


@pytest.mark.parametrize("gated", [False, True])
def test_wait_limit_in_the_widest_tiles_of_gathered_rows(runtime, gated):
    """A limit of one cycle runs out where the whole sum is waited for; it is reported, and the next
    call is right.  (Parts of fp32 sums come sooner than the limit is looked at.)"""
    g = torch.Generator(device="cuda").manual_seed(3)
    rows, n, k = 9000, 256 if gated else 512, 4096
    x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    w = torch.randn(2, n * (2 if gated else 1), k, generator=g, device="cuda").mul(k**-0.5).bfloat16()
    cut = rows // 3
    offsets = torch.tensor([0, cut, rows], dtype=torch.int32, device="cuda")
    order = torch.randperm(rows, generator=g, device="cuda").int()
    out = torch.zeros(rows, n, device="cuda").bfloat16()
    xs = x.double()[order.long()]
    want = torch.cat([xs[:cut] @ w[0].double().t(), xs[cut:] @ w[1].double().t()])
    mass = torch.cat([xs[:cut].abs() @ w[0].double().abs().t(), xs[cut:].abs() @ w[1].double().abs().t()])
    if gated:
        mass = mass[:, :n] * want[:, n:].abs() + want[:, :n].abs() * mass[:, n:]
        want = want[:, :n] * want[:, n:]
    torch.cuda.synchronize()

    def call():
        runtime.experts_linear_device(
            x.data_ptr(), w.data_ptr(), out.data_ptr(), offsets=offsets.data_ptr(),
            order=order.data_ptr(), tokens=rows, top_k=1, num_experts=2, n=n, k=k, gated=gated)
        runtime.sync()

    runtime.set_wait_limit(1)
    try:
        with pytest.raises(DeviceTimeoutError):
            call()
    finally:
        runtime.set_wait_limit(0)
    call()
    # (k / 16 + 16) cut additions of 2^-23, gated of both sums, and the output's rounding.
    tol = (k / 16 + 16) * 2.0**-23 * 1.001 * mass + (2.0**-8 + 2.0**-23) * want.abs()
    assert ((out.double() - want).abs() <= tol).all()
