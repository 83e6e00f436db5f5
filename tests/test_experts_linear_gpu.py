"""The experts' products (layers.experts_linear / experts_linear_device) on a B200 against the
formula in 64 bits.

Tolerance, per element, with A = sum |x w| + |bias|: as for the linear layer, (k / 16 + 16) 2^-23 A for
the sum, 1.13 for the steepest activation, 2^-20 A for the activation itself.  Gated, the two sums'
errors go through the product: A is |act(g)| A_u + A_g |u|, and the two errors' product is below 2^-12
of that.  bf16 output: 2^-8 of the value."""

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200 import DeviceTimeoutError, InvalidInputError, TX_BF16, TX_F32
from tessery_b200.layers import experts_linear
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def bf16(rng, shape, scale=1.0):
    bits = to_bf16_bits((scale * rng.standard_normal(shape)).astype(np.float32))
    return bits, from_bf16_bits(bits)


def check(got, xf, wf, offsets, **kw):
    g = from_bf16_bits(got) if got.dtype == np.uint16 else got
    want, mass = oracle.experts_linear(xf, wf, offsets, **kw)
    tol = 1.13 * (xf.shape[1] / 16 + 16) * 2.0**-23 * 1.001 * mass + 2.0**-20 * mass
    if got.dtype == np.uint16:
        tol = tol + 2.0**-8 * np.abs(want)
    np.testing.assert_array_less(np.abs(g - want), tol + 1e-30)


def plan(rng, tokens, experts, top_k, skew=0.7):
    """(offsets, order) of a routing that likes some experts more and gives some tokens none."""
    liked = skew * rng.standard_normal(experts) + rng.gumbel(size=(tokens, experts))
    ids = np.argsort(-liked, axis=1)[:, :top_k]
    ids[rng.random(tokens) < 0.1] = experts
    flat = ids.reshape(-1)
    by = np.argsort(flat, kind="stable")
    offsets = np.searchsorted(flat[by], np.arange(experts + 1))
    return offsets, np.where(np.arange(len(flat)) < offsets[-1], by, -1)


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 8, 4), (3, 5, 2), (40, 7, 3),
                                                  (130, 3, 1), (200, 64, 8), (600, 2, 2)])
@pytest.mark.parametrize("n,k", [(1, 1), (8, 9), (65, 63), (136, 200), (300, 72)])
@pytest.mark.parametrize("gated", [False, True])
def test_sizes(runtime, tokens, experts, top_k, n, k, gated):
    rng = np.random.default_rng(tokens + n)
    x, xf = bf16(rng, (tokens, k))
    wide = 2 * n if gated else n
    w, wf = bf16(rng, (experts, wide, k), k**-0.5)
    bias = rng.standard_normal((experts, wide)).astype(np.float32)
    offsets, order = plan(rng, tokens, experts, top_k)
    kw = dict(order=order, top_k=top_k, gated=gated, activation=ACTS[(tokens + n) % 5])
    for out in ("float32", "bf16"):
        check(experts_linear(x, w, offsets, bias=bias, out_dtype=out, runtime=runtime, **kw), xf, wf,
              offsets, bias=bias, **kw)
    rows, rf = bf16(rng, (tokens * top_k, k))
    kw.update(order=None, top_k=1)
    check(experts_linear(rows, w, offsets, runtime=runtime, **kw), rf, wf, offsets, **kw)
    if offsets[-1]:
        assert runtime.last_kernel() == "experts_linear"


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts", [[1] * 9, [0, 5, 0, 300, 128, 129, 0], [2, 7, 8, 9, 16, 17]])
def test_activations(runtime, act, gated, counts):
    rng = np.random.default_rng(len(counts))
    offsets = np.r_[0, np.cumsum(counts)]
    n, k = 72, 136
    x, xf = bf16(rng, (offsets[-1], k), 3.0)
    wide = 2 * n if gated else n
    w, wf = bf16(rng, (len(counts), wide, k), k**-0.5)
    for bias in (None, rng.standard_normal((len(counts), wide)).astype(np.float32)):
        for out in ("float32", "bf16"):
            kw = dict(gated=gated, activation=act, bias=bias)
            check(experts_linear(x, w, offsets, out_dtype=out, runtime=runtime, **kw), xf, wf, offsets,
                  **kw)


@pytest.mark.parametrize("rows,experts,n,k", [(700, 4, 260, 1100), (20, 6, 130, 2056), (3, 2, 16, 9000),
                                              (9000, 5, 40, 600), (12000, 8, 264, 72)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("out", ["float32", "bf16"])
def test_long_sums_and_several_tiles(runtime, rows, experts, n, k, gated, out):
    rng = np.random.default_rng(rows)
    x, xf = bf16(rng, (rows, k))
    wide = 2 * n if gated else n
    w, wf = bf16(rng, (experts, wide, k), k**-0.5)
    offsets = np.sort(np.r_[0, rng.integers(0, rows + 1, experts - 1), rows])
    kw = dict(gated=gated, activation="silu" if gated else "none")
    got = experts_linear(x, w, offsets, out_dtype=out, runtime=runtime, **kw)
    some = np.unique(np.r_[offsets[:-1], offsets[1:] - 1, rng.integers(0, rows, 60)]).clip(0, rows - 1)
    of = np.searchsorted(offsets, some, side="right") - 1
    # The rows looked at, as a problem of their own.
    small = np.searchsorted(of, np.arange(experts + 1))
    check(got[some], xf[some], wf, small, **kw)
    assert np.array_equal(got, experts_linear(x, w, offsets, out_dtype=out, runtime=runtime, **kw))


@pytest.mark.parametrize("gated,n,k,out", [(True, 150, 200, "bf16"), (True, 128, 64, "float32"),
                                           (False, 300, 72, "bf16"), (False, 257, 513, "bf16"),
                                           (False, 512, 130, "float32"), (False, 1000, 2056, "float32"),
                                           (True, 520, 2056, "float32")])
@pytest.mark.parametrize("gather", [False, True])
def test_tiles_of_two_blocks(runtime, gated, n, k, out, gather):
    """Rows enough for tiles of 256 rows: experts without rows, with one, with half a tile, with several."""
    rng = np.random.default_rng(n + k)
    counts = np.array([0, 3000, 1, 127, 128, 129, 0, 257, 5000, 300, 255, 0])
    rows, experts, top_k = int(counts.sum()), len(counts), 2
    offsets = np.r_[0, np.cumsum(counts)]
    tokens = -(-rows // top_k) + 40  # some tokens without an expert
    order = np.full(tokens * top_k, -1)
    order[:rows] = rng.permutation(tokens * top_k)[:rows]
    x, xf = bf16(rng, (tokens if gather else rows, k))
    wide = 2 * n if gated else n
    w, wf = bf16(rng, (experts, wide, k), k**-0.5)
    bias = rng.standard_normal((experts, wide)).astype(np.float32)
    kw = dict(gated=gated, activation="silu" if gated else "gelu_tanh", bias=bias)
    plan = dict(order=order, top_k=top_k) if gather else {}
    got = experts_linear(x, w, offsets, out_dtype=out, runtime=runtime, **kw, **plan)
    some = np.unique(np.r_[0, offsets[1:] - 1, offsets[:-1], rng.integers(0, rows, 150)])
    some = some[(some >= 0) & (some < rows)]
    of = np.searchsorted(offsets, some, side="right") - 1
    small = np.searchsorted(of, np.arange(experts + 1))
    check(got[some], xf[order[some] // top_k if gather else some], wf, small, **kw)
    assert not got[rows:].any()
    for _ in range(3):
        again = experts_linear(x, w, offsets, out_dtype=out, runtime=runtime, **kw, **plan)
        assert np.array_equal(got, again)


def device_call(runtime, dtype=torch.bfloat16, rows=37, n=24, k=40, experts=4, ldx=56, ldw=48, ldo=29,
                offsets=(0, 9, 9, 30, 33), **kw):
    """A call whose x, w and out lie inside wider rows: (out, untouched mask, exact)."""
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    x = torch.randn(rows, ldx, generator=g, device="cuda").bfloat16()
    w = torch.randn(experts, n + 3, ldw, generator=g, device="cuda").bfloat16()
    x[:, k:], w[:, :, k:] = float("nan"), float("nan")  # columns past k may hold anything
    out = torch.full((rows + 2, ldo), 77.0, device="cuda").to(dtype)
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    runtime.experts_linear_device(
        x.data_ptr(), w.data_ptr(), out.data_ptr(), offsets=at.data_ptr(), tokens=rows, top_k=1,
        num_experts=experts, n=n, k=k, ldx=ldx, ldw=ldw, expert_stride=(n + 3) * ldw, ldo=ldo,
        out_dtype=TX_BF16 if dtype == torch.bfloat16 else TX_F32, **kw)
    runtime.sync(kw.get("stream"))
    return out, x[:, :k].double(), w[:, :n, :k].double()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ldo", [24, 29, 32])
def test_strides_and_rows_behind(runtime, dtype, ldo):
    out, x, w = device_call(runtime, dtype, ldo=ldo)
    for e, (a, b) in enumerate(((0, 9), (9, 9), (9, 30), (30, 33))):
        want = x[a:b] @ w[e].t()
        tol = 2.0**-18 * (x[a:b].abs() @ w[e].abs().t()) + (
            2.0**-8 * want.abs() if dtype == torch.bfloat16 else 0)
        assert ((out[a:b, :24].double() - want).abs() <= tol).all()
    assert (out[33:] == 77).all() and (out[:, 24:] == 77).all()


@pytest.mark.parametrize("offsets", [(0, 9, 5, 30, 33), (0, 9, 9, 40, 33), (0, -4, 9, 30, 33)])
def test_offsets_that_fall_or_leave_the_rows(runtime, offsets):
    with pytest.raises(InvalidInputError):
        device_call(runtime, offsets=offsets)
    device_call(runtime)  # and the runtime goes on


def test_order_outside_x(runtime):
    x = torch.ones(3, 16, device="cuda").bfloat16()
    w = torch.ones(1, 8, 16, device="cuda").bfloat16()
    out = torch.zeros(6, 8, device="cuda")
    offsets = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    for bad in (6, -1, 2**31 - 1):
        order = torch.tensor([0, 1, 2, bad, 4, 5], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        runtime.experts_linear_device(
            x.data_ptr(), w.data_ptr(), out.data_ptr(), offsets=offsets.data_ptr(), tokens=3, top_k=2,
            num_experts=1, n=8, k=16, order=order.data_ptr(), out_dtype=TX_F32)
        with pytest.raises(InvalidInputError):
            runtime.sync()


def test_streams_and_a_graph(runtime):
    """Calls on other streams, and a captured one replayed with other inputs."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(90, 64, generator=g, device="cuda").bfloat16()
    w = torch.randn(3, 80, 64, generator=g, device="cuda").bfloat16()
    offsets = torch.tensor([0, 50, 50, 90], dtype=torch.int32, device="cuda")
    out = torch.zeros(90, 40, device="cuda")

    def call(stream):
        runtime.experts_linear_device(
            x.data_ptr(), w.data_ptr(), out.data_ptr(), offsets=offsets.data_ptr(), tokens=90,
            top_k=1, num_experts=3, n=40, k=64, gated=True, activation="silu", out_dtype=TX_F32,
            stream=stream)

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        call(stream.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(torch.cuda.current_stream().cuda_stream)
        x.neg_()
        offsets.copy_(torch.tensor([0, 0, 88, 90], dtype=torch.int32))
        call(stream.cuda_stream)
        want = out.clone()
        out.zero_()
        graph.replay()
        runtime.sync(stream.cuda_stream)
    assert torch.equal(out, want) and want.any()
    call(0)
    runtime.sync()
    assert torch.equal(out, want)
    del graph
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows,n", [(9000, 256), (100, 40)])
@pytest.mark.parametrize("gather", [False, True])
def test_wait_limit_is_reported_and_the_runtime_goes_on(runtime, rows, n, gather):
    """A limit of one cycle runs out in the waits of either kernel; the next call is right again."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(rows, 4096, generator=g, device="cuda").bfloat16()
    w = torch.randn(2, n, 4096, generator=g, device="cuda").mul(2.0**-6).bfloat16()
    cut = rows // 3
    offsets = torch.tensor([0, cut, rows], dtype=torch.int32, device="cuda")
    order = torch.arange(rows, dtype=torch.int32, device="cuda")
    out = torch.zeros(rows, n, device="cuda").bfloat16()
    want = torch.cat([x[:cut].double() @ w[0].double().t(), x[cut:].double() @ w[1].double().t()])
    torch.cuda.synchronize()

    def call():
        runtime.experts_linear_device(
            x.data_ptr(), w.data_ptr(), out.data_ptr(), offsets=offsets.data_ptr(), tokens=rows,
            top_k=1, num_experts=2, n=n, k=4096, order=order.data_ptr() if gather else None)
        runtime.sync()

    runtime.set_wait_limit(1)
    try:
        with pytest.raises(DeviceTimeoutError):
            call()
    finally:
        runtime.set_wait_limit(0)
    call()
    # bf16's 2^-8 of the value, and 4096 / 16 + 16 cut additions of 2^-23 of sums of about 64.
    assert ((out.double() - want).abs() <= 2.0**-8 * want.abs() + 272 * 2.0**-23 * 64).all()


def test_refusals(runtime):
    b = runtime.buffer(1 << 20)
    p = b.device_ptr
    ok = dict(offsets=p + 1024, tokens=8, top_k=2, num_experts=4, n=16, k=32)
    call = runtime.experts_linear_device
    call(p, p + 65536, p + 262144, **ok)
    for kw in (dict(num_experts=0), dict(num_experts=1025), dict(n=0), dict(k=0), dict(top_k=0),
               dict(ldx=24), dict(ldx=36), dict(ldw=24), dict(ldw=36), dict(ldo=15),
               dict(expert_stride=16 * 32 - 8), dict(expert_stride=16 * 32 + 4), dict(bias=p + 2),
               dict(offsets=p + 2), dict(order=p + 1), dict(out_dtype=2), dict(activation="other"),
               dict(gated=True, expert_stride=16 * 32), dict(n=2**30), dict(tokens=2**30, top_k=4)):
        before = runtime.launch_count()
        with pytest.raises(InvalidInputError):
            call(p, p + 65536, p + 262144, **{**ok, **kw})
        assert runtime.launch_count() == before
    for at in ((0, p, p), (p, 0, p), (p, p, 0), (p + 8, p, p + 512), (p, p + 8, p + 512),
               (p, p + 512, p + 1), (p, p + 512, p)):
        with pytest.raises(InvalidInputError):
            call(*at, **ok)
    call(p, p + 65536, p + 262144, **{**ok, "tokens": 0})
    runtime.sync()
    b.close()
