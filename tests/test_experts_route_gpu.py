"""Routing of tokens to experts (layers.experts_route / experts_route_device) on a B200 against the
formula in 64 bits.  Experts and the plan have to be equal; the weights, with logits of at most 12:
the difference of two logits is off by 2^-20, which is as much of its exponential, the exponential
by 2 units (2^-22), and sums of at most 1024 terms, a quotient and a product add less than 2^-19 in
all: 2^-18 of the value."""

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200 import InvalidInputError, TX_BF16
from tessery_b200.layers import experts_route
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def check(got, logits, top_k, **kw):
    want = oracle.experts_route(logits, top_k, **kw)
    for a, b in zip((got.experts, got.offsets, got.order, got.places),
                    (want[0], want[2], want[3], want[4]), strict=True):
        np.testing.assert_array_equal(a, b)
    np.testing.assert_allclose(got.weights, want[1], rtol=2.0**-18, atol=1e-37)


def logits_of(rng, tokens, experts, dtype="f32"):
    x = (1.5 * rng.standard_normal((tokens, experts))).astype(np.float32).clip(-12, 12)
    return (to_bf16_bits(x), from_bf16_bits(to_bf16_bits(x))) if dtype == "bf16" else (x, x)


@pytest.mark.parametrize("experts", [1, 2, 4, 7, 16, 17, 32, 33, 60, 64, 100, 128, 160, 256, 300, 512,
                                     1000, 1024])
@pytest.mark.parametrize("tokens,dtype", [(1, "f32"), (37, "bf16"), (300, "f32")])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_sizes(runtime, experts, tokens, dtype, scores):
    rng = np.random.default_rng(experts + tokens)
    x, xf = logits_of(rng, tokens, experts, dtype)
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32)
    for top_k in {1, min(8, experts), min(32, experts)}:
        for b in (None, bias):
            for renormalise in (True, False):
                kw = dict(scores=scores, bias=b, renormalise=renormalise, scale=1.5)
                check(experts_route(x, top_k, runtime=runtime, **kw), xf, top_k, **kw)
    assert runtime.last_kernel() == "experts_route"


@pytest.mark.parametrize("experts,groups,top_groups", [(8, 2, 1), (60, 4, 3), (64, 8, 2), (160, 8, 5),
                                                       (256, 8, 4), (256, 64, 9), (48, 48, 20),
                                                       (1024, 16, 3), (9, 3, 3)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("with_bias", [True, False])
def test_groups(runtime, experts, groups, top_groups, best, with_bias):
    rng = np.random.default_rng(groups)
    x, xf = logits_of(rng, 150, experts, "bf16" if best == 1 else "f32")
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32) if with_bias else None
    top_k = min(8, experts // groups * top_groups)
    kw = dict(scores="sigmoid" if best == 2 else "softmax", bias=bias, groups=groups,
              top_groups=top_groups, group_best=best)
    check(experts_route(x, top_k, runtime=runtime, **kw), xf, top_k, **kw)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_ties_go_to_the_lower_index(runtime, scores):
    rng = np.random.default_rng(3)
    x = rng.integers(-2, 3, (200, 40)).astype(np.float32)
    for kw in (dict(), dict(bias=np.zeros(40, np.float32)), dict(groups=5, top_groups=2),
               dict(bias=np.repeat(np.float32([0.5, 0.25, 0, 0.5]), 10))):
        check(experts_route(x, 6, scores=scores, runtime=runtime, **kw), x, 6, scores=scores, **kw)
    zero = np.where(rng.random((64, 40)) < 0.5, np.float32(0.0), np.float32(-0.0))
    assert np.all(experts_route(zero, 3, runtime=runtime).experts == [0, 1, 2])


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_candidates_closer_than_fp32_tells(runtime, scores):
    """Biases that bring every other expert next to the one before it."""
    rng = np.random.default_rng(11)
    differ = 0
    for i in range(60):
        x = rng.standard_normal((1, 32)).astype(np.float32)
        s = 1 / (1 + np.exp(-x[0].astype(np.float64)))
        if scores == "softmax":
            s = np.exp(x[0].astype(np.float64))
            s /= s.sum()
        bias = (0.2 * rng.standard_normal(32)).astype(np.float32)
        for e in range(1, 32, 2):
            bias[e] = s[e - 1] + bias[e - 1] - s[e]
        kw = dict(scores=scores, bias=bias)
        if i % 2:
            kw.update(groups=4, top_groups=2)
        check(experts_route(x, 5, runtime=runtime, **kw), x, 5, **kw)
        c = s + bias
        differ += np.min(np.abs(np.diff(np.sort(c)))) < 2.0**-23
    assert differ > 30


def test_closed_experts_and_rows(runtime):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((90, 24)).astype(np.float32)
    x[rng.random(x.shape) < 0.7] = -np.inf
    x[3] = -np.inf
    bias = rng.standard_normal(24).astype(np.float32)
    bias[[1, 20]] = -np.inf
    lengths = [10, 0, 30]
    for kw in (dict(), dict(bias=bias), dict(bias=bias, groups=4, top_groups=2),
               dict(lengths=lengths, seq=30), dict(bias=bias, lengths=lengths, seq=30)):
        for renormalise in (True, False):
            kw["renormalise"] = renormalise
            check(experts_route(x, 6, runtime=runtime, **kw), x, 6, **kw)
    nothing = experts_route(np.full((5, 8), -np.inf, np.float32), 2, runtime=runtime)
    assert np.all(nothing.experts == -1) and not nothing.weights.any() and not nothing.offsets.any()


def test_nan_ranks_below_every_number(runtime):
    x = np.float32([[1, np.nan, 3, 2], [np.nan, np.nan, -np.inf, -1], [np.nan] * 4])
    got = experts_route(x, 3, scores="sigmoid", renormalise=False, runtime=runtime)
    np.testing.assert_array_equal(got.experts, [[2, 3, 0], [3, 0, 1], [0, 1, 2]])
    assert np.isfinite(got.weights[0]).all() and np.isnan(got.weights[1, 1:]).all()


@pytest.mark.parametrize("experts,top_k", [(16, 4), (40, 4), (64, 10), (640, 4)])
def test_nan_among_softmax_scores(runtime, experts, top_k):
    """One NaN logit leaves the choice among the others as it is without that expert."""
    rng = np.random.default_rng(experts)
    x = rng.standard_normal((9, experts)).astype(np.float32)
    bias = rng.standard_normal(experts).astype(np.float32)
    x[np.arange(9), rng.integers(0, experts, 9)] = np.nan
    without = np.where(np.isnan(x), np.float32(-np.inf), x)
    for kw in (dict(bias=bias), dict(groups=4, top_groups=2), dict(bias=bias, groups=8, top_groups=4)):
        got = experts_route(x, top_k, runtime=runtime, **kw)
        np.testing.assert_array_equal(got.experts, oracle.experts_route(without, top_k, **kw)[0])


@pytest.mark.parametrize("experts,top_k", [(16, 4), (64, 8), (64, 12), (640, 16)])
@pytest.mark.parametrize("level", [100.0, -800.0])
def test_scores_without_a_bias_are_told_apart_by_their_logits(runtime, experts, top_k, level):
    """Sigmoids that 64 bits do not tell apart, in groups of which all stay."""
    rng = np.random.default_rng(experts)
    x = np.float32(level) + rng.permuted(np.tile(np.arange(experts, dtype=np.float32), (7, 1)), axis=1) / 16
    got = experts_route(x, top_k, scores="sigmoid", groups=4, top_groups=4, renormalise=False,
                        runtime=runtime)
    np.testing.assert_array_equal(got.experts, np.argsort(-x, axis=1, kind="stable")[:, :top_k])


def test_far_logits(runtime):
    """Weights whose exponentials leave fp32's range unless a common factor is taken out."""
    x = np.float32([[-120, -121, -300, -119], [200, 199, 198, -200]])
    for scores in ("softmax", "sigmoid"):
        got = experts_route(x, 2, scores=scores, runtime=runtime)
        want = oracle.experts_route(x, 2, scores=scores)
        np.testing.assert_array_equal(got.experts[0], want[0][0])
        np.testing.assert_allclose(got.weights[0], want[1][0], rtol=2.0**-15)  # 2^-17 of 119
    got = experts_route(x[1:], 2, runtime=runtime)
    np.testing.assert_array_equal(got.experts, [[0, 1]])


@pytest.mark.parametrize("tokens,experts,top_k", [(127, 8, 2), (128, 64, 8), (129, 64, 8), (1000, 16, 4),
                                                  (20000, 128, 8), (65537, 8, 1), (5000, 1024, 32)])
def test_plans_of_many_tokens(runtime, tokens, experts, top_k):
    rng = np.random.default_rng(tokens)
    x = rng.standard_normal((tokens, experts)).astype(np.float32)
    x[:, : experts // 2] += 2  # some experts with many rows, some with few
    got = experts_route(x, top_k, runtime=runtime)
    want = np.argsort(-x, axis=1, kind="stable")[:, :top_k]
    np.testing.assert_array_equal(got.experts, want)
    by = np.argsort(want.reshape(-1), kind="stable")
    np.testing.assert_array_equal(got.order, by)
    np.testing.assert_array_equal(got.places.reshape(-1)[by], np.arange(tokens * top_k))
    np.testing.assert_array_equal(got.offsets, np.searchsorted(want.reshape(-1)[by],
                                                               np.arange(experts + 1)))
    np.testing.assert_allclose(got.weights.sum(1), 1.0, rtol=2.0**-20)


@pytest.mark.parametrize("tokens,experts,top_k,groups,top_groups,best", [
    (6000, 256, 8, 8, 4, 2), (6000, 160, 6, 8, 3, 1), (5000, 60, 6, 4, 3, 1), (5000, 128, 8, 1, 1, 2),
    (3000, 512, 8, 16, 5, 2), (4000, 64, 7, 1, 1, 2), (2000, 256, 12, 8, 4, 2)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("kind", ["fp32", "bf16 values", "bias"])
def test_choices_of_many_tokens(runtime, tokens, experts, top_k, groups, top_groups, best, scores, kind):
    """Enough tokens that some have neighbours, and sums of groups, next to one another."""
    rng = np.random.default_rng(tokens + experts)
    x = (1.5 * rng.standard_normal((tokens, experts))).astype(np.float32)
    if kind == "bf16 values":
        x = from_bf16_bits(to_bf16_bits(x))
    bias = (0.1 * rng.standard_normal(experts)).astype(np.float32) if kind == "bias" else None
    got = experts_route(x, top_k, scores=scores, bias=bias, groups=groups, top_groups=top_groups,
                        group_best=best, runtime=runtime)
    z = x.astype(np.float64)
    if scores == "softmax":
        s = np.exp(z - z.max(1, keepdims=True))
        s /= s.sum(1, keepdims=True)
    else:
        s = 1 / (1 + np.exp(-z))
    c = s if bias is None else s + bias
    per = experts // groups
    if groups > 1:
        sums = np.sort(c.reshape(tokens, groups, per), axis=-1)[..., -best:].sum(-1)
        kept = np.argsort(-sums, axis=1, kind="stable")[:, :top_groups]
        mask = np.zeros((tokens, groups), bool)
        np.put_along_axis(mask, kept, True, axis=1)
        c = np.where(np.repeat(mask, per, axis=1), c, -np.inf)
    want = np.argsort(-c, axis=1, kind="stable")[:, :top_k]
    np.testing.assert_array_equal(got.experts, want)
    w = np.take_along_axis(s, want, 1)
    np.testing.assert_allclose(got.weights, w / w.sum(1, keepdims=True), rtol=2.0**-18)


@pytest.mark.parametrize("experts", [20, 64, 128, 200, 400])
def test_logits_an_ulp_apart(runtime, experts):
    """fp32 logits of few values, each also an ulp up and down: equals, neighbours, and more candidates
    for the last place than are put in order at once."""
    rng = np.random.default_rng(experts)
    base = np.float32(rng.standard_normal(6))
    x = base[rng.integers(0, 6, (800, experts))]
    step = rng.integers(-1, 2, x.shape)
    x = np.where(step > 0, np.nextafter(x, np.float32(9)), np.where(step < 0, np.nextafter(
        x, np.float32(-9)), x)).astype(np.float32)
    for top_k in (1, 5, 8):
        got = experts_route(x, top_k, runtime=runtime)
        np.testing.assert_array_equal(got.experts, np.argsort(-x, axis=1, kind="stable")[:, :top_k])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ld,start", [(64, 0), (67, 1), (72, 8), (65, 3)])
def test_row_strides_and_rows_behind(runtime, dtype, ld, start):
    """Logits inside wider rows; neither the plan's tail nor anything behind the outputs changes."""
    g = torch.Generator(device="cuda").manual_seed(ld)
    wide = torch.randn(50, ld + 8, generator=g, device="cuda").to(dtype)
    x = wide[:, start:start + 60]
    ids = torch.full((50 * 4 + 9,), 77, dtype=torch.int32, device="cuda")
    order, places = ids.clone(), ids.clone()
    weights = torch.full((50 * 4 + 9,), 77.0, device="cuda")
    offsets = torch.full((70,), 77, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([7, 0, 20], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    runtime.experts_route_device(
        x.data_ptr(), ids.data_ptr(), weights.data_ptr(), tokens=50, num_experts=60, top_k=4,
        ld=x.stride(0), logits_dtype=TX_BF16 if dtype == torch.bfloat16 else 0, seq=20,
        lengths=lengths.data_ptr(), offsets=offsets.data_ptr(), order=order.data_ptr(),
        places=places.data_ptr())
    runtime.sync()
    want = oracle.experts_route(x.float().cpu().numpy(), 4, lengths=[7, 0, 20], seq=20)
    np.testing.assert_array_equal(ids[:200].cpu().view(50, 4), want[0])
    np.testing.assert_array_equal(places[:200].cpu().view(50, 4), want[4])
    np.testing.assert_array_equal(offsets[:61].cpu(), want[2])
    used = want[2][-1]
    assert used < 200
    np.testing.assert_array_equal(order[:used].cpu(), want[3][:used])
    for rest in (ids[200:], order[used:], places[200:], weights[200:], offsets[61:]):
        assert (rest == 77).all()


def test_without_a_plan_and_no_tokens(runtime):
    x = torch.randn(300, 16, device="cuda")
    ids = torch.zeros(300, 2, dtype=torch.int32, device="cuda")
    w = torch.zeros(300, 2, device="cuda")
    offsets = torch.full((17,), 5, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    runtime.experts_route_device(x.data_ptr(), ids.data_ptr(), w.data_ptr(), tokens=300,
                                 num_experts=16, top_k=2)
    runtime.experts_route_device(x.data_ptr(), ids.data_ptr(), w.data_ptr(), tokens=0, num_experts=16,
                                 top_k=2, offsets=offsets.data_ptr(), order=ids.data_ptr(),
                                 places=ids.data_ptr())
    runtime.sync()
    np.testing.assert_array_equal(ids.cpu(), x.topk(2).indices.cpu())
    assert not offsets.any()
    empty = experts_route(np.empty((0, 16), np.float32), 2, runtime=runtime)
    assert empty.experts.shape == (0, 2) and not empty.offsets.any() and not empty.order.size


def test_in_a_graph_while_larger_calls_run(runtime):
    """Two launches and their counts in a graph; eager calls between its replays need more scratch."""
    def call(x, k):
        t, e = x.shape
        out = [torch.zeros(t, k, dtype=torch.int32, device="cuda") for _ in range(3)]
        out += [torch.zeros(t, k, device="cuda"),
                torch.zeros(e + 1, dtype=torch.int32, device="cuda")]

        def go(stream):
            runtime.experts_route_device(
                x.data_ptr(), out[0].data_ptr(), out[3].data_ptr(), tokens=t, num_experts=e, top_k=k,
                order=out[1].data_ptr(), places=out[2].data_ptr(), offsets=out[4].data_ptr(),
                stream=stream)
        return go, out

    x, y = torch.randn(1000, 32, device="cuda"), torch.randn(40000, 512, device="cuda")
    (small, out), (large, other) = call(x, 4), call(y, 8)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        small(stream.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            small(torch.cuda.current_stream().cuda_stream)
        large(stream.cuda_stream)
        want = [o.clone() for o in other]
        x.neg_()
        small(stream.cuda_stream)
        first = [o.clone() for o in out]
        for _ in range(3):
            for o in out:
                o.zero_()
            large(stream.cuda_stream)
            graph.replay()
            large(stream.cuda_stream)
        runtime.sync(stream.cuda_stream)
    assert all(torch.equal(a, b) for a, b in zip(out, first, strict=True))
    assert all(torch.equal(a, b) for a, b in zip(other, want, strict=True))
    del graph
    torch.cuda.synchronize()


def test_refusals(runtime):
    b = runtime.buffer(65536)
    p = b.device_ptr
    ok = dict(tokens=8, num_experts=16, top_k=2)
    plan = dict(offsets=p + 4096, order=p + 8192, places=p + 12288)
    runtime.experts_route_device(p, p + 16384, p + 32768, **ok, **plan)
    for kw in (dict(num_experts=0), dict(num_experts=1025), dict(top_k=0), dict(top_k=17),
               dict(groups=3), dict(groups=0), dict(num_experts=128, groups=128), dict(top_groups=2), dict(groups=4, top_groups=5),
               dict(groups=8, top_groups=1, top_k=3), dict(groups=4, top_groups=2, group_best=3),
               dict(scores="other"), dict(scale=np.inf), dict(scale=np.nan), dict(ld=15),
               dict(logits_dtype=2), dict(lengths=p), dict(bias=p + 2), dict(order=None),
               dict(places=None), dict(offsets=None), dict(offsets=p + 4097),
               dict(tokens=2**30, top_k=2)):
        before = runtime.launch_count()
        with pytest.raises(InvalidInputError):
            runtime.experts_route_device(p, p + 16384, p + 32768, **{**ok, **plan, **kw})
        assert runtime.launch_count() == before
    for at in ((0, p, p), (p, 0, p), (p, p, 0), (p + 2, p, p), (p, p + 1, p)):
        with pytest.raises(InvalidInputError):
            runtime.experts_route_device(*at, **ok)
    runtime.sync()
    b.close()
