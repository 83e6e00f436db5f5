"""Routing of tokens to experts on a B200 where its choice or its weights hang on what fp32 does not
hold: groups whose sums cancel, experts closed by their bias, groups far below the largest logit.
Experts have to be equal to those of the formula in 64 bits; weights to 2^-18 of the value, as in
test_experts_route_gpu.py (two logits at most 24 apart: their difference is off by 2^-20)."""

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200.layers import experts_route

pytestmark = pytest.mark.gpu


def scores_of(x, scores):
    x = x.astype(np.float64)
    if scores == "sigmoid":
        return 1 / (1 + np.exp(-x))
    s = np.exp(x - x.max(-1, keepdims=True))
    return s / s.sum(-1, keepdims=True)


def best_of_groups(c, groups):
    """The sum of the best two of each group."""
    return np.sort(c.reshape(groups, -1), axis=1)[:, -2:].sum(1)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [2.0, 40.0, 1000.0])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", [
    (64, 8, 4, 8), (128, 8, 3, 6), (128, 32, 9, 8), (256, 8, 4, 8), (256, 64, 20, 8), (60, 4, 2, 5),
    (256, 8, 4, 12), (1024, 16, 5, 8)])
def test_groups_whose_sums_cancel(runtime, scores, size, experts, groups, top_groups, top_k):
    """The best two of every group lie near `size` and -`size`, and one bias brings the first group
    that is left out next to the last one that stays: their sums are told apart by what the rounding
    of each term to fp32 takes away."""
    rng = np.random.default_rng(experts + groups + top_k)
    per, close = experts // groups, 0
    for _ in range(50):
        x = rng.standard_normal((1, experts)).astype(np.float32)
        s = scores_of(x[0], scores)
        bias = np.full(experts, -3 * size, np.float32)
        pairs = np.array([g * per + rng.permutation(per)[:2] for g in range(groups)])
        bias[pairs[:, 0]] = size * rng.uniform(0.97, 1.03, groups)
        bias[pairs[:, 1]] = -size * rng.uniform(0.97, 1.03, groups)
        sums = best_of_groups(s + bias, groups)
        by = np.argsort(-sums, kind="stable")
        stays, leaves = by[top_groups - 1], by[top_groups]
        bias[pairs[leaves, 1]] += sums[stays] - sums[leaves]
        sums = best_of_groups(s + bias, groups)
        close += abs(sums[stays] - sums[leaves]) <= size * 2.0**-23
        kw = dict(scores=scores, bias=bias, groups=groups, top_groups=top_groups)
        got = experts_route(x, top_k, runtime=runtime, **kw)
        np.testing.assert_array_equal(got.experts, oracle.experts_route(x, top_k, **kw)[0])
    assert close > 40


@pytest.mark.parametrize("experts,groups,top_groups,top_k", [
    (16, 1, 1, 4), (64, 1, 1, 8), (64, 8, 4, 8), (64, 1, 1, 12), (200, 1, 1, 8), (256, 64, 20, 8),
    (640, 1, 1, 4), (1024, 16, 5, 9)])
@pytest.mark.parametrize("renormalise", [False, True])
@pytest.mark.parametrize("kind", ["spread", "neighbours"])
def test_a_bias_takes_part_in_the_choice_alone(runtime, experts, groups, top_groups, top_k, renormalise,
                                               kind):
    """Experts closed by a bias of -inf, the one with the largest logit among them, keep their place
    in the softmax: the scores by which the others are chosen, and their weights, are those of all
    logits."""
    rng = np.random.default_rng(experts + top_k)
    x = (1.5 * rng.standard_normal((40, experts))).astype(np.float32).clip(-12, 11)
    shut = rng.permutation(experts)[:max(1, experts // 8)]
    x[:, shut[0]] = rng.uniform(2, 12, 40)
    bias = (0.01 * rng.standard_normal(experts)).astype(np.float32)
    bias[shut] = -np.inf
    s = scores_of(x, "softmax")
    if kind == "neighbours":  # of the first token: fp32 does not tell two experts apart
        a, b = [e for e in np.argsort(-(s[0] + bias)) if np.isfinite(bias[e])][:2]
        bias[b] = s[0, a] + bias[a] - s[0, b]
    c = s + bias
    per = experts // groups
    want = []
    for row in c:
        top = np.sort(row.reshape(groups, per), axis=1)[:, -2:]
        # A closed expert is in no sum; a group of closed experts alone comes behind all others.
        sums = np.where(top[:, -1] == -np.inf, -np.inf, np.where(np.isinf(top), 0.0, top).sum(1))
        kept = np.argsort(-sums, kind="stable")[:top_groups]
        row = np.where(np.isin(np.arange(experts) // per, kept), row, -np.inf)
        want.append(np.argsort(-row, kind="stable")[:top_k])
    want = np.array(want)
    assert np.isfinite(np.take_along_axis(c, want, 1)).all()
    w = np.take_along_axis(s, want, 1)
    if renormalise:
        w = w / w.sum(1, keepdims=True)
    kw = dict(bias=bias, groups=groups, top_groups=top_groups, renormalise=renormalise, scale=1.5)
    got = experts_route(x, top_k, runtime=runtime, **kw)
    np.testing.assert_array_equal(got.experts, want)
    np.testing.assert_allclose(got.weights, 1.5 * w, rtol=2.0**-18)
    restated = oracle.experts_route(x, top_k, **kw)
    np.testing.assert_array_equal(restated[0], want)
    np.testing.assert_allclose(restated[1], 1.5 * w, rtol=1e-12)


@pytest.mark.parametrize("experts,groups", [(32, 4), (60, 5), (256, 64), (640, 4), (1024, 8)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_groups_far_below_the_largest_logit(runtime, experts, groups, scores):
    """Scores down to e^-740, of which 64 bits hold a few bits yet, tell groups apart."""
    per = experts // groups
    rng = np.random.default_rng(experts)
    for level in (-600, -690, -710, -720, -738):
        x = (level - 60 + rng.uniform(0, 1, (6, experts))).astype(np.float32)  # in no group's best
        stays = rng.integers(groups // 2, groups, 6)
        for t, g in enumerate(stays):
            for group in range(groups):
                best = level + 2 * (group == g) if group else level + 4 if scores == "sigmoid" else 0
                x[t, group * per:group * per + 2] = best
        got = experts_route(x, 4, scores=scores, groups=groups, top_groups=2, renormalise=False,
                            runtime=runtime)
        want = [[0, 1, g * per, g * per + 1] for g in stays]
        np.testing.assert_array_equal(got.experts, want)
