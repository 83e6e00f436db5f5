"""The example layer of experts (examples/experts_layer.py): positions on several axes, packed
attention, norms on both sides with a gate, routing, the experts' products and their join, run
together.

Tolerance.  A rounding to bf16 is off by 2^-9 / sqrt(3) = r = 2^-9.8 of its values in the mean square;
errors are counted below in squares of r, each product or norm carrying its operand's on.
Attention's part: q and k have 3 each (the norm's row, the product, the rotated head), so the scores, of
variance about 1, have 6, and as much comes to the weighted sum; v has 2, the weights and the sum's own
rounding 1 each, the output product 1: 11 of that part.  x then carries 11 / 2 (two parts as large as
each other), the next norm's row 6.5.  The experts: silu(g) u takes that through u once and through g
1.3 times as steeply (2.7 x 6.5), its rounding and the second product's add 2, the weights, from logits of
about 2 at half the sigmoid's relative slope, 6.5: 26 of this part.  Both parts are as large as each
other, so a row's error is sqrt((11 + 26) / 2) r = 4.3 r = 2^-7.7 of what it gains, over the rows; single
rows, whose experts' rows may half cancel before the norm takes them up again, up to three times that.  The
gate is 2^-6.
The experts are the library's own choice; that it is the right one is tested by the logits in 64 bits.
Those are off by sqrt(6.5) r of about 2, four times that at most among all of them: 2^-5.5, a quarter of it
through the sigmoid, and 2^-8 of a row's largest logit (5 or more) is allowed to each side.
"""

import importlib.util
import sys
import threading
from pathlib import Path

import numpy as np
import pytest

import tessery_b200 as tx
from oracle import layers as oracle
from tessery_b200 import rotary_frequencies, rotary_pair_axes
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

_spec = importlib.util.spec_from_file_location(
    "experts_layer", Path(__file__).resolve().parents[1] / "examples" / "experts_layer.py")
example = importlib.util.module_from_spec(_spec)
sys.modules[_spec.name] = example
_spec.loader.exec_module(example)


def exact(cfg, weights, x, cu, pos, gate, chosen):
    """(rows, the router's logits) in 64 bits, for the experts given."""
    w = {k: (v if k == "router_bias" else from_bf16_bits(to_bf16_bits(v))).astype(np.float64)
         for k, v in weights.items()}
    tokens, qd, kd = len(x), cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim

    def norm(name):
        return dict(kind="rms", weight=w[name], eps=cfg.eps)

    h = oracle.norm(x.astype(np.float64), **norm("norm"))
    qkv = h @ w["qkv"].T
    freq = rotary_frequencies(2 * sum(cfg.sections), cfg.theta)[0]
    axes = rotary_pair_axes(cfg.sections, cycle=True)
    q = oracle.rotary_axes(qkv[:, :qd].reshape(tokens, cfg.heads, -1), pos, axes, freq,
                           weight=w["q_norm"], eps=cfg.eps)
    k = oracle.rotary_axes(qkv[:, qd:qd + kd].reshape(tokens, cfg.kv_heads, -1), pos, axes, freq,
                           weight=w["k_norm"], eps=cfg.eps)
    v = qkv[:, qd + kd:].reshape(tokens, cfg.kv_heads, -1)
    a = np.concatenate([oracle.attention_scored(q[s:t], k[s:t], v[s:t])[0]
                        for s, t in zip(cu[:-1], cu[1:], strict=True)]).reshape(tokens, qd)
    of = np.repeat(np.arange(len(cu) - 1), np.diff(cu))
    x1, h = oracle.block_norm(x, a @ w["o"].T, after=norm("attn_norm"), before=norm("mlp_norm"),
                              gate=gate, gate_row=of)
    logits = h @ w["router"].T
    z = np.zeros_like(x1)
    for t in range(tokens):
        s = 1 / (1 + np.exp(-logits[t, chosen[t]]))
        for e, share in zip(chosen[t], cfg.scale * s / s.sum(), strict=True):
            y = w["up"][e] @ h[t]
            n = cfg.expert_width
            z[t] += share * (w["down"][e] @ (oracle.activate(y[:n], "silu") * y[n:]))
    return oracle.block_norm(x1, z, after=norm("experts_norm"))[0], logits


@pytest.mark.parametrize("heads,kv_heads,dim,sections,experts,top_k,groups,top_groups", [
    (4, 2, 32, (4, 6, 6), 8, 2, 1, 1), (3, 1, 40, (3, 5, 4), 24, 5, 4, 2), (2, 2, 64, (8, 12, 12), 64, 8, 8, 4)])
def test_layer(runtime, heads, kv_heads, dim, sections, experts, top_k, groups, top_groups):
    cfg = example.LayerConfig(hidden=96, heads=heads, kv_heads=kv_heads, head_dim=dim,
                              sections=sections, experts=experts, top_k=top_k, expert_width=72,
                              groups=groups, top_groups=top_groups)
    weights = example.random_weights(cfg, seed=dim)
    rng = np.random.default_rng(dim)
    pos = np.concatenate([example.text_positions(0, 90), example.text_positions(0, 5),
                          example.image_positions(5, 6, 9), example.text_positions(11, 30),
                          example.text_positions(0, 1)], axis=1).astype(np.int32)
    cu = np.array([0, 90, 90, 179, 180], np.int32)  # an empty sequence and one of a token among them
    tokens = pos.shape[1]
    assert tokens == cu[-1]
    x = rng.standard_normal((tokens, cfg.hidden)).astype(np.float32)
    gate = rng.random((4, cfg.hidden)).astype(np.float32) + 0.5
    layer = example.Layer(runtime, cfg, weights)
    dev = [torch.from_numpy(a).cuda() for a in (x, cu, pos, gate)]
    chosen = torch.full((tokens, top_k), -7, dtype=torch.int32, device="cuda")
    share = torch.zeros(tokens, top_k, device="cuda")
    torch.cuda.synchronize()

    def run(stream):
        layer.run(dev[0].data_ptr(), tokens, dev[1].data_ptr(), 4, 90, dev[2].data_ptr(),
                  dev[3].data_ptr(), experts=chosen.data_ptr(), weights=share.data_ptr(), stream=stream)

    run(None)
    runtime.sync()
    got, ids = dev[0].cpu().numpy(), chosen.cpu().numpy()
    want, logits = exact(cfg, weights, x, cu, pos, gate, ids)
    gained = np.linalg.norm(want - x, axis=-1)
    assert np.max(np.linalg.norm(got - want, axis=-1) / gained) < 2.0**-6

    # The choice, with every logit allowed its error.
    c = 1 / (1 + np.exp(-logits)) + weights["router_bias"]
    slack = 2.0**-8 * np.abs(logits).max(axis=-1)  # a sigmoid is a quarter as steep at most
    per = experts // groups
    for t in range(tokens):
        assert len(set(ids[t])) == top_k
        used = set(ids[t] // per)
        assert len(used) <= top_groups
        best = np.sort(c[t].reshape(groups, per), axis=-1)[:, -2:].sum(axis=-1)
        inside = [e for e in range(experts) if e // per in used and e not in ids[t]]
        assert all(c[t, e] <= c[t, ids[t]].min() + slack[t] for e in inside)
        shut = [g for g in range(groups) if np.sum(best > best[g] + slack[t]) >= top_groups]
        assert not used & set(shut)

    # The same on another stream and in a graph, bit by bit.
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        dev[0].copy_(torch.from_numpy(x))
        run(stream.cuda_stream)
        runtime.sync(stream.cuda_stream)
        assert np.array_equal(dev[0].cpu().numpy(), got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run(torch.cuda.current_stream().cuda_stream)
        dev[0].copy_(torch.from_numpy(x))
        chosen.zero_()
        graph.replay()
        runtime.sync(stream.cuda_stream)
    assert np.array_equal(dev[0].cpu().numpy(), got) and np.array_equal(chosen.cpu().numpy(), ids)
    del graph
    layer.close()


def test_threads_on_one_runtime(runtime):
    """The operators on arrays from three threads: each call's result is the one it has alone."""
    rng = np.random.default_rng(1)
    cases = []
    for n in (40, 300, 1100):
        logits = rng.standard_normal((n, 16)).astype(np.float32)
        x = to_bf16_bits(rng.standard_normal((n, 64)).astype(np.float32))
        w = to_bf16_bits(rng.standard_normal((16, 96, 64)).astype(np.float32))
        r = tx.experts_route(logits, 2, runtime=runtime)
        cases.append((
            lambda v=logits: np.concatenate([a.ravel() for a in tx.experts_route(v, 2, runtime=runtime)]),
            lambda x=x, w=w, r=r: tx.experts_linear(x, w, r.offsets, order=r.order, top_k=2,
                                                    runtime=runtime),
            lambda x=x: tx.block_norm(x, x, before=dict(kind="layer"), runtime=runtime)[1]))
    want = [[call() for call in case] for case in cases]
    wrong = []

    def work(i):
        try:
            for _ in range(15):
                for call, w in zip(cases[i], want[i], strict=True):
                    if not np.array_equal(call(), w):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001 - reported below
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_arrays_one_after_another(runtime):
    """The operators on arrays as a caller puts them together, against 64 bits."""
    rng = np.random.default_rng(9)
    tokens, hidden, experts, width, top_k = 70, 64, 16, 40, 4

    def f(*shape):
        return rng.standard_normal(shape).astype(np.float32)

    def b(*shape):
        return from_bf16_bits(to_bf16_bits(f(*shape) * shape[-1] ** -0.5))

    x, o, gate, logits = f(tokens, hidden), f(tokens, hidden), f(3, hidden), f(tokens, experts)
    up, down = b(experts, 2 * width, hidden), b(experts, hidden, width)
    w1, w2, w3 = f(3, hidden)
    balance, cu = 0.1 * f(experts), np.array([0, 30, 30, 70], np.int32)
    bits = to_bf16_bits
    x1, h = tx.block_norm(x, o, after={"kind": "rms", "weight": w1}, before={"kind": "rms", "weight": w2},
                          gate=gate, cu_seqlens=cu, runtime=runtime)
    r = tx.experts_route(logits, top_k, bias=balance, scores="sigmoid", groups=4, top_groups=2, scale=2.5,
                         runtime=runtime)
    u = tx.experts_linear(h, bits(up), r.offsets, order=r.order, top_k=top_k, gated=True, activation="silu",
                          runtime=runtime)
    d = tx.experts_linear(u, bits(down), r.offsets, runtime=runtime)
    x2, h2 = tx.block_norm(x1, d, places=r.places, weights=r.weights,
                           before={"kind": "rms", "weight": w3}, runtime=runtime)

    of = np.repeat([0, 2], [30, 40])
    e1, eh = oracle.block_norm(x, o, after=dict(kind="rms", weight=w1), before=dict(kind="rms", weight=w2),
                               gate=gate, gate_row=of)
    want = oracle.experts_route(logits, top_k, bias=balance, scores="sigmoid", groups=4, top_groups=2,
                                scale=2.5)
    np.testing.assert_array_equal(r.experts, want[0])
    eu, _ = oracle.experts_linear(eh, up, want[2], order=want[3], top_k=top_k, gated=True,
                                  activation="silu")
    ed, _ = oracle.experts_linear(eu, down, want[2])
    z = np.einsum("tj,tjc->tc", want[1], ed[want[4]])
    e2 = e1 + z
    # fp32: the norm's factor 2^-22, three products and the sum 2^-24 each, of parts up to three times the sum.
    def size(v):
        return np.linalg.norm(v, axis=-1)

    assert np.max(size(x1 - e1) / size(e1)) < 2.0**-18
    # In squares of r (above): h 1, silu(g) u takes that through u once and through g 1.3 times as steeply,
    # 2.7; u's and d's own roundings 2: 4.7, 2^-8.7 of the joined rows' size, single ones up to four times that.
    parts = (want[1][:, :, None] * ed[want[4]]).reshape(tokens, -1)
    assert np.max(size(x2 - e2) / size(parts)) < 2.0**-6.5
    e3 = oracle.norm(x2.astype(np.float64), kind="rms", weight=w3)
    assert np.all(np.abs(from_bf16_bits(h2) - e3) <= (2.0**-8 + 2.0**-18) * np.abs(e3))
