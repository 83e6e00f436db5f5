"""The example layer (examples/encoder_layer.py): the rotation, attention under a score rule and
the linear layers run together, a text read at once and token by token.

Tolerance.  The layer rounds to bf16 at eight places between its fp32 residual rows.  A rounding
is off by 2^-9 of its value at most and by 2^-9 / sqrt(3) = 2^-9.8 in the mean square; eight of
them, each carried on by products that keep relative sizes, make sqrt(8) 2^-9.8 = 2^-8.3 of the
part that a row gains from the layer, measured over a row.  The gate is 2^-7 of that part: the
library against 64 bits with no rounding between, or one way through the library against the
other."""

import importlib.util
import sys
from pathlib import Path

import numpy as np
import pytest

from oracle import layers as oracle
from tessery_b200 import rotary_frequencies
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu

_spec = importlib.util.spec_from_file_location(
    "encoder_layer", Path(__file__).resolve().parents[1] / "examples" / "encoder_layer.py")
example = importlib.util.module_from_spec(_spec)
sys.modules[_spec.name] = example
_spec.loader.exec_module(example)


def exact(cfg, weights, x, prefix):
    """One text's rows [tokens, hidden] through the layer in 64 bits."""
    w = {k: (v if k.endswith("bias") else from_bf16_bits(to_bf16_bits(v))).astype(np.float64)
         for k, v in weights.items()}
    qd, tokens = cfg.heads * cfg.head_dim, len(x)

    def norm(y, g):
        return y / np.sqrt(np.mean(y * y, axis=-1, keepdims=True) + cfg.eps) * g

    h = norm(x.astype(np.float64), w["norm"])
    qk = oracle.linear_fused(h, w["qk"], bias=w["qk_bias"])
    v = oracle.linear_fused(h, w["v"]).reshape(tokens, cfg.kv_heads, cfg.head_dim)
    freq, amplitude = rotary_frequencies(cfg.head_dim, cfg.theta, scaling="yarn",
                                         factor=cfg.factor, original=cfg.original)
    pos = np.arange(tokens)
    q = oracle.rotary(qk[:, :qd].reshape(tokens, cfg.heads, cfg.head_dim), pos, freq,
                      amplitude=amplitude, weight=w["q_norm"], eps=cfg.eps)
    k = oracle.rotary(qk[:, qd:].reshape(tokens, cfg.kv_heads, cfg.head_dim), pos, freq,
                      amplitude=amplitude, weight=w["k_norm"], eps=cfg.eps)
    a = oracle.attention_scored(q, k, v, softcap=cfg.softcap, causal=True, window=(cfg.left, -1),
                                prefix=prefix)[0].reshape(tokens, qd)
    x = oracle.linear_fused(a, w["o"], residual=x.astype(np.float64))
    up = oracle.linear_fused(norm(x, w["mlp_norm"]), w["up"], bias=w["up_bias"],
                             activation="gelu_tanh")
    return oracle.linear_fused(up, w["down"], residual=x)


def apart(got, want, x):
    """The largest difference of a row, relative to what the row gained from the layer."""
    return np.max(np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want - x, axis=-1))


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 32), (6, 1, 40), (2, 2, 128)])
def test_layer(runtime, heads, kv_heads, dim):
    cfg = example.LayerConfig(hidden=96, intermediate=200, heads=heads, kv_heads=kv_heads,
                              head_dim=dim, left=60)
    weights = example.random_weights(cfg, seed=dim)
    rng = np.random.default_rng(dim)
    capacity, lengths, prefix = 190, np.array([190, 1, 77], np.int32), [9, 0, 70]
    x = rng.standard_normal((3, capacity, cfg.hidden)).astype(np.float32)
    layer = example.Layer(runtime, cfg, weights, 3, capacity)
    buf = runtime.buffer(x.nbytes, x)
    layer.read(buf.device_ptr, lengths, prefix)
    runtime.sync()
    got = runtime.read(buf, x.shape)
    for b, n in enumerate(lengths):
        assert apart(got[b, :n], exact(cfg, weights, x[b, :n], prefix[b]), x[b, :n]) < 2.0**-7
    layer.close()
    buf.close()


def test_layer_token_by_token(runtime):
    cfg = example.LayerConfig(hidden=64, intermediate=136, heads=4, kv_heads=2, head_dim=64, left=50)
    weights = example.random_weights(cfg)
    rng = np.random.default_rng(5)
    batch, tokens, new = 3, 130, 4
    x = rng.standard_normal((batch, tokens + new, cfg.hidden)).astype(np.float32)
    layer = example.Layer(runtime, cfg, weights, batch, tokens + new)
    buf = runtime.buffer(x.nbytes, x)
    layer.read(buf.device_ptr, [tokens + new] * batch, [3] * batch)
    runtime.sync()
    whole = runtime.read(buf, x.shape)
    buf.write(x)
    layer.read(buf.device_ptr, [tokens] * batch, [3] * batch)
    for i in range(tokens, tokens + new):
        row = runtime.buffer(batch * cfg.hidden * 4, np.ascontiguousarray(x[:, i]))
        layer.step(row.device_ptr, i, [3] * batch)
        runtime.sync()
        got = runtime.read(row, (batch, cfg.hidden))
        assert apart(got, whole[:, i], x[:, i]) < 2.0**-7
        row.close()
    with pytest.raises(ValueError):
        layer.step(buf.device_ptr, tokens + new)
    layer.close()
    buf.close()
