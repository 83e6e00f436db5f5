"""A transformer layer built from the library's operators: the per-head norms and the rotation
with long-context frequencies (rotary_device), attention under a score rule (a capped score, a
window, an open prefix; attention_scored_device) and the linear layers with bias, activation and
residual in their epilogues (linear_fused_device).

A layer reads a padded batch of texts (`read`), keeps their keys and values, and then takes one
new token of every text at a time against what it kept (`step`).  The residual stream stays on
the device in fp32; everything between is bf16.

    python examples/encoder_layer.py        # on a machine with a B200
"""

from __future__ import annotations

import sys
from dataclasses import dataclass
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from tessery_b200 import TX_F32, CudaRuntime, rotary_frequencies  # noqa: E402
from tessery_b200.workloads import to_bf16_bits  # noqa: E402


@dataclass(frozen=True)
class LayerConfig:
    hidden: int = 1024
    intermediate: int = 4096
    heads: int = 16
    kv_heads: int = 8
    head_dim: int = 64
    theta: float = 1e4
    factor: float = 4.0  # positions up to factor x original
    original: int = 2048
    softcap: float = 30.0
    left: int = 1023  # keys before a token that it sees, beside the prefix
    eps: float = 1e-6


def random_weights(cfg: LayerConfig, seed: int = 0) -> dict[str, np.ndarray]:
    """float32 weights of one layer, each already a bf16 value except the biases."""
    rng = np.random.default_rng(seed)
    qd, kd = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim

    def matrix(n: int, k: int) -> np.ndarray:
        return rng.standard_normal((n, k)).astype(np.float32) * k**-0.5

    def norm(n: int) -> np.ndarray:
        return 1.0 + 0.1 * rng.standard_normal(n).astype(np.float32)

    return {
        "norm": norm(cfg.hidden), "mlp_norm": norm(cfg.hidden),
        "q_norm": norm(cfg.head_dim), "k_norm": norm(cfg.head_dim),
        "qk": matrix(qd + kd, cfg.hidden), "v": matrix(kd, cfg.hidden),
        "o": matrix(cfg.hidden, qd), "up": matrix(cfg.intermediate, cfg.hidden),
        "down": matrix(cfg.hidden, cfg.intermediate),
        "qk_bias": 0.1 * rng.standard_normal(qd + kd).astype(np.float32),
        "up_bias": 0.1 * rng.standard_normal(cfg.intermediate).astype(np.float32),
    }


class Layer:
    """One layer and the keys and values it keeps: `batch` texts of up to `capacity` tokens."""

    def __init__(self, rt: CudaRuntime, cfg: LayerConfig, weights: dict[str, np.ndarray],
                 batch: int, capacity: int) -> None:
        self.rt, self.cfg, self.batch, self.capacity = rt, cfg, batch, capacity
        self._w = {}
        for name, w in weights.items():
            data = w if name.endswith("bias") else to_bf16_bits(w)
            self._w[name] = rt.buffer(data.nbytes, np.ascontiguousarray(data))
        freq, self.amplitude = rotary_frequencies(
            cfg.head_dim, cfg.theta, scaling="yarn", factor=cfg.factor, original=cfg.original)
        self._w["freq"] = rt.buffer(freq.nbytes, freq)
        self.kv_row = cfg.kv_heads * cfg.head_dim  # elements of a token's keys, or values
        kept = batch * capacity * self.kv_row * 2
        self.k, self.v = rt.buffer(kept), rt.buffer(kept)
        self._lengths, self._prefix, self._positions = (rt.buffer(4 * batch) for _ in range(3))

    def _run(self, x: int, rows: int, k_out: int, v_out: int, kv_stride: int, prefix,
             where: dict, layout: dict) -> None:
        """The layer over `rows` rows of the fp32 residual stream at `x`, updated in place.  New
        keys and values go to k_out and v_out, rows kv_stride elements apart."""
        rt, cfg, w = self.rt, self.cfg, {k: b.device_ptr for k, b in self._w.items()}
        qd, kd, hidden = cfg.heads * cfg.head_dim, self.kv_row, cfg.hidden
        h, qk, q, a, up = (rt.workspace("layer_" + name, rows * width * 2).device_ptr
                           for name, width in (("h", hidden), ("qk", qd + kd), ("q", qd),
                                               ("a", qd), ("up", cfg.intermediate)))
        rt.rms_norm_rows_device(x, w["norm"], h, rows=rows, cols=hidden, eps=cfg.eps)
        rt.linear_fused_device(h, w["qk"], qk, m=rows, n=qd + kd, k=hidden, bias=w["qk_bias"])
        rt.linear_fused_device(h, w["v"], v_out, m=rows, n=kd, k=hidden, ldo=kv_stride)
        inner = (qd + kd, cfg.head_dim)  # (row, head) strides inside the product's rows
        rt.rotary_device(qk, qk + 2 * qd, q, k_out, tokens=rows, heads=cfg.heads,
                         kv_heads=cfg.kv_heads, dim=cfg.head_dim, inv_freq=w["freq"],
                         amplitude=self.amplitude, q_norm_weight=w["q_norm"],
                         k_norm_weight=w["k_norm"], eps=cfg.eps, q_strides=inner,
                         k_strides=inner, k_out_strides=(kv_stride, cfg.head_dim), **where)
        if prefix is not None:
            self._prefix.write(np.asarray(prefix, np.int32))
        rt.attention_scored_device(
            q, self.k.device_ptr, self.v.device_ptr, a, nseq=self.batch, heads=cfg.heads,
            kv_heads=cfg.kv_heads, dim=cfg.head_dim, rows_q=rows,
            rows_k=self.batch * self.capacity, max_k=self.capacity,
            k_lengths=self._lengths.device_ptr, softcap=cfg.softcap, window=(cfg.left, -1),
            prefix=None if prefix is None else self._prefix.device_ptr, **layout)
        rt.linear_fused_device(a, w["o"], x, m=rows, n=hidden, k=qd, residual=x, out_dtype=TX_F32)
        rt.rms_norm_rows_device(x, w["mlp_norm"], h, rows=rows, cols=hidden, eps=cfg.eps)
        rt.linear_fused_device(h, w["up"], up, m=rows, n=cfg.intermediate, k=hidden,
                               bias=w["up_bias"], activation="gelu_tanh")
        rt.linear_fused_device(up, w["down"], x, m=rows, n=hidden, k=cfg.intermediate, residual=x,
                               out_dtype=TX_F32)

    def read(self, x: int, lengths, prefix=None) -> None:
        """Takes the texts: x is the device address of fp32 [batch, capacity, hidden], of which
        the first lengths[b] rows of text b are tokens.  The first prefix[b] tokens are open to
        all of text b."""
        self._lengths.write(np.asarray(lengths, np.int32))
        self._run(x, self.batch * self.capacity, self.k.device_ptr, self.v.device_ptr, self.kv_row,
                  prefix, {"seq": self.capacity},
                  {"max_q": self.capacity, "q_lengths": self._lengths.device_ptr})

    def step(self, x: int, position: int, prefix=None) -> None:
        """Takes one new token of every text, at `position` of each (the number of tokens before
        it): x is the device address of fp32 [batch, hidden]."""
        if not 0 <= position < self.capacity:
            raise ValueError("position")
        self._lengths.write(np.full(self.batch, position + 1, np.int32))
        self._positions.write(np.full(self.batch, position, np.int32))
        at = 2 * position * self.kv_row
        self._run(x, self.batch, self.k.device_ptr + at, self.v.device_ptr + at,
                  self.capacity * self.kv_row, prefix, {"positions": self._positions.device_ptr},
                  {"max_q": 1})

    def close(self) -> None:
        for b in (*self._w.values(), self.k, self.v, self._lengths, self._prefix, self._positions):
            b.close()


def main() -> None:
    cfg, batch, tokens, new = LayerConfig(), 4, 600, 3
    rng = np.random.default_rng(1)
    x = rng.standard_normal((batch, tokens + new, cfg.hidden)).astype(np.float32)
    prefix = [16] * batch
    with CudaRuntime() as rt:
        weights = random_weights(cfg)
        whole = Layer(rt, cfg, weights, batch, tokens + new)
        buf = rt.buffer(x.nbytes, x)
        whole.read(buf.device_ptr, [tokens + new] * batch, prefix)
        rt.sync()
        want = rt.read(buf, x.shape)

        parts = Layer(rt, cfg, weights, batch, tokens + new)
        buf.write(x)
        parts.read(buf.device_ptr, [tokens] * batch, prefix)
        for i in range(tokens, tokens + new):
            row = rt.buffer(batch * cfg.hidden * 4, np.ascontiguousarray(x[:, i]))
            parts.step(row.device_ptr, i, prefix)
            rt.sync()
            got = rt.read(row, (batch, cfg.hidden))
            diff = np.linalg.norm(got - want[:, i]) / np.linalg.norm(want[:, i])
            print(f"token {i}: one at a time against the whole text, relative difference {diff:.1e}")
            row.close()
        for layer in (whole, parts):
            layer.close()
        buf.close()


if __name__ == "__main__":
    main()
