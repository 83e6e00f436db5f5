"""A transformer layer of experts over texts and images, built from the library's operators: positions
with a time, a row and a column (rotary_axes_device), attention over packed sequences
(attention_scored_device), norms on both sides of each block with a gate by sequence
(block_norm_device), and a feed-forward part of which each token takes a few experts
(experts_route_device, experts_linear_device twice, and block_norm_device to join their rows).

The residual stream stays on the device in fp32; everything between is bf16.

    python examples/experts_layer.py        # on a machine with a B200
"""

from __future__ import annotations

import sys
from dataclasses import dataclass
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from tessery_b200 import TX_BF16, TX_F32, CudaRuntime, rotary_frequencies, rotary_pair_axes  # noqa: E402
from tessery_b200.workloads import to_bf16_bits  # noqa: E402


@dataclass(frozen=True)
class LayerConfig:
    hidden: int = 1024
    heads: int = 16
    kv_heads: int = 8
    head_dim: int = 64
    sections: tuple[int, ...] = (8, 12, 12)  # rotated pairs by time, row and column
    theta: float = 1e4
    experts: int = 64
    top_k: int = 8
    expert_width: int = 512
    groups: int = 8
    top_groups: int = 4
    scale: float = 2.5  # of the experts' weights
    eps: float = 1e-6


def random_weights(cfg: LayerConfig, seed: int = 0) -> dict[str, np.ndarray]:
    """float32 weights of one layer; all but the router's bias are bf16 values."""
    rng = np.random.default_rng(seed)
    qd, kd = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim

    def matrix(*shape: int) -> np.ndarray:
        return rng.standard_normal(shape).astype(np.float32) * shape[-1] ** -0.5

    def norm(n: int) -> np.ndarray:
        return 1.0 + 0.1 * rng.standard_normal(n).astype(np.float32)

    return {
        "norm": norm(cfg.hidden), "attn_norm": norm(cfg.hidden), "mlp_norm": norm(cfg.hidden),
        "experts_norm": norm(cfg.hidden), "q_norm": norm(cfg.head_dim), "k_norm": norm(cfg.head_dim),
        "qkv": matrix(qd + 2 * kd, cfg.hidden), "o": matrix(cfg.hidden, qd),
        "router": 2.0 * matrix(cfg.experts, cfg.hidden),
        "up": matrix(cfg.experts, 2 * cfg.expert_width, cfg.hidden),
        "down": matrix(cfg.experts, cfg.hidden, cfg.expert_width),
        "router_bias": 0.05 * rng.standard_normal(cfg.experts).astype(np.float32),
    }


class Layer:
    """One layer on `rt`."""

    def __init__(self, rt: CudaRuntime, cfg: LayerConfig, weights: dict[str, np.ndarray]) -> None:
        self.rt, self.cfg = rt, cfg
        self._w = {}
        freq = rotary_frequencies(2 * sum(cfg.sections), cfg.theta)[0]
        tables = {"freq": freq, "pair_axes": rotary_pair_axes(cfg.sections, cycle=True)}
        for name, w in {**weights, **tables}.items():
            data = w if name in ("router_bias", *tables) else to_bf16_bits(w)
            self._w[name] = rt.buffer(data.nbytes, np.ascontiguousarray(data))

    def run(self, x: int, tokens: int, cu_seqlens: int, nseq: int, max_len: int, positions: int,
            gate: int, *, experts: int, weights: int, stream: int | None = None) -> None:
        """Updates the fp32 rows [tokens, hidden] at `x` in place.  Device addresses throughout:
        cu_seqlens int32 [nseq + 1], positions int32 [axes, tokens], gate fp32 [nseq, hidden] of the
        attention's part.  The chosen experts (int32) and their weights (fp32) [tokens, top_k] are
        left at `experts` and `weights`."""
        rt, cfg, w = self.rt, self.cfg, {k: b.device_ptr for k, b in self._w.items()}
        qd, kd, pairs = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim, tokens * cfg.top_k
        room = {name: rt.workspace("experts_layer_" + name, size).device_ptr for name, size in (
            ("h", tokens * cfg.hidden * 2), ("qkv", tokens * (qd + 2 * kd) * 2),
            ("a", tokens * qd * 2), ("y", tokens * cfg.hidden * 2), ("logits", tokens * cfg.experts * 4),
            ("offsets", 4 * (cfg.experts + 1)), ("order", 4 * pairs), ("places", 4 * pairs),
            ("up", pairs * cfg.expert_width * 2), ("down", pairs * cfg.hidden * 2))}
        h, qkv = room["h"], room["qkv"]
        rows = {"rows": tokens, "cols": cfg.hidden, "stream": stream}

        def norm(name: str) -> dict:
            return {"kind": "rms", "weight": w[name], "dtype": TX_BF16, "eps": cfg.eps}

        rt.block_norm_device(x, None, h=h, before=norm("norm"), **rows)
        rt.linear_fused_device(h, w["qkv"], qkv, m=tokens, n=qd + 2 * kd, k=cfg.hidden, stream=stream)
        inner = (qd + 2 * kd, cfg.head_dim)  # (row, head) strides inside the product's rows
        rt.rotary_axes_device(
            qkv, qkv + 2 * qd, qkv, qkv + 2 * qd, tokens=tokens, heads=cfg.heads,
            kv_heads=cfg.kv_heads, dim=cfg.head_dim, inv_freq=w["freq"],
            rot_dim=2 * sum(cfg.sections), pair_axes=w["pair_axes"], positions=positions,
            axes=len(cfg.sections), q_norm_weight=w["q_norm"], k_norm_weight=w["k_norm"], eps=cfg.eps,
            q_strides=inner, k_strides=inner, q_out_strides=inner, k_out_strides=inner, stream=stream)
        rt.attention_scored_device(
            qkv, qkv + 2 * qd, qkv + 2 * (qd + kd), room["a"], nseq=nseq, rows_q=tokens, rows_k=tokens,
            max_q=max_len, max_k=max_len, heads=cfg.heads, kv_heads=cfg.kv_heads, dim=cfg.head_dim,
            cu_q=cu_seqlens, cu_k=cu_seqlens, causal=False, q_strides=inner, k_strides=inner,
            v_strides=inner, stream=stream)
        rt.linear_fused_device(room["a"], w["o"], room["y"], m=tokens, n=cfg.hidden, k=qd, stream=stream)
        rt.block_norm_device(x, room["y"], out=x, h=h, after=norm("attn_norm"),
                             before=norm("mlp_norm"), gate=gate, gate_rows=nseq,
                             cu_seqlens=cu_seqlens, **rows)
        rt.linear_fused_device(h, w["router"], room["logits"], m=tokens, n=cfg.experts, k=cfg.hidden,
                               out_dtype=TX_F32, stream=stream)
        rt.experts_route_device(
            room["logits"], experts, weights, tokens=tokens, num_experts=cfg.experts, top_k=cfg.top_k,
            bias=w["router_bias"], scores="sigmoid", groups=cfg.groups, top_groups=cfg.top_groups,
            scale=cfg.scale, offsets=room["offsets"], order=room["order"], places=room["places"],
            stream=stream)
        plan = {"offsets": room["offsets"], "tokens": tokens, "top_k": cfg.top_k,
                "num_experts": cfg.experts, "stream": stream}
        rt.experts_linear_device(h, w["up"], room["up"], order=room["order"], n=cfg.expert_width,
                                 k=cfg.hidden, gated=True, activation="silu", **plan)
        rt.experts_linear_device(room["up"], w["down"], room["down"], n=cfg.hidden,
                                 k=cfg.expert_width, **plan)
        rt.block_norm_device(x, room["down"], out=x, after=norm("experts_norm"),
                             places=room["places"], weights=weights, top_k=cfg.top_k, y_rows=pairs,
                             **rows)

    def close(self) -> None:
        for b in self._w.values():
            b.close()


def text_positions(start: int, count: int) -> np.ndarray:
    """[3, count]: text stands at one position on all axes."""
    return np.tile(np.arange(start, start + count), (3, 1))


def image_positions(start: int, height: int, width: int) -> np.ndarray:
    """[3, height * width]: one moment, rows and columns from `start` on."""
    row, col = np.divmod(np.arange(height * width), width)
    return np.stack([np.full(height * width, start), start + row, start + col])


def main() -> None:
    cfg = LayerConfig()
    rng = np.random.default_rng(1)
    # Two texts, the second around an image of 24 x 16 patches.
    pos = np.concatenate([text_positions(0, 700), text_positions(0, 40), image_positions(40, 24, 16),
                          text_positions(64, 300)], axis=1).astype(np.int32)
    cu = np.array([0, 700, pos.shape[1]], np.int32)
    tokens = pos.shape[1]
    x = rng.standard_normal((tokens, cfg.hidden)).astype(np.float32)
    gate = np.ones((2, cfg.hidden), np.float32)
    with CudaRuntime() as rt:
        layer = Layer(rt, cfg, random_weights(cfg))
        buffers = [rt.buffer(a.nbytes, np.ascontiguousarray(a)) for a in (x, cu, pos, gate)]
        chosen, weights = (rt.buffer(4 * tokens * cfg.top_k) for _ in range(2))
        at = [b.device_ptr for b in buffers]
        layer.run(at[0], tokens, at[1], 2, int(np.diff(cu).max()), at[2], at[3],
                  experts=chosen.device_ptr, weights=weights.device_ptr)
        rt.sync()
        y = rt.read(buffers[0], x.shape)
        ids = rt.read(chosen, (tokens, cfg.top_k), np.int32)
        print(f"{tokens} tokens, rows of rms {np.sqrt(np.mean(y * y)):.3f}; tokens of an expert: "
              f"{np.bincount(ids.ravel(), minlength=cfg.experts)}")
        layer.close()
        for b in (*buffers, chosen, weights):
            b.close()


if __name__ == "__main__":
    main()
