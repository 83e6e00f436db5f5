"""Measured cases of the operators for encoder layers of experts: the routing of tokens to
experts with the plan of their rows, the experts' products over those rows, the norms after and
before a block with its gate and residual (the experts' rows joined among them), and the rotation
by positions with several axes.

`run` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at
the end; the choice of experts in 64, where two scores may lie next to one another), or, where
`own` is true, through this package's operators on the same inputs.  `exact` is the same result
from the definition in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_package = {}


# ---- cases --------------------------------------------------------------------------------
def _route(name, tokens, experts, top_k, *, dtype="f32", scores="softmax", bias=False, groups=1,
           top_groups=1, group_best=2, renormalise=True, scale=1.0, seq=0, pitch=0, lens=1):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k,
            "dtype": dtype, "scores": scores, "bias": bias, "groups": groups,
            "top_groups": top_groups, "group_best": group_best, "renormalise": renormalise,
            "scale": scale, "seq": seq, "pitch": pitch, "lens": lens}


def _product(name, tokens, experts, top_k, n, k, *, gated=False, act="none", bias=False,
             gather=True, out="bf16", skew=0.5, padded=0.0, lens=1):
    return {"name": name, "op": "product", "tokens": tokens, "experts": experts, "top_k": top_k,
            "n": n, "k": k, "gated": gated, "act": act, "bias": bias, "gather": gather,
            "out": out, "skew": skew, "padded": padded, "lens": lens}


def _norm(name, rows, cols, *, x="f32", y="bf16", out="f32", h="bf16", after="rms", before="rms",
          gate="none", seq=0, packed=False, top_k=0, experts=0, shift=0.0, x_scale=1.0, y_scale=1.0,
          lens=1):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "x": x, "y": y, "out": out,
            "h": h, "after": after, "before": before, "gate": gate, "seq": seq, "packed": packed,
            "top_k": top_k, "experts": experts, "shift": shift, "x_scale": x_scale,
            "y_scale": y_scale, "lens": lens}


def _rotary(name, tokens, sections, *, heads=16, kv_heads=8, dim=128, dtype="bf16", cycle=False,
            interleaved=False, norm=True, fused=False, lens=1):
    return {"name": name, "op": "rotary", "tokens": tokens, "sections": sections,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "cycle": cycle,
            "interleaved": interleaved, "norm": norm, "fused": fused, "lens": lens}


def listed():
    return [
        # One new token of each of 8 texts: every launch counts.
        _route("route-8-tokens", 8, 64, 8),
        # A large packed batch over many experts, scores of their own, kept in balance by a bias
        # and limited to a few groups.
        _route("route-groups-bias-16k", 16384, 256, 8, scores="sigmoid", bias=True, groups=8,
               top_groups=4, scale=2.5),
        # The bf16 logits of a padded batch of 512 texts, as the projection wrote them.
        _route("route-bf16-padded-64k", 65536, 128, 8, dtype="bf16", seq=128),
        # The widening product of 8 new tokens, each with experts of its own.
        _product("experts-gated-8-tokens", 8, 64, 8, 512, 1024, gated=True, act="silu"),
        # A batch of 777 tokens over few experts, widths that divide nothing.
        _product("experts-odd-gelu", 777, 8, 2, 1000, 1001, act="gelu", bias=True, padded=0.1),
        # The widening product of a large packed batch.
        _product("experts-gated-8k", 8192, 64, 8, 512, 1024, gated=True, act="silu"),
        # The narrowing product behind it, over rows that lie by expert already.
        _product("experts-down-8k", 8192, 64, 8, 1024, 512, gather=False),
        # One new token of each of 8 texts: join the experts' rows, add, norm of the next block.
        _norm("norm-join-8-tokens", 8, 1024, top_k=8, experts=64, after="none"),
        # A large packed batch between two blocks, normed on both sides.
        _norm("norm-both-sides-33500", 33500, 1024),
        # The experts' rows of a large batch joined, gated by sequence, normed for the next block.
        _norm("norm-join-gate-8k", 8192, 1024, top_k=8, experts=64, gate="sequence", seq=512,
              before="layer"),
        # Text and video tokens of a packed batch inside the fused rows of the projection.
        _rotary("rotary-three-axes-64k", 65536, "16/24/24", fused=True, cycle=True),
        # The patches of one small image in fp32, rows and columns in a half of each head each.
        _rotary("rotary-image-fp32", 196, "8/8", heads=12, kv_heads=12, dim=32, dtype="f32",
                norm=False, interleaved=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "product", "product", "norm", "rotary"])
    if op == "route":
        experts = rng.choice([4, 8, 16, 60, 64, 96, 128, 160, 256, 512])
        tokens = _log(rng, 1, min(65536, 65536 * 128 // experts))
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if experts % g == 0])
        top_groups = rng.randint(1, groups)
        return _nameless(_route(
            "", tokens, experts, rng.randint(1, min(8, experts // groups * top_groups)),
            dtype=rng.choice(["f32", "f32", "bf16"]), scores=rng.choice(["softmax", "sigmoid"]),
            bias=rng.random() < 0.5, groups=groups, top_groups=top_groups,
            group_best=rng.choice([1, 2]), renormalise=rng.random() < 0.7,
            scale=rng.choice([1.0, 2.5]), seq=rng.choice([0, 0, _log(rng, 1, 512)]),
            pitch=rng.choice([0, 0, 3]), lens=rng.randrange(1 << 20)))
    if op == "product":
        experts = rng.choice([4, 8, 16, 60, 64, 128])
        top_k = rng.randint(1, min(8, experts))
        n, k, gated = _log(rng, 64, 2048), _log(rng, 64, 2048), rng.random() < 0.5
        most = 8192 * 8 * 512 * 1024 // (n * k * top_k) // (1 if gated else 2) * 2
        return _nameless(_product(
            "", _log(rng, 1, max(2, min(8192, most))), experts, top_k, n, k, gated=gated,
            act=rng.choice(["silu", "gelu", "gelu_tanh"] if gated else
                           ["none", "none", "relu", "gelu", "gelu_tanh", "silu"]),
            bias=rng.random() < 0.4, gather=rng.random() < 0.6,
            out=rng.choice(["bf16", "bf16", "f32"]), skew=rng.choice([0.0, 0.5, 1.5]),
            padded=rng.choice([0.0, 0.0, 0.2]), lens=rng.randrange(1 << 20)))
    if op == "norm":
        cols = rng.choice([384, 768, 1024, 2048, 4096, _log(rng, 32, 4096)])
        top_k = rng.choice([0, 0, 2, 4, 8])
        rows = _log(rng, 1, min(33500, 33500 * 1024 // (cols * max(1, top_k // 2))))
        return _nameless(_norm(
            "", rows, cols, x=rng.choice(["f32", "f32", "bf16"]), y=rng.choice(["bf16", "f32"]),
            out=rng.choice(["f32", "f32", "bf16"]), h=rng.choice(["bf16", "bf16", "f32"]),
            after=rng.choice(["rms", "layer", "none"]), before=rng.choice(["rms", "layer"]),
            gate=rng.choice(["none", "column", "sequence", "row"]), seq=_log(rng, 1, 512),
            packed=rng.random() < 0.5, top_k=top_k, experts=64 if top_k else 0,
            shift=rng.choice([0.0, 1.0]), x_scale=rng.choice([1.0, 0.5]),
            y_scale=rng.choice([1.0, 0.22]), lens=rng.randrange(1 << 20)))
    heads, kv_heads, dim, sections = rng.choice([
        (16, 8, 128, "16/24/24"), (16, 8, 128, "24/20/20"), (12, 12, 64, "16/16"),
        (12, 12, 32, "8/8"), (9, 3, 80, "8/16/16"), (32, 8, 128, "10/11/11"),
        (8, 1, 256, "32/32/32/32"), (6, 2, 96, "5/7")])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    top = 65536 * 24 * 128 * 2 // ((heads + kv_heads) * dim * (4 if dtype == "f32" else 2))
    return _nameless(_rotary(
        "", _log(rng, 1, min(top, 131072)), sections, heads=heads, kv_heads=kv_heads, dim=dim,
        dtype=dtype, cycle=rng.random() < 0.5, interleaved=rng.random() < 0.5,
        norm=rng.random() < 0.5, fused=rng.random() < 0.5, lens=rng.randrange(1 << 20)))


def _nameless(case):
    del case["name"]
    return case


# ---- what follows from a case alone -----------------------------------------------------------
def _lengths(c):
    """Valid rows of each sequence of a padded batch."""
    return np.random.default_rng(c["lens"]).integers(0, c["seq"] + 1, -(-c["tokens"] // c["seq"]))


def _sections(c):
    """Rotated pairs of each axis."""
    return [int(x) for x in c["sections"].split("/")]


def _plan(c):
    """A routing of the case's tokens as a router leaves it: some experts liked more than others,
    padded tokens without any.  Returns (offsets, order, places)."""
    rng = np.random.default_rng(c["lens"])
    t, e, k = c["tokens"] if "tokens" in c else c["rows"], c["experts"], c["top_k"]
    liked = c.get("skew", 0.5) * rng.standard_normal(e) + rng.gumbel(size=(t, e))
    ids = np.argpartition(-liked, k - 1, axis=1)[:, :k]
    ids[rng.random(t) < c.get("padded", 0.0)] = e  # behind all experts: no rows
    flat = ids.reshape(-1)
    by = np.argsort(flat, kind="stable")
    offsets = np.searchsorted(flat[by], np.arange(e + 1))
    places = np.empty(t * k, np.int64)
    places[by] = np.arange(t * k)
    places[flat == e] = -1
    order = np.where(np.arange(t * k) < offsets[e], by, -1)
    return offsets, order, places.reshape(t, k)


def work(c):
    size = {"f32": 4, "bf16": 2, "none": 0}
    if c["op"] == "route":
        t, e, k = c["tokens"], c["experts"], c["top_k"]
        return {"bytes": t * e * size[c["dtype"]] + 16 * t * k + 4 * (e + 1) + 4 * e * c["bias"],
                "flops": t * e * 4}
    if c["op"] == "product":
        offsets, _, _ = _plan(c)
        rows, used = int(offsets[-1]), int(np.count_nonzero(np.diff(offsets)))
        wide = c["n"] * (2 if c["gated"] else 1)
        read = c["tokens"] if c["gather"] and rows else rows
        return {"bytes": 2 * c["k"] * (read + used * wide) + rows * c["n"] * size[c["out"]]
                + 4 * used * wide * c["bias"] + (4 * rows if c["gather"] else 0),
                "flops": 2 * rows * wide * c["k"]}
    if c["op"] == "norm":
        n, e = c["rows"] * c["cols"], max(1, c["top_k"])
        gates = {"none": 0, "column": 1, "sequence": -(-c["rows"] // max(1, c["seq"])),
                 "row": c["rows"]}[c["gate"]]
        return {"bytes": n * (size[c["x"]] + e * size[c["y"]] + size[c["out"]] + size[c["h"]])
                + 4 * gates * c["cols"] + 8 * c["rows"] * c["top_k"], "flops": n * (2 * e + 10)}
    n = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
    return {"bytes": 2 * n * size[c["dtype"]] + 4 * c["tokens"] * len(_sections(c)),
            "flops": n * (6 if c["norm"] else 3)}


# ---- inputs -------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32).to(DEV)


def _normal(g, shape, dtype, scale=1.0, middle=0.0):
    x = torch.empty(shape, dtype=torch.float32, device=DEV).normal_(middle, scale, generator=g)
    return x.to(_TYPES[dtype])


def _prepare_route(c, seed):
    g = _generator(seed)
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    logits = _normal(g, (t, e + c["pitch"]), c["dtype"], 1.5)[:, :e]
    return {"case": c, "logits": logits,
            "bias": _normal(g, (e,), "f32", 0.1) if c["bias"] else None,
            "lengths": _i32(_lengths(c)) if c["seq"] else None,
            "experts": torch.zeros((t, k), dtype=torch.int32, device=DEV),
            "weights": torch.zeros((t, k), dtype=torch.float32, device=DEV),
            "offsets": torch.zeros(e + 1, dtype=torch.int32, device=DEV),
            "order": torch.full((t * k,), -1, dtype=torch.int32, device=DEV),
            "places": torch.zeros((t, k), dtype=torch.int32, device=DEV)}


def _prepare_product(c, seed):
    g = _generator(seed)
    n, k, e = c["n"], c["k"], c["experts"]
    wide = n * (2 if c["gated"] else 1)
    ld = -(-k // 8) * 8  # rows start on 16 bytes, as such a program lays them out
    offsets, order, _ = _plan(c)
    rows = c["tokens"] * c["top_k"]
    return {"case": c, "x": _normal(g, (c["tokens"] if c["gather"] else rows, ld), "bf16")[:, :k],
            "w": _normal(g, (e, wide, ld), "bf16", k ** -0.5)[:, :, :k],
            "bias": _normal(g, (e, wide), "f32") if c["bias"] else None,
            "offsets": _i32(offsets), "order": _i32(order) if c["gather"] else None,
            "bounds": [int(o) for o in offsets],
            "out": torch.zeros((rows, n), dtype=_TYPES[c["out"]], device=DEV)}


def _norm_weights(g, c, kind):
    """(weight, bias): RMS weights are bf16 around 1 (or around 0 where 1 is added to them),
    LayerNorm's fp32."""
    if kind == "none":
        return None, None
    if kind == "rms":
        return _normal(g, (c["cols"],), "bf16", 0.1, 1.0 - c["shift"]), None
    return _normal(g, (c["cols"],), "f32", 0.1, 1.0), _normal(g, (c["cols"],), "f32", 0.1)


def _prepare_norm(c, seed):
    g = _generator(seed)
    rows, cols = c["rows"], c["cols"]
    s = {"case": c, "x": _normal(g, (rows, cols), c["x"]), "places": None, "join": None,
         "y": _normal(g, (rows * max(1, c["top_k"]), cols), c["y"], 2.0),
         "after": _norm_weights(g, c, c["after"]), "before": _norm_weights(g, c, c["before"]),
         "gate": None, "cu": None, "which": None,
         "out": torch.empty((rows, cols), dtype=_TYPES[c["out"]], device=DEV),
         "h": torch.empty((rows, cols), dtype=_TYPES[c["h"]], device=DEV)}
    if c["top_k"]:
        s["places"] = _i32(_plan(c)[2])
        s["join"] = torch.rand((rows, c["top_k"]), generator=g, device=DEV) / c["top_k"]
    if c["gate"] == "column":
        s["gate"] = _normal(g, (1, cols), "f32")
    elif c["gate"] == "row":
        s["gate"] = _normal(g, (rows, cols), "f32")
    elif c["gate"] == "sequence":
        cuts = np.arange(0, rows + c["seq"], c["seq"]).clip(max=rows)
        if c["packed"]:
            inner = np.random.default_rng(c["lens"]).integers(0, rows + 1, len(cuts) - 2)
            cuts = np.r_[0, np.sort(inner), rows]
            s["cu"] = _i32(cuts)
        s["which"] = torch.repeat_interleave(torch.arange(len(cuts) - 1, device=DEV),
                                             torch.from_numpy(np.diff(cuts)).to(DEV))
        s["gate"] = _normal(g, (len(cuts) - 1, cols), "f32")
    return s


def _pair_axes(c):
    """The axis of each rotated pair: one section after the other, or the axes in turn until each
    has had its pairs."""
    if not c["cycle"]:
        return np.repeat(np.arange(len(_sections(c))), _sections(c))
    left, out = _sections(c), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return np.array(out)


def _prepare_rotary(c, seed):
    g = _generator(seed)
    t, h, hk, d, axes = c["tokens"], c["heads"], c["kv_heads"], c["dim"], len(_sections(c))
    if c["fused"]:
        qkv = _normal(g, (t, h + 2 * hk, d), c["dtype"])
        q, k = qkv[:, :h], qkv[:, h:h + hk]
    else:
        q, k = _normal(g, (t, h, d), c["dtype"]), _normal(g, (t, hk, d), c["dtype"])
    pairs = sum(_sections(c))
    s = {"case": c, "q": q, "k": k,
         "q_out": torch.empty((t, h, d), dtype=q.dtype, device=DEV),
         "k_out": torch.empty((t, hk, d), dtype=q.dtype, device=DEV), "qw": None, "kw": None,
         "freq": torch.from_numpy((1e6 ** (-np.arange(pairs) / pairs)).astype(np.float32)).to(DEV),
         "pair_axes": _i32(_pair_axes(c)),
         # Frames and patches of clips that follow one another, the centre of an image at zero.
         "positions": torch.randint(-512, 16384, (axes, t), generator=g, device=DEV,
                                    dtype=torch.int32)}
    if c["norm"]:
        s["qw"], s["kw"] = (_normal(g, (d,), "bf16", 0.02, 1.0) for _ in range(2))
    return s


def prepare(case, seed):
    return {"route": _prepare_route, "product": _prepare_product, "norm": _prepare_norm,
            "rotary": _prepare_rotary}[case["op"]](case, seed)


# ---- the plain forms ------------------------------------------------------------------------
def _plain_route(s):
    c = s["case"]
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    z = s["logits"].double()
    if c["scores"] == "softmax":
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-z))
    rank = p if s["bias"] is None else p + s["bias"].double()
    if c["groups"] > 1:
        best = rank.view(t, c["groups"], -1).sort(dim=-1, descending=True).values
        best = best[..., :c["group_best"]].sum(-1)
        chosen = best.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros((t, c["groups"]), dtype=torch.bool, device=z.device)
        keep.scatter_(1, chosen, True)
        rank = torch.where(keep.repeat_interleave(e // c["groups"], 1), rank, -math.inf)
    ids = rank.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, ids)
    if c["renormalise"]:
        w = w / w.sum(-1, keepdim=True)
    w = w * c["scale"]
    if c["seq"]:
        row = torch.arange(t, device=z.device)
        none = (row % c["seq"] >= s["lengths"][row // c["seq"]])[:, None]
        ids, w = torch.where(none, -1, ids), torch.where(none, 0.0, w)
    flat = torch.where(ids < 0, e, ids).reshape(-1)
    by = flat.sort(stable=True).indices
    counts = torch.zeros(e + 1, dtype=torch.int64, device=z.device)
    counts.scatter_add_(0, flat, torch.ones_like(flat))
    offsets = counts.cumsum(0) - counts
    at = torch.arange(t * k, device=z.device)
    order = torch.where(at < offsets[e], by, -1)
    places = torch.empty_like(by).scatter_(0, by, at)
    places = torch.where(flat < e, places, -1).view(t, k)
    return ids.int(), w.float(), offsets.int(), order.int(), places.int()


def _activate(y, act):
    if act == "relu":
        return torch.where(y > 0, y, 0.0)
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y / (1 + torch.exp(-y)) if act == "silu" else y


def _plain_product(s):
    c, n = s["case"], s["case"]["n"]
    out = torch.zeros_like(s["out"])
    for e in range(c["experts"]):
        a, b = s["bounds"][e], s["bounds"][e + 1]
        if a == b:
            continue
        x = s["x"][s["order"][a:b] // c["top_k"]] if c["gather"] else s["x"][a:b]
        y = x.float() @ s["w"][e].float().t()
        if s["bias"] is not None:
            y = y + s["bias"][e]
        if c["gated"]:
            y = _activate(y[:, :n], c["act"]) * y[:, n:]
        else:
            y = _activate(y, c["act"])
        out[a:b] = y.to(out.dtype)
    return out


def _plain_norm_of(z, kind, weights, shift):
    if kind == "none":
        return z
    if kind == "rms":
        return z * torch.rsqrt((z * z).mean(-1, keepdim=True) + 1e-6) * (weights[0].float() + shift)
    z = z - z.mean(-1, keepdim=True)
    return z * torch.rsqrt((z * z).mean(-1, keepdim=True) + 1e-6) * weights[0] + weights[1]


def _plain_norm(s):
    c = s["case"]
    if c["top_k"]:
        z = torch.zeros((c["rows"], c["cols"]), dtype=torch.float32, device=DEV)
        for j in range(c["top_k"]):
            z = z + s["join"][:, j, None] * s["y"][s["places"][:, j]].float()
    else:
        z = s["y"].float()
    z = _plain_norm_of(z, c["after"], s["after"], c["shift"])
    if s["gate"] is not None:
        z = z * (s["gate"] if s["which"] is None else s["gate"][s["which"]])
    r = c["x_scale"] * s["x"].float() + c["y_scale"] * z
    h = _plain_norm_of(r, c["before"], s["before"], c["shift"])
    return r.to(s["out"].dtype), h.to(s["h"].dtype)


def _plain_rotary(s):
    c, half = s["case"], sum(_sections(s["case"]))
    angle = (s["positions"].float()[s["pair_axes"].long()].t() * s["freq"])[:, None, :]
    cos, sin = torch.cos(angle), torch.sin(angle)

    def turn(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
        if c["interleaved"]:
            a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
            z = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:2 * half]
            z = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([z, y[..., 2 * half:]], -1).to(x.dtype)

    return turn(s["q"], s["qw"]), turn(s["k"], s["kw"])


# ---- the package's operators ----------------------------------------------------------------
def _runtime():
    if "rt" not in _package:
        from tessery_b200 import TX_BF16, TX_F32, CudaRuntime

        _package.update(rt=CudaRuntime(torch.cuda.current_device()),
                        types={torch.bfloat16: TX_BF16, torch.float32: TX_F32})
    return _package["rt"], _package["types"]


def _ptr(x):
    return None if x is None else x.data_ptr()


def _stream():
    # torch's default stream is the legacy stream, which CUDA names 1 (0 would be the
    # runtime's own stream here).
    return torch.cuda.current_stream().cuda_stream or 1


def _own_route(s):
    rt, types = _runtime()
    c, z = s["case"], s["logits"]
    rt.experts_route_device(
        z.data_ptr(), s["experts"].data_ptr(), s["weights"].data_ptr(), tokens=c["tokens"],
        num_experts=c["experts"], top_k=c["top_k"], ld=z.stride(0), logits_dtype=types[z.dtype],
        bias=_ptr(s["bias"]), scores=c["scores"], groups=c["groups"], top_groups=c["top_groups"],
        group_best=c["group_best"], renormalise=c["renormalise"], scale=c["scale"],
        lengths=_ptr(s["lengths"]), seq=c["seq"], offsets=s["offsets"].data_ptr(),
        order=s["order"].data_ptr(), places=s["places"].data_ptr(), stream=_stream())
    return s["experts"], s["weights"], s["offsets"], s["order"], s["places"]


def _own_product(s):
    rt, types = _runtime()
    c, x, w = s["case"], s["x"], s["w"]
    rt.experts_linear_device(
        x.data_ptr(), w.data_ptr(), s["out"].data_ptr(), offsets=s["offsets"].data_ptr(),
        order=_ptr(s["order"]), tokens=c["tokens"], top_k=c["top_k"], num_experts=c["experts"],
        n=c["n"], k=c["k"], gated=c["gated"], activation=c["act"], bias=_ptr(s["bias"]),
        ldx=x.stride(0), ldw=w.stride(1), expert_stride=w.stride(0),
        out_dtype=types[s["out"].dtype], stream=_stream())
    return s["out"]


def _own_norm(s):
    rt, types = _runtime()
    c = s["case"]

    def norm(kind, weights):
        if kind == "none":
            return None
        return {"kind": kind, "weight": weights[0].data_ptr(), "bias": _ptr(weights[1]),
                "dtype": types[weights[0].dtype], "eps": 1e-6,
                "offset": c["shift"] if kind == "rms" else 0.0}

    gate = {}
    if s["gate"] is not None:
        gate = {"gate": s["gate"].data_ptr(), "gate_rows": s["gate"].shape[0]}
        if s["cu"] is not None:
            gate["cu_seqlens"] = s["cu"].data_ptr()
        elif c["gate"] != "column":
            gate["seq"] = 1 if c["gate"] == "row" else c["seq"]
    join = {}
    if c["top_k"]:
        join = {"places": s["places"].data_ptr(), "weights": s["join"].data_ptr(),
                "top_k": c["top_k"], "y_rows": s["y"].shape[0]}
    rt.block_norm_device(
        s["x"].data_ptr(), s["y"].data_ptr(), rows=c["rows"], cols=c["cols"],
        x_dtype=types[s["x"].dtype], y_dtype=types[s["y"].dtype], out=s["out"].data_ptr(),
        out_dtype=types[s["out"].dtype], h=s["h"].data_ptr(), h_dtype=types[s["h"].dtype],
        after=norm(c["after"], s["after"]), before=norm(c["before"], s["before"]),
        x_scale=c["x_scale"], y_scale=c["y_scale"], **gate, **join, stream=_stream())
    return s["out"], s["h"]


def _own_rotary(s):
    rt, types = _runtime()
    c, q, k = s["case"], s["q"], s["k"]
    rt.rotary_axes_device(
        q.data_ptr(), k.data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr(),
        tokens=c["tokens"], heads=c["heads"], kv_heads=c["kv_heads"], dim=c["dim"],
        inv_freq=s["freq"].data_ptr(), rot_dim=2 * s["freq"].numel(),
        pair_axes=s["pair_axes"].data_ptr(), positions=s["positions"].data_ptr(),
        axes=s["positions"].shape[0], interleaved=c["interleaved"], q_norm_weight=_ptr(s["qw"]),
        k_norm_weight=_ptr(s["kw"]), eps=1e-6, in_dtype=types[q.dtype], out_dtype=types[q.dtype],
        q_strides=q.stride()[:2], k_strides=k.stride()[:2], stream=_stream())
    return s["q_out"], s["k_out"]


def run(state):
    form = {"route": (_plain_route, _own_route), "product": (_plain_product, _own_product),
            "norm": (_plain_norm, _own_norm),
            "rotary": (_plain_rotary, _own_rotary)}[state["case"]["op"]][1 if own else 0]
    return form(state)


# ---- the definitions in 64 bits -------------------------------------------------------------
def _place_of(values):
    """The place of each value of a row from the largest down, the lower index first among equals:
    how many values come before it."""
    before = torch.zeros(values.shape, dtype=torch.int64, device=values.device)
    at = torch.arange(values.shape[1], device=values.device)
    for j in range(values.shape[1]):
        v = values[:, j:j + 1]
        before += (v > values) | ((v == values) & (j < at))
    return before


def _exact_route(c, s):
    t, e, k, per = c["tokens"], c["experts"], c["top_k"], c["experts"] // c["groups"]
    z = s["logits"].double()
    p = torch.softmax(z, -1) if c["scores"] == "softmax" else torch.sigmoid(z)
    rank = p.clone()
    if s["bias"] is not None:
        rank += s["bias"].double()
    if c["groups"] > 1:
        sums = [rank[:, g * per:(g + 1) * per].topk(min(per, c["group_best"])).values.sum(-1)
                for g in range(c["groups"])]
        out = _place_of(torch.stack(sums, 1)) >= c["top_groups"]
        for g in range(c["groups"]):
            rank[:, g * per:(g + 1) * per].masked_fill_(out[:, g:g + 1], -math.inf)
    place = _place_of(rank)
    ids = torch.stack([torch.nonzero(place == j)[:, 1] for j in range(k)], 1)
    w = torch.gather(p, 1, ids)
    if c["renormalise"]:
        w /= w.sum(-1, keepdim=True)
    w *= c["scale"]
    ids = ids.cpu().numpy()
    if c["seq"]:
        for b, n in enumerate(_lengths(c)):
            ids[b * c["seq"] + n:(b + 1) * c["seq"]] = -1
            w[b * c["seq"] + int(n):(b + 1) * c["seq"]] = 0
    pairs = [np.flatnonzero(ids.reshape(-1) == x) for x in range(e)]
    offsets = np.concatenate([[0], np.cumsum([len(x) for x in pairs])])
    order, places = np.full(t * k, -1), np.full(t * k, -1)
    order[:offsets[-1]] = np.concatenate(pairs)
    places[order[:offsets[-1]]] = np.arange(offsets[-1])
    return _i32(ids), w, _i32(offsets), _i32(order), _i32(places.reshape(t, k))


def _exact_product(c, s):
    offsets, order, _ = _plan(c)
    y = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    for e in np.flatnonzero(np.diff(offsets)):
        at = np.arange(offsets[e], offsets[e + 1])
        rows = torch.from_numpy(order[at] // c["top_k"] if c["gather"] else at).to(DEV)
        z = s["x"].index_select(0, rows).double() @ s["w"][e].double().t()
        if s["bias"] is not None:
            z += s["bias"][e].double()
        u = z
        if c["gated"]:
            u, z = z.split(c["n"], 1)
        if c["act"] == "relu":
            f = u.clamp(min=0)
        elif c["act"] == "gelu":
            f = u * torch.special.ndtr(u)
        elif c["act"] == "gelu_tanh":
            # (1 + tanh v) / 2 is the logistic function of 2v
            f = u * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3))
        elif c["act"] == "silu":
            f = u * torch.sigmoid(u)
        else:
            f = u
        y[int(offsets[e]):int(offsets[e + 1])] = f * z if c["gated"] else f
    return y


def _exact_norm(c, s):
    def norm(z, kind, weights):
        if kind == "none":
            return z
        w = weights[0].double()
        if kind == "rms":
            return z / (z.square().sum(-1, keepdim=True) / c["cols"] + 1e-6).sqrt() * (
                w + c["shift"])
        var, mean = torch.var_mean(z, -1, keepdim=True, correction=0)
        return (z - mean) / (var + 1e-6).sqrt() * w + weights[1].double()

    z = s["y"].double()
    if c["top_k"]:
        z = (z[s["places"].long().flatten()] * s["join"].double().reshape(-1, 1)).view(
            c["rows"], c["top_k"], c["cols"]).sum(1)
    z = norm(z, c["after"], s["after"])
    if c["gate"] == "sequence":
        z = z * s["gate"].double().index_select(0, s["which"])
    elif c["gate"] != "none":
        z = z * s["gate"].double()
    r = s["x"].double() * c["x_scale"] + z * c["y_scale"]
    return r, norm(r, c["before"], s["before"])


def _exact_rotary(c, s):
    half = sum(_sections(c))
    # The angle is by definition the fp32 product of position and frequency.
    pos = s["positions"].cpu().numpy().astype(np.float32)[_pair_axes(c)]
    angle = (pos.T * s["freq"].cpu().numpy()[None]).astype(np.float64)
    turn = torch.polar(torch.ones(angle.shape, dtype=torch.float64),
                       torch.from_numpy(angle)).to(DEV)[:, None]

    def one(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / c["dim"] + 1e-6) * w.double()
        y = y.clone()
        first = slice(0, 2 * half, 2) if c["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if c["interleaved"] else slice(half, 2 * half)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return one(s["q"], s["qw"]), one(s["k"], s["kw"])


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    return {"route": _exact_route, "product": _exact_product, "norm": _exact_norm,
            "rotary": _exact_rotary}[c["op"]](c, s)
