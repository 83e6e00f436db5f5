"""Measured cases of the encoder-layer operators: the position rotation of q and k (with
their per-head norms), attention under a score rule (cap, distance bias, window, prefix,
documents), and the linear layer with bias, activation and residual.

`run` computes a case in its plain form (elementary torch operations in 32 bits, rounded
once at the end), or, where `own` is true, through this package's operators on the same
inputs.  `exact` is the same result from the definition in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_package = {}


# ---- cases --------------------------------------------------------------------------------
def _rotary(name, tokens, *, heads=16, kv_heads=8, dim=128, rot=128, dtype="bf16",
            interleaved=False, norm=True, positions="packed", scaled=False, fused=False, lens=1):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "dtype": dtype, "interleaved": interleaved, "norm": norm,
            "positions": positions, "scaled": scaled, "fused": fused, "lens": lens}


def _attend(name, nseq, longest, *, shortest=1, new=0, heads=16, kv_heads=8, dim=128,
            dtype="bf16", causal=True, left=-1, right=-1, cap=0.0, bias="none", reach=0, prefix=0,
            docs=0, padded=False, fused=False, lens=1):
    return {"name": name, "op": "attend", "nseq": nseq, "longest": longest, "shortest": shortest,
            "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "causal": causal, "left": left, "right": right, "cap": cap, "bias": bias,
            "reach": reach, "prefix": prefix, "docs": docs, "padded": padded, "fused": fused,
            "lens": lens}


def _linear(name, m, n, k, *, act="none", bias=True, residual="none", out="bf16"):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "act": act, "bias": bias,
            "residual": residual, "out": out}


def listed():
    return [
        # One new token of each of 8 texts, far into long contexts, frequencies stretched.
        _rotary("rotary-8-new-tokens", 8, positions="given", scaled=True),
        # A packed batch of documents inside the fused q/k/v rows of the projection.
        _rotary("rotary-norm-packed-64k", 65536, fused=True),
        # A small fp32 encoder: interleaved pairs over half of each head, padded texts.
        _rotary("rotary-fp32-interleaved", 8192, heads=12, kv_heads=12, dim=32, rot=16,
                dtype="f32", interleaved=True, norm=False, positions="padded"),
        # One more token of each of 8 texts against the keys kept for it.
        _attend("attend-one-token-cap", 8, 2048, shortest=64, new=1, cap=30.0, padded=True),
        # The ordinary ragged batch of the embedding encoder, scores capped.
        _attend("attend-causal-cap-packed", 32, 512, shortest=32, cap=50.0, fused=True),
        # A small fp32 encoder whose scores fall with the distance; 64 short texts.
        _attend("attend-fp32-slopes", 64, 128, shortest=16, heads=12, kv_heads=12, dim=32,
                dtype="f32", causal=False, bias="slopes"),
        # One long document, each token seeing the 4096 before it.
        _attend("attend-long-window", 1, 8192, shortest=8192, left=4095),
        # Rows packed from several documents, a bias per distance, an open prefix.
        _attend("attend-documents-table", 8, 2048, shortest=1500, heads=12, kv_heads=12, dim=64,
                causal=False, bias="table", reach=128, prefix=64, docs=400),
        # A single row: the projection of one new token.
        _linear("linear-one-row-silu", 1, 1024, 1024, act="silu"),
        # Odd sizes: a batch of 777 tokens, widths that divide nothing.
        _linear("linear-odd-gelu", 777, 1000, 1001, act="gelu_tanh"),
        # The small encoder's widening layer over 64 texts of 128.
        _linear("linear-widen-gelu", 8192, 1536, 384, act="gelu"),
        # The output projection of a large packed batch into the fp32 residual stream.
        _linear("linear-residual-33500", 33500, 1024, 2048, bias=False, residual="f32", out="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "attend", "attend", "linear"])
    if op == "rotary":
        heads, kv_heads, dim = rng.choice([(16, 8, 128), (12, 12, 32), (12, 12, 64), (9, 3, 80),
                                           (8, 1, 256), (32, 8, 128), (6, 2, 96)])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        top = 65536 * 24 * 128 * 2 // ((heads + kv_heads) * dim * (4 if dtype == "f32" else 2))
        return _nameless(_rotary(
            "", _log(rng, 1, min(top, 131072)), heads=heads, kv_heads=kv_heads, dim=dim,
            rot=rng.choice([dim, dim, dim // 2, dim // 4]), dtype=dtype,
            interleaved=rng.random() < 0.5, norm=rng.random() < 0.5,
            positions=rng.choice(["given", "packed", "padded"]), scaled=rng.random() < 0.5,
            fused=rng.random() < 0.5, lens=rng.randrange(1 << 20)))
    if op == "linear":
        n, k = _log(rng, 64, 4096), _log(rng, 64, 4096)
        m = _log(rng, 1, max(2, min(33500, 33500 * 1024 * 2048 // (n * k))))
        return _nameless(_linear(
            "", m, n, k, act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
            bias=rng.random() < 0.6, residual=rng.choice(["none", "f32", "bf16"]),
            out=rng.choice(["bf16", "f32"])))
    heads, kv_heads, dim = rng.choice([(16, 8, 128), (12, 12, 32), (12, 12, 64), (9, 3, 80),
                                       (8, 1, 128), (32, 8, 128), (6, 2, 96)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    new = rng.choice([0, 0, 0, 1, 1, 5, 17])
    most = 16 * 8192 * 3000 // (4 if dtype == "f32" else 1)  # query rows x keys x heads
    longest = _log(rng, 1, 8192 if new else min(8192, math.isqrt(most // heads)))
    rows = longest * kv_heads * dim * (2 if dtype == "f32" else 1)
    nseq = _log(rng, 1, max(1, min(256, most // (heads * longest * (new or longest)),
                                   190_000_000 // rows)))
    bias = rng.choice(["none", "none", "slopes", "table"])
    docs = rng.random() < 0.25 and not new
    causal = rng.random() < 0.6
    return _nameless(_attend(
        "", nseq, longest, shortest=_log(rng, 1, longest), new=new, heads=heads,
        kv_heads=kv_heads, dim=dim, dtype=dtype, causal=causal,
        left=rng.choice([-1, -1, _log(rng, 1, 2048)]),
        right=-1 if causal else rng.choice([-1, -1, _log(rng, 1, 2048)]),
        cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=bias,
        reach=_log(rng, 8, 512) if bias == "table" else 0,
        prefix=rng.choice([0, 0, _log(rng, 1, 300)]), docs=_log(rng, 20, 1000) if docs else 0,
        padded=rng.random() < 0.4, fused=not new and rng.random() < 0.5,
        lens=rng.randrange(1 << 20)))


def _nameless(case):
    del case["name"]
    return case


# ---- what follows from a case alone: lengths, prefixes, documents ---------------------------
def _attend_shape(c):
    """Per sequence: key rows and query rows; per sequence the prefix; per token its document
    (a packed row's documents follow one another; about one in sixteen is padding, -1)."""
    rng = np.random.default_rng(c["lens"])
    nk = rng.integers(c["shortest"], c["longest"] + 1, size=c["nseq"])
    nk[0] = c["longest"]
    nq = np.minimum(nk, c["new"]) if c["new"] else nk
    prefix = rng.integers(0, c["prefix"] + 1, size=c["nseq"]) if c["prefix"] else None
    docs = None
    if c["docs"]:
        docs = []
        for n in nk:
            ids = np.cumsum(rng.random(n) < 1.0 / c["docs"])
            pad = rng.random(int(ids[-1]) + 1) < 1 / 16
            docs.append(np.where(pad[ids], -1, ids))
    return nk.astype(np.int64), nq.astype(np.int64), prefix, docs


def _open_pairs(c):
    """(query, key) pairs that the rule leaves open, per head."""
    nk, nq, prefix, docs = _attend_shape(c)
    total = 0
    for s in range(c["nseq"]):
        p = np.arange(nk[s] - nq[s], nk[s])
        lo = np.maximum(p - c["left"], 0) if c["left"] >= 0 else np.zeros_like(p)
        hi = p + 1 if c["causal"] else np.full_like(p, nk[s])
        if c["right"] >= 0:
            hi = np.minimum(hi, p + c["right"] + 1)
        hi = np.minimum(hi, nk[s])
        pre = min(int(prefix[s]), int(nk[s])) if prefix is not None else 0
        d0, d1 = np.zeros_like(p), np.full_like(p, nk[s])
        if docs is not None:
            ids = docs[s]
            edge = np.flatnonzero(np.diff(ids)) + 1
            starts, ends = np.r_[0, edge], np.r_[edge, nk[s]]
            run_of = np.searchsorted(starts, p, side="right") - 1
            d0 = starts[run_of]
            d1 = np.where(ids[p] >= 0, ends[run_of], d0)
        a0, a1 = np.maximum(lo, d0), np.minimum(hi, d1)
        b0, b1 = d0, np.minimum(pre, d1)
        both = np.maximum(np.minimum(a1, b1) - np.maximum(a0, b0), 0)
        total += int((np.maximum(a1 - a0, 0) + np.maximum(b1 - b0, 0) - both).sum())
    return total


def work(c):
    if c["op"] == "rotary":
        e = 4 if c["dtype"] == "f32" else 2
        n = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        return {"bytes": 2 * n * e, "flops": n * (6 if c["norm"] else 3)}
    if c["op"] == "linear":
        e = {"none": 0, "f32": 4, "bf16": 2}
        return {"bytes": 2 * c["k"] * (c["m"] + c["n"]) + c["m"] * c["n"] * (
            e[c["residual"]] + e[c["out"]]) + (4 * c["n"] if c["bias"] else 0),
            "flops": 2 * c["m"] * c["n"] * c["k"]}
    nk, nq, _, _ = _attend_shape(c)
    e = 4 if c["dtype"] == "f32" else 2
    rows = 2 * int(nq.sum()) * c["heads"] + 2 * int(nk.sum()) * c["kv_heads"]
    return {"bytes": rows * c["dim"] * e, "flops": 4 * c["dim"] * c["heads"] * _open_pairs(c)}


# ---- inputs -------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32).to(DEV)


def _normal(g, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=torch.float32, device=DEV).normal_(generator=g)
    return (x * scale).to(_TYPES[dtype]) if scale != 1.0 else x.to(_TYPES[dtype])


def _qkv(g, c, rows_q, rows_k, dtype):
    """q, k, v [rows, heads, dim]: columns of one fused row, or arrays of their own."""
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    if c["fused"]:
        qkv = _normal(g, (rows_q, h + 2 * hk, d), dtype)
        return qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    return (_normal(g, (rows_q, h, d), dtype), _normal(g, (rows_k, hk, d), dtype),
            _normal(g, (rows_k, hk, d), dtype))


def _frequencies(c):
    """Inverse frequencies theta^(-2c/rot) as fp32; scaled: stretched by 4 in the columns that
    turn less than once over 4096 positions, with the amplitude that goes with it."""
    f = 1e6 ** (-2.0 * np.arange(c["rot"] // 2) / c["rot"])
    if not c["scaled"]:
        return f.astype(np.float32), 1.0
    return np.where(f * 4096 < 2 * np.pi, f / 4, f).astype(np.float32), 0.1 * math.log(4.0) + 1.0


def _prepare_rotary(c, seed):
    g = _generator(seed)
    t, d = c["tokens"], c["dim"]
    q, k, _ = _qkv(g, c, t, t, c["dtype"])
    freq, amplitude = _frequencies(c)
    s = {"case": c, "q": q, "k": k, "freq": torch.from_numpy(freq).to(DEV), "amplitude": amplitude,
         "q_out": torch.empty((t, c["heads"], d), dtype=q.dtype, device=DEV),
         "k_out": torch.empty((t, c["kv_heads"], d), dtype=q.dtype, device=DEV),
         "qw": None, "kw": None, "positions": None, "cu": None, "seq": 0}
    if c["norm"]:
        s["qw"] = (1 + 0.02 * _normal(g, (d,), "f32")).to(torch.bfloat16)
        s["kw"] = (1 + 0.02 * _normal(g, (d,), "f32")).to(torch.bfloat16)
    rng = np.random.default_rng(c["lens"])
    if c["positions"] == "given":
        s["positions"] = torch.randint(0, 32768, (t,), generator=g, device=DEV, dtype=torch.int32)
    elif c["positions"] == "packed":
        cuts = np.unique(np.r_[0, rng.integers(0, t + 1, size=max(1, t // 300)), t])
        s["cu"] = _i32(cuts)
        s["which"] = torch.repeat_interleave(torch.arange(len(cuts) - 1, device=DEV),
                                             torch.from_numpy(np.diff(cuts)).to(DEV))
    else:
        s["seq"] = min(t, 128)
    return s


def _prepare_attend(c, seed):
    g = _generator(seed)
    nk, nq, prefix, docs = _attend_shape(c)
    padded, d, h = c["padded"], c["dim"], c["heads"]
    longest_q, longest_k = int(nq.max()), int(nk.max())
    rows_q = c["nseq"] * longest_q if padded else int(nq.sum())
    rows_k = c["nseq"] * longest_k if padded else int(nk.sum())
    q, k, v = _qkv(g, c, rows_q, rows_k, c["dtype"])
    s = {"case": c, "q": q, "k": k, "v": v, "longest_q": longest_q, "longest_k": longest_k,
         "nq": _i32(nq), "nk": _i32(nk), "cu_q": _i32(np.r_[0, np.cumsum(nq)]),
         "cu_k": _i32(np.r_[0, np.cumsum(nk)]), "slopes": None, "table": None, "prefix": None,
         "docs": None, "out": torch.empty((rows_q, h, d), dtype=q.dtype, device=DEV)}
    if c["bias"] == "slopes":
        s["slopes"] = torch.from_numpy((2.0 ** (-8.0 * (1 + np.arange(h)) / h)).astype(
            np.float32)).to(DEV)
    elif c["bias"] == "table":
        s["table"] = _normal(g, (h, 2 * c["reach"] + 1), "f32")
    if prefix is not None:
        s["prefix"] = _i32(prefix)
    if docs is not None:
        full = np.full((c["nseq"], longest_k), -1)
        for i, row in enumerate(docs):
            full[i, :len(row)] = row
        s["docs"] = _i32(full.reshape(-1) if padded else np.concatenate(docs))
    return s


def _prepare_linear(c, seed):
    g = _generator(seed)
    m, n, k = c["m"], c["n"], c["k"]
    ld = -(-k // 8) * 8  # rows start on 16 bytes, as such a program lays them out
    x = _normal(g, (m, ld), "bf16")[:, :k]
    w = _normal(g, (n, ld), "bf16", k ** -0.5)[:, :k]
    return {"case": c, "x": x, "w": w, "bias": _normal(g, (n,), "f32") if c["bias"] else None,
            "residual": None if c["residual"] == "none" else _normal(g, (m, n), c["residual"]),
            "out": torch.empty((m, n), dtype=_TYPES[c["out"]], device=DEV)}


def prepare(case, seed):
    return {"rotary": _prepare_rotary, "attend": _prepare_attend,
            "linear": _prepare_linear}[case["op"]](case, seed)


# ---- the plain forms ------------------------------------------------------------------------
def _positions(s):
    t = s["case"]["tokens"]
    if s["positions"] is not None:
        return s["positions"]
    if s["cu"] is not None:
        return torch.arange(t, device=DEV) - s["cu"][s["which"]]
    return torch.arange(t, device=DEV) % s["seq"]


def _plain_rotary(s):
    c, r = s["case"], s["case"]["rot"]
    angle = (_positions(s).float()[:, None] * s["freq"])[:, None, :]
    cos, sin = torch.cos(angle) * s["amplitude"], torch.sin(angle) * s["amplitude"]

    def turn(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
        if c["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            z = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :r // 2], y[..., r // 2:r]
            z = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([z, y[..., r:]], -1).to(x.dtype)

    return turn(s["q"], s["qw"]), turn(s["k"], s["kw"])


def _plain_attend(s):
    c = s["case"]
    b, lq, lk, h, hk, d = (c["nseq"], s["longest_q"], s["longest_k"], c["heads"], c["kv_heads"],
                           c["dim"])
    dev = s["q"].device
    i, j = torch.arange(lq, device=dev), torch.arange(lk, device=dev)
    q_in, k_in = i < s["nq"][:, None], j < s["nk"][:, None]  # [b, lq], [b, lk]
    if c["padded"]:
        q, k, v = (x.reshape(b, -1, x.shape[1], d).float() for x in (s["q"], s["k"], s["v"]))
        docs = s["docs"].reshape(b, lk) if s["docs"] is not None else None
    else:
        at_q = (s["cu_q"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
        at_k = (s["cu_k"][:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
        q, k, v = s["q"][at_q].float(), s["k"][at_k].float(), s["v"][at_k].float()
        docs = s["docs"][at_k] if s["docs"] is not None else None
    z = q.view(b, lq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d) @ k.permute(
        0, 2, 3, 1)
    z = z.view(b, h, lq, lk) * d ** -0.5
    if c["cap"]:
        z = c["cap"] * torch.tanh(z / c["cap"])
    p = (i + (s["nk"] - s["nq"])[:, None])[:, :, None]  # the queries' positions, [b, lq, 1]
    if c["bias"] == "slopes":
        z = z - s["slopes"][:, None, None] * (p - j).abs()[:, None]
    elif c["bias"] == "table":
        z = z + s["table"][:, (j - p).clamp(-c["reach"], c["reach"]) + c["reach"]].transpose(0, 1)
    seen = torch.ones((b, lq, lk), dtype=torch.bool, device=dev)
    if c["causal"]:
        seen = seen & (j <= p)
    if c["left"] >= 0:
        seen = seen & (p - j <= c["left"])
    if c["right"] >= 0:
        seen = seen & (j - p <= c["right"])
    if s["prefix"] is not None:
        seen = seen | (j < s["prefix"][:, None, None])
    seen = seen & k_in[:, None, :] & q_in[:, :, None]
    if docs is not None:
        seen = seen & (docs[:, :lq, None] == docs[:, None, :]) & (docs[:, :lq, None] >= 0)
    z = torch.where(seen[:, None], z, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    e = (e / torch.where(total > 0, total, 1.0)).view(b, hk, -1, lk)
    out = (e @ v.transpose(1, 2)).view(b, h, lq, d).transpose(1, 2)
    if c["padded"]:
        return out.reshape(-1, h, d).to(s["q"].dtype)
    rows = torch.arange(s["q"].shape[0], device=dev)
    seq = torch.searchsorted(s["cu_q"], rows, right=True) - 1
    return out[seq, rows - s["cu_q"][seq]].to(s["q"].dtype)


def _plain_linear(s):
    c = s["case"]
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["act"] == "relu":
        y = torch.where(y > 0, y, 0.0)
    elif c["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif c["act"] == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif c["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["out"].dtype)


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


def _own_rotary(s):
    rt, types = _runtime()
    c, q, k = s["case"], s["q"], s["k"]
    rt.rotary_device(
        q.data_ptr(), k.data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr(),
        tokens=c["tokens"], heads=c["heads"], kv_heads=c["kv_heads"], dim=c["dim"],
        inv_freq=s["freq"].data_ptr(), rot_dim=c["rot"], interleaved=c["interleaved"],
        amplitude=s["amplitude"], positions=_ptr(s["positions"]), cu_seqlens=_ptr(s["cu"]),
        nseq=0 if s["cu"] is None else s["cu"].numel() - 1, seq=s["seq"],
        q_norm_weight=_ptr(s["qw"]), k_norm_weight=_ptr(s["kw"]), eps=1e-6,
        in_dtype=types[q.dtype], out_dtype=types[q.dtype], q_strides=q.stride()[:2],
        k_strides=k.stride()[:2], stream=_stream())
    return s["q_out"], s["k_out"]


def _own_attend(s):
    rt, types = _runtime()
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    at = ({"q_lengths": s["nq"].data_ptr(), "k_lengths": s["nk"].data_ptr()} if c["padded"] else
          {"cu_q": s["cu_q"].data_ptr(), "cu_k": s["cu_k"].data_ptr()})
    rt.attention_scored_device(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), s["out"].data_ptr(), **at, nseq=c["nseq"],
        rows_q=q.shape[0], rows_k=k.shape[0], max_q=s["longest_q"], max_k=s["longest_k"],
        heads=c["heads"], kv_heads=c["kv_heads"], dim=c["dim"], in_dtype=types[q.dtype],
        out_dtype=types[q.dtype], causal=c["causal"], window=(c["left"], c["right"]),
        softcap=c["cap"], slopes=_ptr(s["slopes"]), distance_bias=_ptr(s["table"]),
        reach=c["reach"], prefix=_ptr(s["prefix"]), q_docs=_ptr(s["docs"]),
        k_docs=_ptr(s["docs"]), q_strides=q.stride()[:2], k_strides=k.stride()[:2],
        v_strides=v.stride()[:2], stream=_stream())
    return s["out"]


def _own_linear(s):
    rt, types = _runtime()
    c, res = s["case"], s["residual"]
    rt.linear_fused_device(
        s["x"].data_ptr(), s["w"].data_ptr(), s["out"].data_ptr(), m=c["m"], n=c["n"], k=c["k"],
        ldx=s["x"].stride(0), ldw=s["w"].stride(0), bias=_ptr(s["bias"]), activation=c["act"],
        residual=_ptr(res), residual_dtype=types[res.dtype] if res is not None else types[
            torch.float32], out_dtype=types[s["out"].dtype], stream=_stream())
    return s["out"]


def run(state):
    form = {"rotary": (_plain_rotary, _own_rotary), "attend": (_plain_attend, _own_attend),
            "linear": (_plain_linear, _own_linear)}[state["case"]["op"]][1 if own else 0]
    return form(state)


# ---- the definitions in 64 bits -------------------------------------------------------------
def _exact_rotary(c, s):
    r = c["rot"]
    if s["positions"] is not None:
        pos = s["positions"].cpu().numpy().astype(np.int64)
    elif s["cu"] is not None:
        cu = s["cu"].cpu().numpy().astype(np.int64)
        pos = np.arange(c["tokens"]) - np.repeat(cu[:-1], np.diff(cu))
    else:
        pos = np.arange(c["tokens"]) % s["seq"]
    # The angle is by definition the fp32 product of position and frequency.
    angle = (pos.astype(np.float32)[:, None] * s["freq"].cpu().numpy()[None]).astype(np.float64)
    turn = torch.polar(torch.full(angle.shape, s["amplitude"], dtype=torch.float64),
                       torch.from_numpy(angle)).to(DEV)[:, None]

    def one(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / c["dim"] + 1e-6) * w.double()
        y = y.clone()
        first = slice(0, r, 2) if c["interleaved"] else slice(0, r // 2)
        second = slice(1, r, 2) if c["interleaved"] else slice(r // 2, r)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return one(s["q"], s["qw"]), one(s["k"], s["kw"])


def _exact_attend(c, s):
    nk, nq, prefix, docs = _attend_shape(c)
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    q0 = k0 = 0
    for b in range(c["nseq"]):
        if c["padded"]:
            q0, k0 = b * s["longest_q"], b * s["longest_k"]
        n, t = int(nk[b]), int(nq[b])
        p = torch.arange(n - t, n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None]
        shut = torch.zeros((t, n), dtype=torch.bool, device=DEV)
        if c["causal"]:
            shut |= j > p
        if c["left"] >= 0:
            shut |= j < p - c["left"]
        if c["right"] >= 0:
            shut |= j > p + c["right"]
        if prefix is not None:
            shut &= j >= int(prefix[b])
        if docs is not None:
            ids = torch.from_numpy(docs[b].astype(np.int64)).to(DEV)
            shut |= (ids[n - t:, None] != ids[None]) | (ids[None] < 0)
        for h in range(c["heads"]):
            z = s["q"][q0:q0 + t, h].double() @ s["k"][k0:k0 + n, h // group].double().t()
            z /= math.sqrt(c["dim"])
            if c["cap"]:
                z = torch.tanh(z / c["cap"]) * c["cap"]
            if c["bias"] == "slopes":
                z -= s["slopes"][h].double() * (p - j).abs()
            elif c["bias"] == "table":
                z += s["table"][h].double()[torch.clamp(j - p, -c["reach"], c["reach"])
                                            + c["reach"]]
            z.masked_fill_(shut, -math.inf)
            a = torch.softmax(z, -1)
            a.masked_fill_(shut, 0.0)  # a row with nothing open is zeros
            out[q0:q0 + t, h] = a @ s["v"][k0:k0 + n, h // group].double()
        q0, k0 = q0 + t, k0 + n
    return out


def _exact_linear(c, s):
    y = s["x"].double() @ s["w"].double().t()
    if s["bias"] is not None:
        y += s["bias"].double()
    if c["act"] == "relu":
        y.clamp_(min=0)
    elif c["act"] == "gelu":
        y *= torch.special.ndtr(y)
    elif c["act"] == "gelu_tanh":
        # (1 + tanh u) / 2 is the logistic function of 2u
        y *= torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    elif c["act"] == "silu":
        y *= torch.sigmoid(y)
    if s["residual"] is not None:
        y += s["residual"].double()
    return y


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    return {"rotary": _exact_rotary, "attend": _exact_attend,
            "linear": _exact_linear}[c["op"]](c, s)
