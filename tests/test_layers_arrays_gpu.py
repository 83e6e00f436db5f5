"""The encoder-layer operators on arrays (a B200): one after another, each given what the one before
returns, against the formulas in 64 bits; and from several threads on one runtime.

Tolerance of the former, over the whole result: q, k, the attention's output and its weights are rounded to bf16, each
by 2^-9 / sqrt(3) = 2^-9.8 of its values in the mean square.  A rounding of q or k moves scores of
variance about 1 by as much, and so the output, whose values the weights average, by no more than that;
four of them make 2^-8.8.  The gate is 2^-8."""

import threading

import numpy as np
import pytest

import tessery_b200 as tx
from oracle import layers as oracle
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits

pytestmark = pytest.mark.gpu


def test_attention_block_on_arrays(runtime):
    rng = np.random.default_rng(0)
    cu, docs = np.array([0, 130, 131, 300]), np.repeat(np.arange(10), 30).astype(np.int32)
    heads, kv_heads, dim, hidden = 4, 2, 64, 96

    def bits(*shape, scale=1.0):
        return to_bf16_bits((scale * rng.standard_normal(shape)).astype(np.float32))

    q, k, v = bits(300, heads, dim), bits(300, kv_heads, dim), bits(300, kv_heads, dim)
    qw, kw = (to_bf16_bits(1 + 0.1 * rng.standard_normal(dim).astype(np.float32)) for _ in range(2))
    w, b = bits(hidden, heads * dim, scale=(heads * dim) ** -0.5), rng.standard_normal(hidden)
    x = rng.standard_normal((300, hidden)).astype(np.float32)
    prefix = np.array([5, 0, 20])

    freq, amplitude = tx.rotary_frequencies(64, 1e4, scaling="yarn", factor=4, original=2048)
    rq, rk = tx.rotary(q, k, inv_freq=freq, amplitude=amplitude, cu_seqlens=cu, q_norm_weight=qw,
                       k_norm_weight=kw, runtime=runtime)
    a = tx.attention_scored(rq, rk, v, cu_q=cu, window=(40, -1), softcap=30.0, prefix=prefix,
                            q_docs=docs, runtime=runtime)
    y = tx.linear_fused(a.reshape(len(a), -1), w, bias=b, residual=x, out_dtype="float32",
                        runtime=runtime)

    want = np.empty((300, hidden))
    for s in range(3):
        at = slice(cu[s], cu[s + 1])
        pos = np.arange(cu[s + 1] - cu[s])
        eq, ek = (oracle.rotary(from_bf16_bits(t[at]), pos, freq, amplitude=amplitude,
                                weight=from_bf16_bits(n)) for t, n in ((q, qw), (k, kw)))
        ea = oracle.attention_scored(eq, ek, from_bf16_bits(v[at]), softcap=30.0, causal=True,
                                     window=(40, -1), prefix=int(prefix[s]), q_docs=docs[at],
                                     k_docs=docs[at])[0]
        want[at] = oracle.linear_fused(ea.reshape(len(pos), -1), from_bf16_bits(w), bias=b)
    assert np.linalg.norm(y - x - want) < 2.0**-8 * np.linalg.norm(want - b)


def test_threads_on_one_runtime(runtime):
    """Three threads, three sizes: each call's result is the one it has alone."""
    rng = np.random.default_rng(1)
    cases = []
    for n in (40, 300, 1100):
        x = to_bf16_bits(rng.standard_normal((n, 4, 64)).astype(np.float32))
        w = to_bf16_bits(rng.standard_normal((96, 256)).astype(np.float32))
        freq = tx.rotary_frequencies(64)[0]
        cases.append((
            lambda x=x: tx.attention_scored(x, x, x, cu_q=np.array([0, len(x)]), runtime=runtime),
            lambda x=x, f=freq: tx.rotary(x, x, inv_freq=f, seq=len(x), runtime=runtime)[1],
            lambda x=x, w=w: tx.linear_fused(x.reshape(len(x), -1), w, runtime=runtime)))
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
