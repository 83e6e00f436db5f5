"""Counts and strides that do not fit the C calls are refused before any call (no GPU: a stand-in for
the library records what reaches it)."""

import pytest

from tessery_b200 import CudaRuntime, InvalidInputError


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name) or 0


class Runtime(CudaRuntime):
    def __init__(self):
        self._pointer, self._lib = 1, Recorder()

    def __del__(self):
        pass


ROTARY = dict(tokens=4, heads=2, kv_heads=1, dim=32, inv_freq=4096, cu_seqlens=4096, nseq=1)
SCORED = dict(nseq=1, rows_q=8, rows_k=8, max_q=8, max_k=8, heads=2, kv_heads=1, dim=32)
LINEAR = dict(m=4, n=8, k=16)


def rotary(rt, **kw):
    rt.rotary_device(4096, 8192, 4096, 8192, **{**ROTARY, **kw})


def scored(rt, **kw):
    rt.attention_scored_device(4096, 4096, 4096, 8192, **{**SCORED, **kw})


def linear(rt, **kw):
    rt.linear_fused_device(4096, 4096, 8192, **{**LINEAR, **kw})


COUNTS = [(rotary, n) for n in ("tokens", "heads", "kv_heads", "dim", "rot_dim", "nseq", "seq")] + [
    (scored, n) for n in (*SCORED, "reach")] + [(linear, n) for n in LINEAR]
STRIDES = [(rotary, n) for n in ("q_strides", "k_strides", "q_out_strides", "k_out_strides")] + [
    (scored, n) for n in ("q_strides", "k_strides", "v_strides")]


def refused(call, **kw):
    rt = Runtime()
    call(rt)
    assert len(rt._lib.calls) == 1
    with pytest.raises(InvalidInputError):
        call(rt, **kw)
    assert len(rt._lib.calls) == 1


@pytest.mark.parametrize("call,name", COUNTS)
@pytest.mark.parametrize("value", [-1, -2**31, 2**31, 2**32 + 4, 2**70])
def test_counts(call, name, value):
    refused(call, **{name: value})


@pytest.mark.parametrize("call,name", STRIDES)
@pytest.mark.parametrize("value", [(-64, 32), (64, -32), (2**64, 32), (64, 2**63)])
def test_strides(call, name, value):
    refused(call, **{name: value})


@pytest.mark.parametrize("name", ["ldx", "ldw", "ldr", "ldo"])
@pytest.mark.parametrize("value", [-8, 2**64])
def test_row_strides(name, value):
    refused(linear, **{name: value})


@pytest.mark.parametrize("value", [1e39, -1e39])
def test_caps_beyond_fp32(value):
    refused(scored, softcap=value)
