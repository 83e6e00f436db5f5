"""The encoder-layer operators called from several threads on one runtime (no GPU: a runtime that
keeps its buffers in host memory and lets another thread in at every step)."""

import ctypes as ct
import threading
import time

import numpy as np
import pytest

from tessery_b200.layers import attention_scored, linear_fused, rotary
from tessery_b200.workloads import from_bf16_bits, to_bf16_bits


class HostBuffer:
    def __init__(self, size):
        self.data = np.zeros(size, np.uint8)
        self.size, self.pointer = size, self.data.ctypes.data

    @property
    def device_ptr(self):
        assert self.pointer, "buffer was closed under its user"
        return self.pointer

    def write(self, a):
        ct.memmove(self.device_ptr, a.ctypes.data, a.nbytes)
        time.sleep(1e-4)


class HostRuntime:
    """What layers.py uses of a CudaRuntime; each operator is a simple stand-in."""

    def __init__(self):
        self._lock, self._lib, self._workspace, self._kept = threading.RLock(), self, {}, []

    def workspace(self, name, size):
        with self._lock:
            b = self._workspace.get(name)
            if b is None or b.size < size:
                if b is not None:
                    b.pointer = None  # closed; the memory stays for whoever still writes to it
                    self._kept.append(b)
                b = self._workspace[name] = HostBuffer(max(size, 256))
            return b

    def tx_read(self, pointer, to, size):
        assert pointer, "buffer was closed under its user"
        ct.memmove(to, pointer, size)
        return 0

    def sync(self):
        time.sleep(1e-4)

    @staticmethod
    def _at(pointer, count, dtype):
        return np.frombuffer((ct.c_uint8 * (count * np.dtype(dtype).itemsize)).from_address(pointer),
                             dtype)

    def rotary_device(self, q, k, q_out, k_out, *, tokens, heads, kv_heads, dim, **_):
        for x, out, n in ((q, q_out, heads), (k, k_out, kv_heads)):
            self._at(out, tokens * n * dim, np.float32)[:] = self._at(x, tokens * n * dim, np.float32)
            time.sleep(1e-4)

    def attention_scored_device(self, q, k, v, out, *, rows_q, rows_k, heads, kv_heads, dim, **_):
        n, m = rows_q * heads * dim, rows_k * kv_heads * dim
        self._at(out, n, np.float32)[:] = (self._at(q, n, np.float32)
                                           + self._at(k, m, np.float32).max()
                                           + self._at(v, m, np.float32).max())

    def linear_fused_device(self, x, w, out, *, m, n, k, ldx, ldw, **_):
        a, b = (from_bf16_bits(self._at(p, rows * ld, np.uint16)).reshape(rows, ld)[:, :k]
                for p, rows, ld in ((x, m, ldx), (w, n, ldw)))
        self._at(out, m * n, np.float32)[:] = (a @ b.T).ravel()


def rotary_call(rt, i, size):
    q = np.full((size, 2, 8), i, np.float32)
    got, other = rotary(q, -q, inv_freq=np.ones(4, np.float32), seq=size, runtime=rt)
    return np.array_equal(got, q) and np.array_equal(other, -q)


def attention_call(rt, i, size):
    q = np.full((size, 2, 8), i, np.float32)
    got = attention_scored(q, 2 * q, 3 * q, cu_q=np.array([0, size]), runtime=rt)
    return np.array_equal(got, 6 * q)


def linear_call(rt, i, size):
    x = to_bf16_bits(np.full((size, 8), i, np.float32))
    got = linear_fused(x, x, out_dtype="float32", runtime=rt)
    return np.array_equal(got, np.full((size, size), 8.0 * i * i, np.float32))


@pytest.mark.parametrize("call", [rotary_call, attention_call, linear_call])
def test_threads_on_one_runtime(call):
    """Each thread gets its own call's result, also while another's call replaces a buffer by a
    larger one."""
    rt, wrong = HostRuntime(), []

    def work(i):
        try:
            for size in range(4, 40, 3):
                if not call(rt, i, size + 5 * i):
                    wrong.append((i, size))
        except Exception as e:  # noqa: BLE001 - reported below
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in (1, 2, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
