"""The head loss' memory: what a call takes from the pool at its highest, beside the documented bound."""
import ctypes
import gc

import pytest

from gpu_common import cuda_backend
from test_gpu_linear_xent import Head, compare, inputs, reference

pytestmark = pytest.mark.gpu

USED_CURRENT, USED_HIGH = 7, 8  # CUmemPool_attribute
SMALL = 1 << 20                 # buffers are rounded up to 256 bytes, the pool's blocks to some more


class Pool:
    def __init__(self):
        cuda_backend()
        self.cu, self.pool = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p()
        assert self.cu.cuDeviceGetDefaultMemPool(ctypes.byref(self.pool), 0) == 0

    def get(self, what):
        v = ctypes.c_uint64()
        assert self.cu.cuMemPoolGetAttribute(self.pool, what, ctypes.byref(v)) == 0
        return v.value

    def taken(self, call):
        """The bytes that call() had from the pool at once."""
        gc.collect()
        gc.disable()  # storages that go while this looks would count as the call's
        try:
            cuda_backend().Sync()
            zero = ctypes.c_uint64(0)
            assert self.cu.cuMemPoolSetAttribute(self.pool, USED_HIGH, ctypes.byref(zero)) == 0
            before = self.get(USED_CURRENT)
            call()
            cuda_backend().Sync()
            return self.get(USED_HIGH) - before
        finally:
            gc.enable()


def up(n, to):
    return -(-n // to) * to


def bound(M, K, V, dt, workspace):
    """include/gt_cuda.h: what is kept whatever workspace_bytes says, and the larger of it and the smallest piece."""
    if dt:
        return 8 * M + max(workspace, min(M, 128) * (8 * up(V, 2) + 8 * up(K, 2) + 16 * (V // 4096 + 1) + 8)) + SMALL
    fixed = 4 * (M + V) * up(K, 8) + 24 * M + 8 * up(V, 256)
    per_row = 8 * up(V, 128) + up(V, 128) // 128 * 24 + 12
    return fixed + max(workspace, min(M, 256) * per_row) + SMALL


@pytest.mark.parametrize("workspace", [1, 8 << 20, 64 << 20, 300 << 20, 0])
@pytest.mark.parametrize("M,K,V,dt", [(600, 512, 20000, 0), (1000, 64, 3000, 0), (100, 3000, 5000, 0),
                                      (300, 200, 40000, 1), (1000, 64, 3000, 1), (20, 1000, 9000, 1)])
def test_within_the_bound(M, K, V, dt, workspace):
    x, w, b, y = inputs(M, K, V, 1, dt, ignored=0.2)
    h = Head(x, w, b, y, dt, workspace_bytes=workspace)
    taken = Pool().taken(h.call)
    assert taken <= bound(M, K, V, dt, workspace or 2 << 30), (taken, bound(M, K, V, dt, workspace or 2 << 30))
    compare(h.host(), *reference(x, w, b, y, dt))


@pytest.mark.parametrize("M,K,V", [(1, 300, 70000), (8, 2000, 30000), (20, 512, 9000), (64, 100, 20000)])
def test_few_rows(M, K, V):
    x, w, b, y = inputs(M, K, V, 1, 0)
    taken = Pool().taken(Head(x, w, b, y, 0, workspace_bytes=1).call)
    assert taken <= 5 * M * V + V * K // 4 + (20 << 20) + SMALL
