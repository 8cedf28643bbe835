"""The head loss and AdamW in the step runtime: memory, the layers before the head, data parallel shares."""
import ctypes

import numpy as np
import pytest

from gotensor import model as gm
from gotensor._lib import check
from gpu_common import cuda_backend

pytestmark = pytest.mark.gpu


def used():
    be, n, reserved = cuda_backend(), ctypes.c_uint64(), ctypes.c_uint64()
    be.Sync()
    check(be.lib.gt_pool_usage(be.ctx.ptr, ctypes.byref(n), ctypes.byref(reserved)))
    return n.value


def test_switching_the_head_on_releases_the_logits():
    """4096 x 5000 logits, 80 MB: held by an evaluation and by the separate loss, not by the fused head."""
    m = gm.Model([gm.Linear(16, 5000)], [4096, 16])
    m.fused_head()
    lean = used()
    for _ in range(3):
        m.forward()
        assert used() >= lean + 4096 * 5000 * 4
        m.fused_head(False)
        m.fused_head()
        assert used() <= lean + (1 << 20)

