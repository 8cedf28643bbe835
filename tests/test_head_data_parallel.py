"""The fused head under data parallelism, on the CPU.

* Gloo ranks compute the formulas with unequal ignored rows, each dividing by
  the ranks' mean count, and average: loss and gradients of the whole batch.
* The step runtime, its library calls answered by a recorder (a stand-in
  for libgotensor_cuda that knows no GPU), makes the calls that do the same: the
  count, its average on the way during the forward pass, the wait, the head over that average.
"""
import os
import re
import subprocess
import sys

import numpy as np
import pytest

from gotensor import _lib
from test_dist import _init, _run

HERE = os.path.dirname(os.path.abspath(__file__))
IGN = -100


def head(x, w, y, n):
    """Loss, dw and dx of the rows, divided by n."""
    keep = y != IGN
    z = x @ w.T
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    at = np.arange(len(y))
    yy = np.where(keep, y, 0)
    loss = -(np.log(p[at, yy]) * keep).sum() / n
    p[at, yy] -= 1
    g = p * keep[:, None] / n
    return loss, g.T @ x, g @ w


def batch():
    rng = np.random.default_rng(0)
    x, w, y = rng.standard_normal((30, 8)), rng.standard_normal((11, 8)), rng.integers(0, 11, 30)
    y[10:19] = IGN  # rank 1 has one row that counts,
    y[20:] = IGN    # rank 2 none
    return x, w, y


def _rank(rank, world, port, out):
    import torch
    dist = _init(rank, world, port)
    x, w, y = (a if a.shape[0] == 11 else a[10 * rank:10 * rank + 10] for a in batch())
    counted = torch.tensor([float((y != IGN).sum())], dtype=torch.float64)
    dist.all_reduce(counted)
    loss, dw, dx = head(x, w, y, counted.item() / world)
    flat = torch.from_numpy(np.concatenate([[loss], dw.ravel()]))
    dist.all_reduce(flat)
    out.put((rank, (flat / world).numpy(), dx / world))
    dist.destroy_process_group()


def test_ranks_with_unequal_ignored_rows():
    x, w, y = batch()
    loss, dw, dx = head(x, w, y, (y != IGN).sum())
    want = np.concatenate([[loss], dw.ravel()])
    for rank, flat, dx_rows in _run(_rank, 3):
        np.testing.assert_allclose(flat, want, rtol=0, atol=1e-14)
        np.testing.assert_allclose(dx_rows, dx[10 * rank:10 * rank + 10], rtol=0, atol=1e-14)


RECORDER = """
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
typedef long long i64;
char* gt_alloc(void* c, size_t n, void** out) { *out = calloc(1, n + 16); return 0; }
char* gt_release(void* c, void* p) { free(p); return 0; }
char* gt_event_new(void* c, void** out) { *out = malloc(1); return 0; }
void gt_event_free(void* e) { free(e); }
void gt_free_error(char* e) { free(e); }
i64 gt_launch_count(void) { return 0; }
void gt_host_free(void* p) {}
char* gt_count_labels(void* c, const int* y, i64 n, int ignore, double* out) {
  printf("gt_count_labels %lld %d %p\\n", n, ignore, (void*)out); return 0; }
char* gt_allreduce_avg_async(void* c, int dtype, void* p, i64 n) {
  printf("gt_allreduce_avg_async %d %p %lld\\n", dtype, p, n); return 0; }
char* gt_linear_xent_fwd_bwd_over(void* c, int dtype, const void* x, const void* w, const void* b, const int* y, i64 M,
                                  i64 K, i64 V, int ignore, i64 ws, const double* over, void* loss, void* rows, void* dx,
                                  void* dw, void* db, int* bad) {
  printf("gt_linear_xent_fwd_bwd_over %p %d\\n", (void*)over, ignore); return 0; }
"""

DRIVER = """
import ctypes, sys
sys.path.insert(0, sys.argv[2])
from gotensor import _lib
rec = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
host = _lib.host_lib()
world, on = int(sys.argv[3]), int(sys.argv[4])
from gotensor import model as gm
layers = [gm.Linear(8, 6), gm.ReLU(), gm.Linear(6, 11)]
arr, shape, m = (_lib.Layer * 3)(*layers), (ctypes.c_int64 * 2)(10, 8), ctypes.c_void_p()
_lib.check(host.gth_model_new(ctypes.c_void_p(16), 0, arr, 3, shape, 2, ctypes.byref(m)))
_lib.check(host.gth_set_fused_head(m, on, -7))
_lib.check(host.gth_dp_init(m, 0, world, bytes(128), 1000, 1 << 20))
sys.stdout.flush()
print("START", flush=True)
_lib.check(host.gth_forward_backward(m))
ctypes.CDLL(None).fflush(None)
"""


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    at = tmp_path_factory.mktemp("recorder")
    source = RECORDER
    for name, (result, _) in _lib.CUDA_API.items():
        if not re.search(r"\b%s\(" % name, RECORDER) and result == "err":
            source += 'char* %s(void) { printf("%s\\n"); return 0; }\n' % (name, name)
    (at / "recorder.c").write_text(source)
    (at / "driver.py").write_text(DRIVER)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-w", "-o", str(at / "recorder.so"), str(at / "recorder.c")], check=True)
    return at


def calls(recorder, world, on):
    out = subprocess.run([sys.executable, str(recorder / "driver.py"), str(recorder / "recorder.so"),
                          os.path.join(os.path.dirname(HERE), "go-tensor_b200"), str(world), str(on)],
                         env=dict(os.environ, LD_PRELOAD=str(recorder / "recorder.so")), capture_output=True, text=True,
                         timeout=120)
    assert out.returncode == 0, out.stderr[-2000:]
    lines = out.stdout.splitlines()
    return [line.split() for line in lines[lines.index("START") + 1:]]


def test_runtime_counts_over_the_ranks(recorder):
    made = calls(recorder, 4, 1)
    names = [c[0] for c in made]
    count, average = names.index("gt_count_labels"), names.index("gt_allreduce_avg_async")
    forward, wait, head_call = (names.index(n) for n in ("gt_linear_fwd_bits", "gt_comm_wait", "gt_linear_xent_fwd_bwd_over"))
    assert count < average < forward < wait < head_call, names
    assert made[count][1:3] == ["10", "-7"]
    where = made[count][3]
    assert made[average][1:] == ["1", where, "1"]  # float64, the count, one value
    assert made[head_call][1:] == [where, "-7"]
    # between the average and the head's wait nothing else is on its way; the gradients follow
    assert "gt_allreduce_avg_async" not in names[average + 1:head_call]
    assert names[head_call:].count("gt_allreduce_avg_async") >= 2  # gradient buckets and the loss
    assert names.count("gt_linear_xent_fwd_bwd") == 0


def test_runtime_alone_divides_by_its_own_count(recorder):
    names = [c[0] for c in calls(recorder, 1, 1)]
    assert "gt_linear_xent_fwd_bwd" in names and not {"gt_count_labels", "gt_allreduce_avg_async"} & set(names)
    names = [c[0] for c in calls(recorder, 4, 0)]
    assert "gt_xent_fwd_bwd_db" in names and "gt_count_labels" not in names
