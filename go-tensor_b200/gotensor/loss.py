"""The loss of a classifier head over a large vocabulary.

``linear_cross_entropy`` is ``gt_linear_xent_fwd_bwd`` (include/gt_cuda.h): a
Linear, its softmax cross-entropy and every gradient, without keeping the
logits. Buffers are device addresses, or storages of ``gotensor.backend``
(whose lengths and dtypes are then checked). The call is queued on the
context's stream and does not wait.
"""
from __future__ import annotations

from . import _lib
from ._lib import FLOAT32, FLOAT64, check
from .backend import Context, CudaStorage


def address(buf, ctx, n=None, dt=None, what="buffer", size=None):
    """The device address of a storage or of an address, None for None. A storage has to be on ctx's device and is
    checked for n elements of dtype dt, or, with a size, for n values of that many bytes whatever its own dtype."""
    if buf is None:
        return None
    if isinstance(buf, CudaStorage):
        if buf.ctx is not ctx:
            raise TypeError(f"{what}: the storage is not on cuda:{ctx.index}")
        if size is not None and buf.nbytes < n * size:
            raise ValueError(f"{what}: {n * size} bytes wanted, the storage has {buf.nbytes}")
        if size is None and n is not None and buf.n < n:
            raise ValueError(f"{what}: {n} elements wanted, the storage has {buf.n}")
        if dt is not None and buf.dt != dt:
            raise TypeError(f"{what}: mixed dtypes")
        return buf.ptr
    return int(buf)


def linear_cross_entropy(x, w, bias, labels, M, K, V, *, loss, rows=None, dx=None, dw=None, db=None, bad_label=None,
                         ignore_label=-100, workspace_bytes=0, over=None, dtype=FLOAT32, device=0):
    """loss = mean over the rows that count of -log softmax(x w^T + bias)[label], each row's own loss in ``rows`` and
    the gradients in ``dx`` (M, K), ``dw`` (V, K) and ``db`` (V); each of the four may be None. ``labels`` and
    ``bad_label`` are addresses of int32 on the device. Rows labelled ``ignore_label`` take no part. ``over``, a
    double on the device, is what the sums are divided by in place of the number of rows that count (``count_labels``)."""
    ctx = Context.get(device)

    def at(buf, n, what):
        return address(buf, ctx, n, dtype, what)

    inputs = (ctx.ptr, dtype, at(x, M * K, "x"), at(w, V * K, "w"), at(bias, V, "bias"),
              address(labels, ctx, M, None, "labels", size=4), M, K, V, ignore_label, workspace_bytes)
    outputs = (at(loss, 1, "loss"), at(rows, M, "rows"), at(dx, M * K, "dx"), at(dw, V * K, "dw"), at(db, V, "db"),
               address(bad_label, ctx, 1, None, "bad_label", size=4))
    if over is None:
        check(ctx.lib.gt_linear_xent_fwd_bwd(*inputs, *outputs))
    else:
        check(ctx.lib.gt_linear_xent_fwd_bwd_over(*inputs, address(over, ctx, 1, FLOAT64, "over"), *outputs))


def count_labels(labels, n, *, count, ignore_label=-100, device=0):
    """count (a double on the device) = how many of the n labels are not ``ignore_label``."""
    ctx = Context.get(device)
    check(ctx.lib.gt_count_labels(ctx.ptr, address(labels, ctx, n, None, "labels", size=4), n, ignore_label,
                                  address(count, ctx, 1, FLOAT64, "count")))
