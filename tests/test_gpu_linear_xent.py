"""gt_linear_xent_fwd_bwd against the formulas in float64 (numpy).

Tolerances are bounds on the error of each output, element by element,
computed from the inputs in float64:

* A product sum of n terms in float32 from operands in two rounded halves of
  11 bits each: |error| <= c(n) * sum |a||b|, with 3 * 2^-22 for the split (each
  operand keeps all but 2^-22 of itself; the product of the two low halves,
  2^-22, is dropped) and 100 * 2^-23 + (n / 256 + 1) * 2^-24 for the sums (at most 48
  truncating additions of at most 2^-22 each within 256 terms, then rounded
  ones). What lies below 2^-40 of an operand's largest magnitude is lost.
  In float64: (n + 3) * 2^-53. Below the normal range a rounding is off by up
  to half the smallest subnormal, 2^-150 or 2^-1075, whatever the value: n of
  these for a sum of n terms.
* exp and log: 2^-21 (float32) or 2^-51 of their value.
"""
import ctypes
import math

import numpy as np
import pytest

from gotensor import _lib
from gotensor._lib import GTError, check
from gotensor.loss import linear_cross_entropy
from gpu_common import cuda_backend

pytestmark = pytest.mark.gpu

NP = {0: np.float32, 1: np.float64}
IGN = -100


class Ints:
    """int32 values on the device."""

    def __init__(self, values):
        be = cuda_backend()
        v = np.ascontiguousarray(values, dtype=np.int32)
        self.n, self.ctx = v.size, be.ctx
        self.ptr = be.ctx.alloc(max(4, v.nbytes))
        check(be.lib.gt_upload(be.ctx.ptr, self.ptr, v.ctypes.data, v.nbytes))

    def host(self):
        out = np.empty(self.n, dtype=np.int32)
        check(self.ctx.lib.gt_download(self.ctx.ptr, out.ctypes.data, self.ptr, out.nbytes))
        return out

    def __del__(self):
        self.ctx.release(self.ptr)


class Head:
    """One call's device buffers; outputs start as NaN so that what is not written shows."""

    def __init__(self, x, w, b, y, dt, outputs=("rows", "dx", "dw", "db"), **kw):
        be, t = cuda_backend(), NP[dt]
        self.M, self.K = x.shape
        self.V, self.dt, self.kw = w.shape[0], dt, kw
        up = lambda a: be.FromHost(np.ascontiguousarray(a, dtype=t).reshape(-1))  # noqa: E731
        nan = lambda n: up(np.full(n, np.nan))  # noqa: E731
        self.x, self.w, self.b, self.y = up(x), up(w), None if b is None else up(b), Ints(y)
        sizes = {"rows": self.M, "dx": self.M * self.K, "dw": self.V * self.K, "db": self.V}
        self.out = {"loss": nan(1), **{k: nan(sizes[k]) for k in outputs}}
        self.bad = Ints([0])

    def call(self):
        o = self.out
        linear_cross_entropy(self.x, self.w, self.b, self.y.ptr, self.M, self.K, self.V, loss=o["loss"],
                             rows=o.get("rows"), dx=o.get("dx"), dw=o.get("dw"), db=o.get("db"),
                             bad_label=self.bad.ptr, dtype=self.dt, **{"ignore_label": IGN, **self.kw})
        return self

    def host(self):
        shapes = {"dx": (self.M, self.K), "dw": (self.V, self.K)}
        got = {k: cuda_backend().ToHost(s) for k, s in self.out.items()}
        return {k: v.reshape(shapes.get(k, v.shape)) for k, v in got.items()}


def c_sum(n, dt):
    return (n + 3) * 2.0 ** -53 if dt else 3 * 2.0 ** -22 + 100 * 2.0 ** -23 + (n / 256 + 1) * 2.0 ** -24


def reference(x, w, b, y, dt):
    """The outputs in float64 and the bound on each one's error."""
    x, w = np.asarray(x, NP[dt]).astype(np.float64), np.asarray(w, NP[dt]).astype(np.float64)
    y = np.asarray(y)
    b = np.zeros(w.shape[0]) if b is None else np.asarray(b, NP[dt]).astype(np.float64)
    keep = y != IGN
    x = np.where(keep[:, None], x, 0.0)
    M, K = x.shape
    V, n = w.shape[0], max(1, int(keep.sum()))
    u, e = (2.0 ** -53, 2.0 ** -51) if dt else (2.0 ** -24, 2.0 ** -21)
    floor, tiny = (0.0, 0.0) if dt else (2.0 ** -40, 2.0 ** -150)
    ax, aw = np.abs(x) + floor * np.abs(x).max(initial=0), np.abs(w) + floor * np.abs(w).max(initial=0)
    z = x @ w.T + b
    fin = np.isfinite(z)
    ez = c_sum(K, dt) * (ax @ aw.T) + (0 if dt else 2 * floor) * (ax.max(initial=0) * aw.max(initial=0) * K) \
        + u * np.where(np.isfinite(b), np.abs(b), 0)
    m = z.max(1, keepdims=True)
    p = np.exp(z - m)
    s = p.sum(1, keepdims=True)
    p /= s
    yy = np.where(keep, y, 0)
    at = np.arange(M)
    zy = z[at, yy]
    rows = np.where(keep, np.log(s[:, 0]) + (m[:, 0] - zy), 0.0)
    worst = np.where(fin, ez, 0).max(1)
    # |z| where the rounding of z - m reaches p: not at masks so low that p is 0 whatever it is
    spread = np.where(fin & (z > m - 800), np.abs(z), 0).max(1)
    e_rows = np.where(keep, 2 * worst + (e + V * u / 64) + 8 * u * (spread + np.abs(rows) + 1), 0.0)
    g = p * keep[:, None]
    g[at[keep], yy[keep]] -= 1.0
    # p's relative error: its exponent's error, exp's own, the sum's, the roundings on the way to two halves
    rho = 2 * worst[:, None] + 2 * u * (spread[:, None] * 4 + 4) + 2 * e + (V / 64) * u
    eg = (p * rho + 8 * u * np.abs(g) + 2 * floor) * keep[:, None]
    g, eg = g / n, eg / n
    ag = np.abs(g) + eg
    dx, dw, db = g @ w, g.T @ x, g.sum(0)
    want = {"loss": np.array([rows.sum() / n if keep.any() else np.nan]), "rows": rows, "dx": dx, "dw": dw, "db": db}
    tol = {"loss": np.array([e_rows.sum() / n + 2 * u * np.abs(rows).sum() / n]), "rows": e_rows,
           "dx": eg @ aw + c_sum(V, dt) * (ag @ aw) + 4 * u * np.abs(dx) + V * tiny,
           "dw": eg.T @ ax + (c_sum(M, dt) + M * u / 128) * (ag.T @ ax) + 4 * u * np.abs(dw) + M * tiny,
           "db": eg.sum(0) + M * u * ag.sum(0)}
    return want, tol


def compare(got, want, tol):
    for k, v in got.items():
        g = np.asarray(v, dtype=np.float64)
        same = np.isnan(g) & np.isnan(want[k])
        same |= (g == want[k]) & ~np.isfinite(want[k])
        with np.errstate(invalid="ignore"):
            ok = same | (np.abs(g - want[k]) <= tol[k] + 1e-300)
        assert ok.all(), (k, int((~ok).sum()), ok.size, np.argwhere(~ok)[:4].tolist(), g[~ok][:4], want[k][~ok][:4],
                          np.broadcast_to(tol[k], g.shape)[~ok][:4])


def inputs(M, K, V, seed, dt, gain=2.0, bias=True, ignored=0.0):
    rng = np.random.default_rng(seed)
    t = NP[dt]
    x = rng.standard_normal((M, K)).astype(t)
    w = (rng.standard_normal((V, K)) * gain / math.sqrt(K)).astype(t)
    b = (rng.standard_normal(V) * 0.5).astype(t) if bias else None
    y = rng.integers(0, V, M)
    if ignored:
        y = np.where(rng.random(M) < ignored, IGN, y)
        y[M // 2] = V - 1  # at least one row counts
    return x, w, b, y


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("M,K,V", [(1, 1, 1), (1, 1, 2), (1, 16, 200), (2, 3, 5), (7, 96, 517), (31, 33, 255),
                                   (33, 65, 129), (64, 32, 256), (128, 64, 1000), (129, 31, 257), (257, 130, 1025),
                                   (300, 257, 2049), (513, 512, 300), (5, 1000, 4099), (1000, 8, 777), (256, 256, 256),
                                   (100, 20, 1), (100, 1, 2), (70, 3, 33), (500, 16, 7), (65, 1, 1), (66, 7, 128)])
@pytest.mark.parametrize("bias,ignored", [(True, 0.0), (False, 0.3)])
def test_against_float64(dt, M, K, V, bias, ignored):
    x, w, b, y = inputs(M, K, V, M * 7 + K * 3 + V, dt, bias=bias, ignored=ignored)
    h = Head(x, w, b, y, dt).call()
    compare(h.host(), *reference(x, w, b, y, dt))
    assert h.bad.host()[0] == 0


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("M,K,V", [(300, 40, 600), (1025, 130, 514), (129, 257, 1000)])
def test_several_pieces(dt, M, K, V):
    """A workspace of one byte: as many pieces as there can be."""
    x, w, b, y = inputs(M, K, V, 3, dt, ignored=0.2)
    compare(Head(x, w, b, y, dt, workspace_bytes=1).call().host(), *reference(x, w, b, y, dt))


# (the last three: few rows on either side of the choice between the two float32 paths)
@pytest.mark.parametrize("M,K,V", [(2048, 300, 3001), (4100, 64, 1000), (600, 2048, 5003), (40, 520, 8200),
                                   (9, 1030, 14500), (64, 100, 20000)])
def test_larger(M, K, V):
    x, w, b, y = inputs(M, K, V, 11, 0, ignored=0.1)
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y, 0))


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("outputs", [(), ("rows",), ("dx",), ("dw",), ("db",), ("dx", "db"), ("rows", "dw")])
def test_any_outputs(dt, outputs):
    x, w, b, y = inputs(200, 70, 310, 5, dt, ignored=0.1)
    got = Head(x, w, b, y, dt, outputs=outputs).call().host()
    assert set(got) == {"loss", *outputs}
    compare(got, *reference(x, w, b, y, dt))
    full = Head(x, w, b, y, dt).call().host()
    for k in got:  # the same bits, whatever else was asked for
        assert np.array_equal(got[k], full[k]), k


@pytest.mark.parametrize("dt", [0, 1])
def test_masked_classes(dt):
    """-infinity in the bias: probability and gradient exactly 0."""
    x, w, b, y = inputs(130, 48, 700, 6, dt)
    b[::3] = -np.inf
    b[512:] = -np.inf
    y = np.where(np.isinf(b[y]), 1, y)
    got = Head(x, w, b, y, dt).call().host()
    compare(got, *reference(x, w, b, y, dt))
    assert (got["db"][np.isinf(b)] == 0).all() and (got["dw"][np.isinf(b)] == 0).all()


@pytest.mark.parametrize("M", [40, 140])  # on the FP32 pipe and on the tensor cores
@pytest.mark.parametrize("dt", [0, 1])
def test_lowest_value_masks(dt, M):
    """The type's lowest value as a mask, on some classes and on all of them (then the softmax is that of equal logits)."""
    x, w, b, y = inputs(M, 32, 300, 8, dt)
    low = np.finfo(NP[dt]).min
    b[100:] = low
    y = y % 100
    compare(Head(x, w, b, y, dt).call().host(), *reference(x, w, b, y, dt))
    b[:] = low
    got = Head(x, w, b, y, dt).call().host()
    np.testing.assert_allclose(got["rows"], math.log(300), rtol=1e-6)
    np.testing.assert_allclose(got["db"].sum(), 0, atol=1e-5)


@pytest.mark.parametrize("M", [20, 150])  # on the FP32 pipe and on the tensor cores
@pytest.mark.parametrize("dt", [0, 1])
def test_label_on_a_masked_class(dt, M):
    x, w, b, y = inputs(M, 16, 90, 9, dt)
    b[7] = -np.inf
    y[:] = 3
    y[4] = 7
    got = Head(x, w, b, y, dt).call().host()
    assert np.isposinf(got["rows"][4]) and np.isposinf(got["loss"][0])
    assert np.isfinite(got["dx"]).all() and np.isfinite(got["dw"]).all() and got["db"][7] < 0


@pytest.mark.parametrize("M", [20, 150])  # on the FP32 pipe and on the tensor cores
@pytest.mark.parametrize("dt", [0, 1])
def test_every_class_masked(dt, M):
    x, w, b, y = inputs(M, 16, 300, 10, dt)
    b[:] = -np.inf
    got = Head(x, w, b, y, dt).call().host()
    for k in got:
        assert np.isnan(got[k]).all(), k


@pytest.mark.parametrize("dt", [0, 1])
def test_ignored_rows_may_hold_anything(dt):
    x, w, b, y = inputs(150, 40, 333, 12, dt, ignored=0.4)
    want, tol = reference(x, w, b, y, dt)
    drop = y == IGN
    clean = Head(x, w, b, y, dt).call().host()
    x[drop] = np.nan
    x[np.argmax(drop)] = np.inf
    got = Head(x, w, b, y, dt).call().host()
    compare(got, want, tol)
    assert (got["rows"][drop] == 0).all() and (got["dx"][drop] == 0).all()
    for k in got:
        assert np.array_equal(got[k], clean[k]), k


# Every tile of the float64 products, odd pitches (8-byte copies), K split over the SMs, rows of one and of several
# segments of 4096 classes, pieces of 128 rows.
@pytest.mark.parametrize("M,K,V,workspace", [
    (1, 1, 1, 0), (2, 1, 5000, 0), (3, 70, 20011, 0), (14, 33, 9000, 0), (16, 1000, 257, 0), (20, 100, 4096, 0),
    (30, 64, 4097, 0), (70, 129, 8193, 0), (142, 407, 3555, 0), (300, 20, 1000, 0), (1000, 40, 300, 0),
    (777, 17, 5000, 1), (129, 500, 4095, 1), (400, 31, 30, 0), (130, 2000, 2000, 0)])
@pytest.mark.parametrize("ignored", [0.0, 0.3])
def test_float64_shapes(M, K, V, workspace, ignored):
    x, w, b, y = inputs(M, K, V, M + K + V, 1, ignored=ignored)
    compare(Head(x, w, b, y, 1, workspace_bytes=workspace).call().host(), *reference(x, w, b, y, 1))
    evaluated = Head(x, w, b, y, 1, outputs=("rows",), workspace_bytes=workspace).call().host()
    full = Head(x, w, b, y, 1, workspace_bytes=workspace).call().host()
    for k in evaluated:
        assert np.array_equal(evaluated[k], full[k], equal_nan=True), k


@pytest.mark.parametrize("low", [-np.inf, np.finfo(np.float64).min])
@pytest.mark.parametrize("segment", [0, 1, 2])
def test_float64_masked_segment(segment, low):
    """All 4096 classes that a block has of a row masked: its maximum is the mask's value."""
    M, K, V = 9, 24, 2 * 4096 + 1000
    x, w, b, y = inputs(M, K, V, 31, 1)
    b[segment * 4096:(segment + 1) * 4096] = low
    y = (segment + 1) % 3 * 4096 + np.arange(M) * 100  # in the segment after it, its first class among them
    got = Head(x, w, b, y, 1).call().host()
    compare(got, *reference(x, w, b, y, 1))
    masked = slice(segment * 4096, (segment + 1) * 4096)
    assert (got["db"][masked] == 0).all() and (got["dw"][masked] == 0).all()


@pytest.mark.parametrize("at", [0, 4095, 4096, 4097, 8191, 8192, 9000])
def test_float64_label_in_any_segment(at):
    M, K, V = 5, 24, 9001
    x, w, b, _ = inputs(M, K, V, 32, 1)
    y = np.full(M, at)
    compare(Head(x, w, b, y, 1).call().host(), *reference(x, w, b, y, 1))


@pytest.mark.parametrize("value", [np.inf, np.nan])
@pytest.mark.parametrize("dt,M,K,V", [(0, 6, 70, 517), (0, 20, 70, 517), (0, 60, 33, 517), (0, 300, 70, 2049),
                                      (1, 6, 70, 517), (1, 150, 33, 517)])
def test_ignored_rows_beside_a_weight_that_is_not_finite(dt, M, K, V, value):
    """They take no part, so their dx and loss stay 0; the rows that count carry the weight's NaN."""
    x, w, b, y = inputs(M, K, V, M, dt)
    y[1::2] = IGN
    w[V // 3, K // 2] = value
    got = Head(x, w, b, y, dt).call().host()
    assert (got["dx"][1::2] == 0).all() and (got["rows"][1::2] == 0).all()
    assert np.isnan(got["dx"][0::2, K // 2]).all()
    got = Head(x, w, b, np.full(M, IGN), dt).call().host()
    for k in ("rows", "dx", "dw", "db"):
        assert (got[k] == 0).all(), k


@pytest.mark.parametrize("M,V,workspace", [(700, 2049, 1), (1500, 9000, 16 << 20), (1100, 20011, 0), (300, 260, 0)])
@pytest.mark.parametrize("which", ["half", "most", "first", "last", "one", "all but one", "a piece"])
def test_rows_that_count_anywhere(M, V, workspace, which):
    """Only the rows that count go through the products: their order, pieces without one, counts at and beside the
    multiples of 32 and 256."""
    x, w, b, y = inputs(M, 70, V, M + V, 0)
    m = np.arange(M)
    drop = {"half": np.random.default_rng(2).random(M) < 0.5, "most": np.random.default_rng(3).random(M) < 0.97,
            "first": m < M - 257, "last": m >= 256, "one": m != M // 2, "all but one": m == M - 1,
            "a piece": (m // 256) % 2 == 0}[which]
    y = np.where(drop, IGN, y)
    x[drop] = np.nan
    clean = np.where(drop[:, None], 0, x)
    h = Head(x, w, b, y, 0, workspace_bytes=workspace).call()
    compare(h.host(), *reference(clean, w, b, y, 0))


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("M,workspace", [(70, 0), (10, 0), (600, 1)])
def test_every_row_ignored(dt, M, workspace):
    x, w, b, _ = inputs(M, 16, 300, 13, dt)
    x[3] = np.nan
    h = Head(x, w, b, np.full(M, IGN), dt, workspace_bytes=workspace).call()
    got = h.host()
    assert np.isnan(got["loss"]).all() and h.bad.host()[0] == 0
    for k in ("rows", "dx", "dw", "db"):
        assert (got[k] == 0).all(), k


@pytest.mark.parametrize("M", [20, 150])  # on the FP32 pipe and on the tensor cores
@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("label", [-1, 90, 2 ** 31 - 1, -2 ** 31])
def test_label_outside(dt, label, M):
    x, w, b, y = inputs(M, 16, 90, 14, dt)
    y[5] = label
    h = Head(x, w, b, y, dt).call()
    got = h.host()
    assert h.bad.host()[0] == 1 and np.isnan(got["rows"][5]) and np.isnan(got["loss"][0])
    assert np.isfinite(np.delete(got["rows"], 5)).all()


@pytest.mark.parametrize("M", [60, 200])  # on the FP32 pipe and on the tensor cores
@pytest.mark.parametrize("dt", [0, 1])
def test_ignored_label_may_be_a_class(dt, M):
    x, w, b, y = inputs(M, 16, 90, 15, dt)
    y[::4] = 17
    want, tol = reference(x, w, b, np.where(y == 17, IGN, y), dt)
    compare(Head(x, w, b, y, dt, ignore_label=17).call().host(), want, tol)


@pytest.mark.parametrize("xs,ws", [(1e-12, 1e12), (1e8, 1e-8), (1e-30, 1.0), (2.0 ** 60, 2.0 ** -62), (1.0, 30.0),
                                   (1e-38, 1e30), (2.0 ** 100, 2.0 ** -99)])
def test_scales_of_the_operands(xs, ws):
    x, w, b, y = inputs(100, 64, 500, 16, 0)
    x, w = (x * np.float32(xs)).astype(np.float32), (w * np.float32(ws)).astype(np.float32)
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y, 0))


def test_uneven_rows():
    """A row of x a thousand times the others, rows of w from 2^-20 to 1, an all-zero row of each."""
    x, w, b, y = inputs(140, 64, 500, 17, 0)
    x[3] *= 100
    x[9] = 0
    w *= np.exp2(-np.arange(500) / 25.0)[:, None].astype(np.float32)
    w[11] = 0
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y, 0))


@pytest.mark.parametrize("M", [40, 140])
def test_all_zero_operands(M):
    x, w, b, y = inputs(M, 32, 260, 18, 0)
    compare(Head(x * 0, w, b, y, 0).call().host(), *reference(x * 0, w, b, y, 0))
    compare(Head(x, w * 0, b, y, 0).call().host(), *reference(x, w * 0, b, y, 0))


@pytest.mark.parametrize("M", [40, 140])  # on the FP32 pipe and on the tensor cores
@pytest.mark.parametrize("what", ["x", "w"])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_not_finite_in_a_row_that_counts(what, value, M):
    """The other rows' losses do not see it in x; in w every row does."""
    x, w, b, y = inputs(M, 32, 260, 19, 0)
    want, tol = reference(x, w, b, y, 0)
    (x if what == "x" else w)[6, 5] = value
    got = Head(x, w, b, y, 0).call().host()
    assert np.isnan(got["loss"][0]) or np.isinf(got["loss"][0])
    if what == "x":
        rest = np.arange(M) != 6
        assert (np.abs(got["rows"] - want["rows"])[rest] <= tol["rows"][rest]).all()
        assert (np.abs(got["dx"] - want["dx"])[rest] <= tol["dx"][rest]).all()
        assert not np.isfinite(got["rows"][6])


@pytest.mark.parametrize("dt", [0, 1])
def test_same_bits_again(dt):
    x, w, b, y = inputs(700, 200, 1500, 20, dt, ignored=0.1)
    h = Head(x, w, b, y, dt)
    first = h.call().host()
    for _ in range(3):
        again = h.call().host()
        for k in first:
            assert np.array_equal(first[k], again[k]), k


def test_gradient_against_differences():
    """float64: central differences of the loss over entries of x, w and b, step 1e-5: the remainder is the third
    derivative's h^2 / 6 ~ 2e-11 times its size (a few units), and the loss's rounding 1e-15 / h = 1e-10."""
    x, w, b, y = inputs(9, 12, 30, 21, 1, ignored=0.2)
    got = Head(x, w, b, y, 1).call().host()
    loss = lambda: float(Head(x, w, b, y, 1, outputs=()).call().host()["loss"][0])  # noqa: E731
    h = 1e-5
    for name, a, grad in (("x", x, got["dx"]), ("w", w, got["dw"]), ("b", b, got["db"])):
        for at in [tuple(i) for i in np.random.default_rng(1).integers(0, a.shape, (8, a.ndim))]:
            old = a[at]
            a[at] = old + h
            up = loss()
            a[at] = old - h
            down = loss()
            a[at] = old
            assert abs((up - down) / (2 * h) - grad[at]) < 1e-9, (name, at)


@pytest.mark.parametrize("dt", [0, 1])
def test_captured_and_replayed(dt):
    be = cuda_backend()
    x, w, b, y = inputs(260, 72, 900, 22, dt, ignored=0.1)
    h = Head(x, w, b, y, dt)
    eager = h.call().host()
    be.Sync()
    check(be.lib.gt_capture_begin(be.ctx.ptr))
    h.call()
    graph = ctypes.c_void_p()
    check(be.lib.gt_capture_end(be.ctx.ptr, ctypes.byref(graph)))
    x2 = (x * np.asarray(0.5, x.dtype)).astype(x.dtype)
    check(be.lib.gt_upload(be.ctx.ptr, h.x.ptr, x2.ctypes.data, x2.nbytes))
    check(be.lib.gt_graph_launch(be.ctx.ptr, graph))
    compare(h.host(), *reference(x2, w, b, y, dt))
    check(be.lib.gt_upload(be.ctx.ptr, h.x.ptr, x.ctypes.data, x.nbytes))
    check(be.lib.gt_graph_launch(be.ctx.ptr, graph))
    got = h.host()
    for k in got:
        assert np.array_equal(got[k], eager[k]), k
    be.lib.gt_graph_free(graph)


def test_two_calls_in_a_row_without_waiting():
    a = Head(*inputs(300, 90, 700, 23, 0), 0)
    b = Head(*inputs(130, 33, 1100, 24, 0), 0)
    alone = a.call().host(), b.call().host()
    a.call()
    b.call()
    a.call()
    for h, want in zip((a, b), alone):
        got = h.host()
        for k in got:
            assert np.array_equal(got[k], want[k]), k


@pytest.mark.parametrize("M,K,V", [(16, 30, 3336), (60, 100, 2000), (200, 64, 900), (7, 33, 500)])
def test_calls_with_other_counts_without_waiting(M, K, V):
    """Calls of one shape whose rows that count differ, one after another: they use the same workspace, and nothing of
    the call before may be read from it."""
    heads = [Head(*inputs(M, K, V, 30 + i, 0, ignored=p), 0) for i, p in enumerate((0.1, 0.8, 0.5))]
    alone = []
    for h in heads:
        alone.append(h.call().host())
    for _ in range(20):
        for h in heads:
            h.call()
    for h, want in zip(heads, alone):
        got = h.host()
        for k in got:
            assert np.array_equal(got[k], want[k]), k


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("M,K,V", [(20, 36, 300), (150, 64, 520), (300, 33, 129)])
def test_addresses_beside_16_bytes(dt, M, K, V):
    """Every operand and result one element past a 16-byte boundary, in pieces and at once; what lies around them stays."""
    from test_gpu_adamw import Raw
    t, es = NP[dt], 8 if dt else 4
    x, w, b, y = inputs(M, K, V, 27, dt, ignored=0.2)
    want, tol = reference(x, w, b, y, dt)
    be = cuda_backend()
    held = {k: Raw(np.full(a.size + 8, 7.0, t)) for k, a in (("x", x), ("w", w), ("b", b))}
    for k, a in (("x", x), ("w", w), ("b", b)):
        v = np.full(a.size + 8, 7.0, t)
        v[1:1 + a.size] = a.reshape(-1)
        held[k].set(v)
    out = {k: Raw(np.full(a.size + 8, 7.0, t)) for k, a in want.items()}
    labels = Ints(np.concatenate([[5], y]))
    for workspace in (0, 1):
        linear_cross_entropy(held["x"].ptr + es, held["w"].ptr + es, held["b"].ptr + es, labels.ptr + 4, M, K, V,
                             **{k: r.ptr + es for k, r in out.items()}, dtype=dt, workspace_bytes=workspace)
        be.Sync()
        got = {}
        for k, r in out.items():
            v = r.host()
            n = want[k].size
            assert v[0] == 7 and (v[1 + n:] == 7).all(), k
            got[k] = v[1:1 + n].reshape(want[k].shape)
        compare(got, want, tol)


def test_two_contexts_at_once():
    """Two contexts of one device (two streams) run calls at the same time; each gets its own results."""
    be = cuda_backend()
    lib = be.lib
    other = ctypes.c_void_p()
    check(lib.gt_init(0, ctypes.byref(other)))
    try:
        heads = [Head(*inputs(500, 128, 3000, 40 + i, 0, ignored=0.3 * i), 0) for i in range(2)]
        alone = [h.call().host() for h in heads]
        be.Sync()
        for _ in range(10):
            for h, ctx in zip(heads, (be.ctx.ptr, other)):
                o = h.out
                check(lib.gt_linear_xent_fwd_bwd(ctx, 0, h.x.ptr, h.w.ptr, h.b.ptr, h.y.ptr, h.M, h.K, h.V, IGN, 0,
                                                 o["loss"].ptr, o["rows"].ptr, o["dx"].ptr, o["dw"].ptr, o["db"].ptr, None))
        check(lib.gt_sync(other))
        be.Sync()
        for h, want in zip(heads, alone):
            got = h.host()
            for k in got:
                assert np.array_equal(got[k], want[k]), k
    finally:
        check(lib.gt_destroy(other))


def test_timed_out_wait_returns_an_error_and_the_context_recovers():
    """The bounded waits of the split GEMM: with the limit at 20 ms, the peer CTA of each pair withholds one arrival, so
    the MMA issuer's wait runs out and the kernel returns; gt_sync reports it, and the next call is right."""
    be = cuda_backend()
    h = Head(*inputs(300, 90, 700, 23, 0), 0)
    want = h.call().host()
    be.Sync()
    be.lib.gt_debug_set_tc_wait_limit_us(20000)
    try:
        be.lib.gt_debug_tc_withhold_arrive()
        h.call()
        with pytest.raises(GTError, match=r"split GEMM: a pipeline wait timed out \(site \d\)"):
            be.Sync()
        be.Sync()
    finally:
        be.lib.gt_debug_set_tc_wait_limit_us(0)
    got = h.call().host()
    for k in got:
        assert np.array_equal(got[k], want[k]), k


def test_storages_are_checked():
    h = Head(*inputs(8, 8, 8, 25, 0), 0)
    with pytest.raises(ValueError, match="elements"):
        linear_cross_entropy(h.x, h.w, None, h.y.ptr, 9, 8, 8, loss=h.out["loss"])
    with pytest.raises(TypeError, match="dtypes"):
        linear_cross_entropy(h.x, h.w, None, h.y.ptr, 8, 8, 8, loss=h.out["loss"], dtype=_lib.FLOAT64)
    with pytest.raises(GTError, match="overlap"):
        linear_cross_entropy(h.x, h.w, None, h.y.ptr, 8, 8, 8, loss=h.out["loss"], dx=h.x)
