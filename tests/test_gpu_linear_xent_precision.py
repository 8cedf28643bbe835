"""What the float32 head loss keeps of small values, against the formulas in
float64: rows of x and of w far apart in size, classes that are far from
likely, and many terms per sum.

The bounds, element by element, from the inputs in float64. A value is held in
two halves of 11 bits: off by at most 2^-22 of itself, or by 2^-39 of the
largest it shares a scale with: the row, for x and w; for n G, weighted by what
it is multiplied with, 128 classes of a row (dx) or 128 rows of a class (dw).
A sum of n products: 3 * 2^-22 for the halves (the product of the two low ones is
dropped), at most 24 truncating additions of at most 2^-22 each within 128
terms, then rounded ones. exp and log: 2^-21 of their value. On the FP32 pipe (few rows)
all of this is smaller.
"""
import numpy as np
import pytest

from test_gpu_linear_xent import IGN, Head, compare, inputs

pytestmark = pytest.mark.gpu

U, SHARED, TINY = 2.0 ** -24, 2.0 ** -39, 2.0 ** -120


def c_sum(n):
    return 3 * 2.0 ** -22 + 50 * 2.0 ** -23 + (n / 128 + 1) * U


def shared(a, axis):
    """Per line along `axis`: its length times the largest value, group by group of 128."""
    at = np.arange(0, a.shape[axis], 128)
    counts = np.diff(np.append(at, a.shape[axis]))
    return np.moveaxis(np.maximum.reduceat(a, at, axis=axis), axis, -1) @ counts


def reference(x, w, b, y):
    """The outputs in float64 and the bound on each one's error."""
    keep = np.asarray(y) != IGN
    x32, w, b = np.asarray(x, np.float32), np.asarray(w, np.float32).astype(np.float64), np.asarray(b, np.float64)
    x, yk, n = x32[keep].astype(np.float64), np.asarray(y)[keep], int(keep.sum())
    M, K = x.shape
    V = w.shape[0]
    ax, aw = np.abs(x), np.abs(w)
    xm, wm = ax.max(1), aw.max(1)
    z = x @ w.T + b
    fin = np.isfinite(z)
    ez = np.where(fin, c_sum(K) * (ax @ aw.T) + 2 * SHARED * K * np.outer(xm, wm)
                  + U * (np.where(fin, np.abs(b), 0) + np.where(fin, np.abs(z), 0)), 0)
    top = z.max(1, keepdims=True)
    p = np.exp(z - top)
    s = p.sum(1, keepdims=True)
    p /= s
    at = np.arange(M)
    rows = np.log(s[:, 0]) + (top[:, 0] - z[at, yk])
    # what moves lse: the classes' own errors, weighted by their probabilities (twice: the weights move too)
    e_lse = 2 * (p * ez).sum(1) + 2.0 ** -21 + V * U / 64
    with np.errstate(invalid="ignore"):
        away = np.where(fin & (z > top - 800), np.abs(z - top), 0)
    spread = np.where(p > 0, away, 0)
    e_rows = e_lse + ez[at, yk] + 4 * U * (np.abs(rows) + np.abs(top[:, 0]))
    rho = ez + e_lse[:, None] + 4 * U * (spread + np.abs(top)) + 2.0 ** -20
    g = p.copy()
    g[at, yk] -= 1.0
    eg = np.where(rho < 1, p * np.expm1(np.minimum(rho, 1)), 1) + 4 * U * np.abs(g) + TINY
    ag = np.abs(g) + eg
    dx, dw, db = g @ w / n, g.T @ x / n, g.sum(0) / n
    tol = {"dx": (eg @ aw + c_sum(V) * (ag @ aw) + 2 * SHARED * shared(ag * wm, 1)[:, None]) / n + 4 * U * np.abs(dx),
           "dw": (eg.T @ ax + c_sum(M) * (ag.T @ ax) + 2 * SHARED * shared(ag * xm[:, None], 0)[:, None]) / n
           + 4 * U * np.abs(dw),
           "db": (eg.sum(0) + M * U * ag.sum(0)) / n}
    want = {"loss": np.array([rows.sum() / n]), "dw": dw, "db": db}
    tol["loss"] = np.array([e_rows.sum() / n + 2 * U * np.abs(rows).sum() / n])
    for k, v, e in (("rows", rows, e_rows), ("dx", dx, tol["dx"])):
        want[k], tol[k] = np.zeros((len(keep),) + v.shape[1:]), np.zeros((len(keep),) + v.shape[1:])
        want[k][keep], tol[k][keep] = v, e
    # (what float32 itself cannot hold: half its smallest value)
    return want, {k: t + 2.0 ** -149 * (1 + np.abs(want[k])) for k, t in tol.items()}


@pytest.mark.parametrize("M", [40, 140, 300])  # on the FP32 pipe and on the tensor cores
@pytest.mark.parametrize("factor", [1e4, 1e10, 1e20])
def test_one_large_row_of_x(M, factor):
    """The other rows' losses are what they are without it, and every output keeps its bound."""
    x, w, b, y = inputs(M, 64, 500, 1, 0)
    alone = Head(x, w, b, y, 0, outputs=("rows",)).call().host()["rows"]
    x[7] *= np.float32(factor)
    got = Head(x, w, b, y, 0).call().host()
    rest = np.arange(M) != 7
    assert np.array_equal(got["rows"][rest], alone[rest])
    compare(got, *reference(x, w, b, y))


@pytest.mark.parametrize("M", [40, 140, 300])
@pytest.mark.parametrize("factor", [1e4, 1e10, 1e20])
def test_large_weights_of_masked_classes(M, factor):
    """A padded vocabulary whose padding holds anything: classes masked by the bias, their rows of w far larger."""
    x, w, b, y = inputs(M, 64, 500, 2, 0)
    b[[3, 200, 450, 499]] = -np.inf
    y = np.where(np.isinf(b[y]), 1, y)
    alone = Head(x, w, b, y, 0).call().host()
    w[[3, 200, 450, 499]] *= np.float32(factor)
    got = Head(x, w, b, y, 0).call().host()
    compare(got, *reference(x, w, b, y))
    for k in ("rows", "db"):
        assert np.array_equal(got[k], alone[k]), k


@pytest.mark.parametrize("M,K,V", [(256, 64, 1000), (333, 48, 777), (1024, 64, 4000)])
@pytest.mark.parametrize("gain", [2.0, 6.0, 9.0, 12.0, 25.0])
def test_unlikely_classes(M, K, V, gain):
    """Logits of standard deviation `gain`, most labels the likeliest class: the rows of dw of classes whose
    probabilities are 2^-20 to 2^-100 keep their digits."""
    x, w, b, y = inputs(M, K, V, 3, 0, gain=gain, ignored=0.1)
    z = x.astype(np.float64) @ w.astype(np.float64).T + b
    y = np.where((np.arange(M) % 8 > 0) & (y != IGN), z.argmax(1), y)
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y))


@pytest.mark.parametrize("M", [140, 500])
@pytest.mark.parametrize("span", [20, 60, 100])
def test_rows_of_all_sizes(M, span):
    """Rows of x and of w from 2^-span to 1, in an order of their own."""
    x, w, b, y = inputs(M, 64, 900, 4, 0)
    rng = np.random.default_rng(5)
    x *= np.exp2(-span * rng.random(M))[:, None].astype(np.float32)
    w *= np.exp2(-span * rng.random(900))[:, None].astype(np.float32)
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y))


@pytest.mark.parametrize("workspace", [0, 1])
def test_far_apart_in_several_pieces(workspace):
    """Several pieces and K-splits; the unlikely classes and the large rows at once, a third of the rows ignored."""
    x, w, b, y = inputs(900, 130, 1500, 6, 0, gain=10.0, ignored=0.3)
    x[::50] *= np.float32(100)
    compare(Head(x, w, b, y, 0, workspace_bytes=workspace).call().host(), *reference(x, w, b, y))


@pytest.mark.parametrize("K", [512, 1000, 2048])
def test_truncated_sums_stay_short(K):
    """Sums of positive products, where truncation adds up: a label of weight 0 makes a row's loss the other class'
    logit. Of 24 additions within 128 terms, the s-th truncates a sum that is s / 24 of the partial one by half a unit of
    2^-23 at most on average: 6.25 * 2^-23 of the logit in all, and 2^-22 for the dropped products; the roundings are as
    often up as down (2^-24 / 10 for the mean of 300 rows)."""
    rng = np.random.default_rng(8)
    x, w = rng.uniform(1, 2, (300, K)).astype(np.float32), rng.uniform(1, 2, (2, K)).astype(np.float32)
    w[0] = 0
    got = Head(x, w, None, np.zeros(300, np.int64), 0, outputs=("rows",)).call().host()["rows"]
    z = x.astype(np.float64) @ w[1].astype(np.float64)
    off = float(((got - z) / z).mean())
    assert abs(off) <= 6.25 * 2.0 ** -23 + 2.0 ** -22 + 2.0 ** -24 / 10


@pytest.mark.parametrize("M", [1, 5, 8])
@pytest.mark.parametrize("K", [40000, 131072])
def test_long_sums_of_few_rows(M, K):
    """At most 8 rows: 32 lanes share a sum. Runs of at most 256 terms per lane, each rounded (2^-24 of what it holds by
    then: half the run's sum on average for positive products, 128 * 2^-24 at most of it in all), 5 joins of the lanes, and
    one addition per run."""
    rng = np.random.default_rng(9)
    x, w = rng.uniform(1, 2, (M, K)).astype(np.float32), rng.uniform(1, 2, (2, K)).astype(np.float32)
    x[:] = np.float32(1.9) + np.float32(2.0 ** -20)  # equal terms: the roundings of a run go the same way
    w[1] = np.float32(1.7) + np.float32(2.0 ** -21)
    w[0] = 0
    got = Head(x, w, None, np.zeros(M, np.int64), 0, outputs=("rows",)).call().host()["rows"]
    z = x.astype(np.float64) @ w[1].astype(np.float64)
    runs = -(-K // 8192)
    assert (np.abs((got - z) / z) <= (128 + 5 + runs + 1) * U).all()


@pytest.mark.parametrize("what", ["x", "w"])
@pytest.mark.parametrize("M", [140, 300])
def test_rows_of_zeros(M, what):
    """Every other row of x, or of w, is zero: they add nothing to dw, or dx, so what they carry of G may not cost the
    others' digits. The rows that are not zero are sure of their labels (their G is 2^-20 and below); those that are see
    equal logits, or the classes of zeros are the likely ones."""
    x, w, b, y = inputs(M, 64, 600, 10, 0, gain=12.0)
    if what == "x":
        z = x.astype(np.float64) @ w.astype(np.float64).T + b
        y = np.where(np.arange(M) % 2 == 0, z.argmax(1), y)
        for i in range(0, M, 2):  # far ahead of the second
            w[y[i]] += 0.5 * x[i]
        z = x.astype(np.float64) @ w.astype(np.float64).T + b
        y = np.where(np.arange(M) % 2 == 0, z.argmax(1), y)
        x[1::2] = 0
    else:
        w[1::2] = 0
        b[1::2] = 40
        b[0::2] -= 20
        y = y // 2 * 2 + 1
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y))


@pytest.mark.parametrize("factor", [1e20, 1e30, 1e36])
def test_unlikely_classes_beside_large_masked_ones(factor):
    """Far larger weights of a masked class in each group of 128; the classes that are left are 2^-20 to 2^-60 likely but
    for one in the first group, and its row of w is zero: dx is what they add."""
    x, w, b, y = inputs(200, 64, 1000, 11, 0, gain=3.0)
    w[5] = 0
    y[:] = 5
    b[:] -= 40
    b[5] = 0
    b[64::128] = -np.inf
    w[64::128] *= np.float32(factor)
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y))
