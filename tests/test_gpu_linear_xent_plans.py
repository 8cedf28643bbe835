"""The head loss where its work is divided otherwise: outputs left out on the paths of few rows, sums in several stages,
tiles planned anew for the rows that count, K-splits, classes and rows at the tiles' borders."""
import ctypes

import numpy as np
import pytest

from gotensor._lib import check
from gpu_common import cuda_backend
from test_gpu_adamw import Raw
from test_gpu_linear_xent import IGN, Head, compare, inputs, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("outputs", [(), ("rows",), ("dx",), ("dw",), ("db",), ("dx", "db"), ("dw", "db"), ("dx", "dw"),
                                     ("rows", "dw")])
@pytest.mark.parametrize("M,K,V", [(1, 70, 310), (7, 130, 1000), (8, 64, 4200), (20, 129, 700), (33, 70, 310),
                                   (64, 128, 2049), (300, 300, 1000)])
def test_outputs_left_out(M, K, V, outputs):
    x, w, b, y = inputs(M, K, V, 5, 0, ignored=0.2)
    got = Head(x, w, b, y, 0, outputs=outputs).call().host()
    assert set(got) == {"loss", *outputs}
    compare(got, *reference(x, w, b, y, 0))
    full = Head(x, w, b, y, 0).call().host()
    for k in got:  # the same bits, whatever else was asked for
        assert np.array_equal(got[k], full[k]), k


@pytest.mark.parametrize("M", [1, 5, 8])
@pytest.mark.parametrize("K", [1024, 1025, 1153, 2556, 4096, 9000])
@pytest.mark.parametrize("V", [33, 517])
def test_few_rows_in_several_stages(M, K, V):
    x, w, b, y = inputs(M, K, V, K + V, 0, ignored=0.1 if M > 1 else 0.0)
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y, 0))


@pytest.mark.parametrize("M", [5, 20])
@pytest.mark.parametrize("K", [1024, 2556])
def test_few_rows_beside_16_bytes(M, K):
    """w, x and the results one value past a 16-byte boundary."""
    from gotensor.loss import linear_cross_entropy
    from test_gpu_linear_xent import Ints
    V = 300
    x, w, b, y = inputs(M, K, V, 3, 0, ignored=0.2)
    want, tol = reference(x, w, b, y, 0)
    held = {k: Raw(np.concatenate([[7], a.reshape(-1), [7]]).astype(np.float32)) for k, a in (("x", x), ("w", w), ("b", b))}
    out = {k: Raw(np.full(a.size + 2, 7, np.float32)) for k, a in want.items()}
    labels = Ints(y)
    linear_cross_entropy(held["x"].ptr + 4, held["w"].ptr + 4, held["b"].ptr + 4, labels.ptr, M, K, V,
                         **{k: r.ptr + 4 for k, r in out.items()})
    cuda_backend().Sync()
    got = {k: r.host() for k, r in out.items()}
    for k, v in got.items():
        assert v[0] == 7 and v[-1] == 7, k
    compare({k: v[1:-1].reshape(want[k].shape) for k, v in got.items()}, want, tol)


@pytest.mark.parametrize("ignored", [0.0, 0.05, 0.3, 0.6, 0.95])
def test_tiles_planned_again(ignored):
    """dx has 88 tiles of 256 x 256 for 74 pairs of SMs: the last round's are split along K; with fewer rows that count
    the device plans them anew, on either side of one round of tiles."""
    x, w, b, y = inputs(2600, 2048, 4000, 7, 0, ignored=ignored)
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y, 0))


@pytest.mark.parametrize("M,K,V", [(300, 70, 5003), (129, 33, 20011), (5000, 40, 200), (3000, 300, 130), (700, 1000, 700),
                                   (4097, 257, 513)])
@pytest.mark.parametrize("ignored", [0.0, 0.5, 0.97])
def test_split_sums(M, K, V, ignored):
    """dx and dw in ranges of K that start at whole groups of 128, some of them empty where few rows count."""
    x, w, b, y = inputs(M, K, V, 9, 0, ignored=ignored)
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y, 0))


@pytest.mark.parametrize("M", [65, 127, 128, 129, 160, 161, 255, 256, 257, 384, 385])
@pytest.mark.parametrize("V", [1, 31, 127, 128, 129, 255, 256, 257, 383, 385])
def test_borders_of_the_tiles(M, V):
    x, w, b, y = inputs(M, 40, V, M + V, 0)
    y[0], y[-1] = 0, V - 1
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y, 0))


@pytest.mark.parametrize("K", [1, 7, 8, 9, 1016, 1024, 1032, 1111, 2047, 2056])
def test_lengths_of_rows(K):
    x, w, b, y = inputs(100, K, 700, K, 0, ignored=0.1)
    compare(Head(x, w, b, y, 0).call().host(), *reference(x, w, b, y, 0))


@pytest.mark.parametrize("M", [5, 200])
def test_row_without_a_distribution_among_others(M):
    """x of one row is infinite: its row and what sums over it is NaN, the other rows' losses and dx are not."""
    x, w, b, y = inputs(M, 32, 400, 12, 0)
    clean = Head(x, w, b, y, 0).call().host()
    x[3, 4] = np.inf
    got = Head(x, w, b, y, 0).call().host()
    rest = np.arange(M) != 3
    assert np.array_equal(got["rows"][rest], clean["rows"][rest]) and not np.isfinite(got["rows"][3])
    assert np.array_equal(got["dx"][rest], clean["dx"][rest]) and np.isnan(got["dx"][3]).all()
    assert np.isnan(got["dw"]).all() and np.isnan(got["db"]).all()


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("M", [6, 150])
def test_over_in_a_captured_graph(dt, M):
    """The divisor is read when the graph is replayed."""
    be = cuda_backend()
    x, w, b, y = inputs(M, 40, 300, 13, dt, ignored=0.2)
    over = Raw(np.array([3.0]))
    h = Head(x, w, b, y, dt, over=over.ptr)
    h.call()
    be.Sync()
    check(be.lib.gt_capture_begin(be.ctx.ptr))
    h.call()
    graph = ctypes.c_void_p()
    check(be.lib.gt_capture_end(be.ctx.ptr, ctypes.byref(graph)))
    want, tol = reference(x, w, b, y, dt)
    n = (y != IGN).sum()
    u = 2.0 ** -53 if dt else 2.0 ** -24
    for d in (7.0, 0.5, float(n), 1e6):
        over.set(np.array([d]))
        check(be.lib.gt_graph_launch(be.ctx.ptr, graph))
        scaled = {k: v if k == "rows" else v * (n / d) for k, v in want.items()}
        compare(h.host(), scaled, {k: (t if k == "rows" else t * (n / d)) + 8 * u * np.abs(scaled[k]) for k, t in tol.items()})
    be.lib.gt_graph_free(graph)
