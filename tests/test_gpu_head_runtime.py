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


def net(kind, dt):
    """Layers before the head of 50 classes, for a batch of 70: (layers, input shape)."""
    layers, shape = {
        "flatten": ([gm.Flatten(), gm.Linear(3 * 4 * 5, 50)], [70, 3, 4, 5]),
        "activation": ([gm.Linear(20, 30), gm.Flatten(), gm.Tanh(), gm.Linear(30, 50)], [70, 20]),
        "activation only": ([gm.ReLU(), gm.Linear(20, 50)], [70, 20]),
        "two linears": ([gm.Linear(20, 30), gm.Linear(30, 50)], [70, 20]),
        "conv": ([gm.Conv2d(2, 5, 3), gm.ReLU(), gm.Flatten(), gm.Linear(5 * 6 * 6, 50)], [70, 2, 8, 8]),
        "pool": ([gm.Conv2d(2, 5, 3), gm.ReLU(), gm.MaxPool2d(2), gm.Flatten(), gm.Linear(5 * 3 * 3, 50)], [70, 2, 8, 8]),
        "two convs": ([gm.Conv2d(2, 5, 3, padding=1), gm.ReLU(), gm.MaxPool2d(2), gm.Conv2d(5, 7, 3), gm.ReLU(),
                       gm.MaxPool2d(2), gm.Flatten(), gm.Linear(7, 50)], [70, 2, 8, 8]),
        "pool without relu": ([gm.Conv2d(2, 5, 3), gm.MaxPool2d(3, 1), gm.Flatten(), gm.Linear(5 * 4 * 4, 50)],
                              [70, 2, 8, 8]),
    }[kind]
    m = gm.Model(layers, shape, dtype=dt)
    t = [np.float32, np.float64][dt]
    m.set_flat_params((np.random.default_rng(1).standard_normal(m.num_params) * 0.3).astype(t))
    return m, shape, t


@pytest.mark.parametrize("dt,tol", [(0, 1e-4), (1, 1e-10)])
@pytest.mark.parametrize("kind", ["flatten", "activation", "activation only", "two linears", "conv", "pool", "two convs",
                                  "pool without relu"])
def test_layers_before_the_head(kind, dt, tol):
    """The framework's tolerances between its own paths: 1e-4 and 1e-10 of max(1, value); steps, evaluation between."""
    m, shape, t = net(kind, dt)
    rng = np.random.default_rng(2)
    x, y = rng.standard_normal(shape).astype(t), rng.integers(0, 50, shape[0])
    m.set_batch(x, y)
    m.forward_backward()
    want, loss, logits = m.grads(), m.loss(), m.forward()
    m.fused_head()
    m.forward_backward()
    assert abs(m.loss() - loss) <= tol * max(1, abs(loss))
    for k, v in m.grads().items():
        assert (np.abs(v - want[k]) <= tol * np.maximum(1, np.abs(want[k]))).all(), k
        assert np.abs(want[k]).max() > 1e-4, k
    assert np.array_equal(m.forward(), logits)
    before = m.flat_params()
    m.adamw(lr=1e-3, max_norm=1.0)
    m.enable_graph(True)
    losses = []
    for _ in range(6):
        m.train_step()
        losses.append(m.loss())
    assert np.isfinite(losses).all() and (m.flat_params() != before).any()


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("M,K,V", [(10, 40, 333), (30, 40, 333), (300, 40, 333), (300, 33, 9000)])
@pytest.mark.parametrize("ignored", [(0.0, 0.9, 0.3), (0.2, 1.0, 0.0), (1.0, 1.0, 0.5)])
def test_shares_of_a_batch(dt, M, K, V, ignored):
    """Three shards with unequal padding, one call each over the mean of their counts (what three ranks compute): the
    means of loss, dw and db are those of the whole batch, dx is three times its rows. The shards' bounds add up to the
    whole's; 8 roundings of the results come on top."""
    from gotensor.loss import count_labels
    from test_gpu_adamw import Raw
    from test_gpu_linear_xent import IGN, Head, Ints, compare, inputs, reference
    x, w, b, y = inputs(3 * M, K, V, 6, dt)
    drop = np.concatenate([np.random.default_rng(i).random(M) < p for i, p in enumerate(ignored)])
    y = np.where(drop, IGN, y)
    counts = []
    for i in range(3):
        n = Raw(np.full(1, -1.0))
        count_labels(Ints(y[i * M:(i + 1) * M]).ptr, M, count=n.ptr)
        cuda_backend().Sync()
        counts.append(n.host()[0])
        assert counts[-1] == (~drop[i * M:(i + 1) * M]).sum()
    over = Raw(np.array([np.mean(counts)]))
    got = [Head(x[i * M:(i + 1) * M], w, b, y[i * M:(i + 1) * M], dt, over=over.ptr).call().host() for i in range(3)]
    want, tol = reference(x, w, b, y, dt)
    u = 2.0 ** -53 if dt else 2.0 ** -24
    mean = {k: np.mean([g[k].astype(np.float64) for g in got], axis=0) for k in ("loss", "dw", "db")}
    mean["dx"] = np.concatenate([g["dx"].astype(np.float64) / 3 for g in got])
    mean["rows"] = np.concatenate([g["rows"] for g in got])
    compare(mean, want, {k: t + 8 * u * np.abs(want[k]) for k, t in tol.items()})
    for g, n in zip(got, counts):
        if n == 0:
            assert g["loss"][0] == 0 and not g["dx"].any() and not g["dw"].any() and not g["db"].any()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("state", [0, 1])
def test_learning_rate_schedule(state, graph):
    """The rate of each step, moments kept: bit for bit the operator's steps with that rate, also when the captured step
    is replayed."""
    from gpu_common import assert_bits
    from test_gpu_head_step import ADAM, ByHand, batches, make
    m = make()
    m.fused_head()
    m.adamw(state=state, max_norm=0.3, seed=11, **ADAM)
    m.enable_graph(graph)
    hand = ByHand(m, state, 0.3)
    x, y = batches(1)[0]
    m.set_batch(x, y)
    for i, lr in enumerate([None, 1e-3, 4e-3, 4e-3, 0.0, 2e-4]):
        if lr is not None:
            m.adamw_lr(lr)
            hand.opt.cfg.lr = lr
        before = m.flat_params()
        m.train_step()
        hand.step(x, y)
        for k, v in m.state_dict().items():
            assert_bits(v.reshape(-1), hand.p[k].host().reshape(-1), (i, k))
        assert (m.flat_params() != before).any() == (lr != 0.0)


def test_learning_rate_refusals():
    from gotensor._lib import GTError
    m = gm.Model([gm.Linear(4, 4)], [2, 4])
    with pytest.raises(GTError, match="needs AdamW"):
        m.adamw_lr(1e-3)
    m.adamw()
    for lr in (float("nan"), float("inf")):
        with pytest.raises(GTError, match="finite"):
            m.adamw_lr(lr)
