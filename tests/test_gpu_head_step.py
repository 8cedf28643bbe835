"""The large-vocabulary head and AdamW in the step runtime: a training step is,
bit for bit, the calls that a user would make one after another (each tested on
its own), eagerly and as a captured graph; and with float64 the fused head's
gradients are those of the separate Linear and loss (the framework's 1e-10)."""
import numpy as np
import pytest

from gotensor import _lib, model as gm, optim
from gotensor._lib import GTError, check
from gotensor.loss import linear_cross_entropy
from gpu_common import assert_bits, assert_close, cuda_backend
from test_gpu_adamw import Raw
from test_gpu_linear_xent import Ints

pytestmark = pytest.mark.gpu

NP = {0: np.float32, 1: np.float64}
B, D, H, V = 200, 48, 70, 1500
ADAM = dict(lr=2e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


def make(dt=0, act=gm.ReLU, batch=B):
    m = gm.Model([gm.Linear(D, H), act(), gm.Linear(H, V)], [batch, D], dtype=dt)
    rng = np.random.default_rng(4)
    m.set_flat_params((rng.standard_normal(m.num_params) * 0.2).astype(NP[dt]))
    return m


def batches(n, dt=0, ignored=0.2):
    rng = np.random.default_rng(7)
    out = []
    for _ in range(n):
        y = rng.integers(0, V, B)
        out.append((rng.standard_normal((B, D)).astype(NP[dt]), np.where(rng.random(B) < ignored, -100, y)))
    return out


class ByHand:
    """The same model and step out of the entry points."""

    def __init__(self, m, state, max_norm):
        be = cuda_backend()
        self.lib, self.ctx, self.max_norm = be.lib, be.ctx.ptr, max_norm
        sd = m.state_dict()
        self.p = {k: Raw(v) for k, v in sd.items()}
        self.g = {k: Raw(np.zeros_like(v)) for k, v in sd.items()}
        self.shape = {k: v.shape for k, v in sd.items()}
        f = np.float32
        self.x, self.h, self.dh = Raw(np.zeros((B, D), f)), Raw(np.zeros((B, H), f)), Raw(np.zeros((B, H), f))
        self.bits = Raw(np.zeros(((B + 31) // 32, H), np.uint32))
        self.loss, self.step_dev, self.clip = Raw(np.zeros(1, f)), Raw(np.zeros(1, np.int64)), Raw(np.zeros(2))
        code = np.uint8 if state else f
        self.m, self.v = ({k: Raw(np.zeros(a.shape, code)) for k, a in sd.items()} for _ in range(2))
        self.ms, self.vs = ({k: Raw(np.zeros(-(-a.size // 256), f)) for k, a in sd.items()} for _ in range(2))
        self.opt = optim.AdamW([optim.Tensor(p=self.p[k].ptr, g=self.g[k].ptr, m=self.m[k].ptr, v=self.v[k].ptr,
                                             n=sd[k].size, wd_mul=float(sd[k].ndim > 1), m_scale=self.ms[k].ptr,
                                             v_scale=self.vs[k].ptr) for k in sd],
                               step=self.step_dev.ptr, state=state, seed=11, **ADAM)

    def step(self, x, y):
        lib, c, p, g = self.lib, self.ctx, self.p, self.g
        self.x.set(x)
        self.y = Ints(y)
        check(lib.gt_linear_fwd_bits(c, 0, self.x.ptr, p["0.weight"].ptr, p["0.bias"].ptr, self.h.ptr, self.bits.ptr, B,
                                     D, H))
        linear_cross_entropy(self.h.ptr, p["2.weight"].ptr, p["2.bias"].ptr, self.y.ptr, B, H, V, loss=self.loss.ptr,
                             dx=self.dh.ptr, dw=g["2.weight"].ptr, db=g["2.bias"].ptr)
        check(lib.gt_act_bwd(c, 0, 1, self.dh.ptr, self.h.ptr, self.dh.ptr, B * H))
        check(lib.gt_linear_bwd_weight(c, 0, self.x.ptr, self.dh.ptr, g["0.weight"].ptr, g["0.bias"].ptr, B, D, H))
        if self.max_norm:
            self.opt.clip_grad_norm(self.max_norm, self.clip.ptr)
        self.opt.step()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("state,max_norm", [(0, 0.0), (0, 0.3), (1, 0.0), (1, 0.3)])
def test_step_is_the_calls(state, max_norm, graph):
    m = make()
    m.fused_head()
    m.adamw(state=state, max_norm=max_norm, seed=11, **ADAM)
    m.enable_graph(graph)
    hand = ByHand(m, state, max_norm)
    losses = []
    for x, y in batches(5):
        m.set_batch(x, y)
        m.train_step()
        hand.step(x, y)
        assert m.loss() == hand.loss.host()[0]
        losses.append(m.loss())
        if max_norm:
            assert m.grad_norm() == hand.clip.host()[0]
    for k, v in m.grads().items():
        assert_bits(v.reshape(-1), hand.g[k].host().reshape(-1), k)
    for k, v in m.state_dict().items():
        assert_bits(v.reshape(-1), hand.p[k].host().reshape(-1), k)
    assert len(set(losses)) == 5 and np.isfinite(losses).all()


@pytest.mark.parametrize("act", [gm.ReLU, gm.Tanh, gm.Sigmoid])
def test_fused_head_gradients_float64(act):
    x, y = batches(1, 1, ignored=0.0)[0]
    a, b = make(1, act), make(1, act)
    b.fused_head()
    for m in (a, b):
        m.set_batch(x, y)
        m.forward_backward()
    assert abs(a.loss() - b.loss()) <= 1e-10 * max(1, abs(a.loss()))
    for k, v in a.grads().items():
        assert_close(b.grads()[k], v, 1e-10, k)
        assert np.abs(v).max() > 1e-6


def test_head_alone_and_evaluation():
    """A model of one Linear (no dx); evaluation gives the same logits with the fused head as without, also between
    steps, and switching the head off gives the earlier gradients bit for bit."""
    rng = np.random.default_rng(1)
    m = gm.Model([gm.Linear(D, V)], [B, D])
    m.set_flat_params(rng.standard_normal(m.num_params).astype(np.float32) * 0.1)
    x, y = batches(1, ignored=0.0)[0]
    m.set_batch(x, y)
    m.forward_backward()
    logits, grads, loss = m.forward(), m.grads(), m.loss()
    m.fused_head()
    m.forward_backward()
    # two float32 computations of the same loss: 2^-20 of the largest logit and of the loss apart at most
    assert abs(m.loss() - loss) <= 2.0 ** -20 * (np.abs(logits).max() + abs(loss))
    assert np.array_equal(m.forward(), logits)
    m.adamw(**ADAM)
    before = m.flat_params()
    m.train_step()
    assert not np.array_equal(m.flat_params(), before)
    m.set_flat_params(before)
    assert np.array_equal(m.forward(), logits) and m.count_correct() == int((logits.argmax(1) == y).sum())
    m.fused_head(False)
    m.forward_backward()
    assert m.loss() == loss
    for k, v in grads.items():
        assert_bits(m.grads()[k].reshape(-1), v.reshape(-1), k)


def test_optimizers_can_be_exchanged():
    m = make()
    x, y = batches(1, ignored=0.0)[0]
    m.set_batch(x, y)
    for state in (0, 1, 0):
        m.adamw(state=state, **ADAM)
        for _ in range(2):
            m.train_step()
        m.sgd(0.01)
        m.train_step()
        m.adam(1e-3)
        m.train_step()
    assert np.isfinite(m.flat_params()).all()


def test_refusals():
    m = make()
    with pytest.raises(GTError, match="8-bit"):
        make(1).adamw(state=_lib.STATE_E4M3)
    with pytest.raises(GTError, match="state format"):
        m.adamw(state=5)
    with pytest.raises(GTError, match="max_norm"):
        m.adamw(max_norm=-1.0)
    with pytest.raises(GTError, match="clipping"):
        m.grad_norm()
    m.adamw()
    with pytest.raises(GTError, match="clipping"):
        m.grad_norm()
    with pytest.raises(GTError, match="end in a Linear"):
        gm.Model([gm.Linear(4, 4), gm.ReLU()], [2, 4]).fused_head()
    x, y = batches(1)[0]
    with pytest.raises(ValueError, match="label"):
        m.set_batch(x, np.full(B, -100))  # without the fused head every label is a class
    m.fused_head()
    m.set_batch(x, np.full(B, -100))
    with pytest.raises(ValueError, match="label"):
        m.set_batch(x, np.full(B, V))
