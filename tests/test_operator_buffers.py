"""What the Python side of the head loss and AdamW checks of storages before it passes their addresses on (no GPU
needed: the storages are addresses that are never read, and a call that passes reaches the missing context)."""
from types import SimpleNamespace

import pytest

from gotensor import _lib, loss, optim
from gotensor._lib import FLOAT32, FLOAT64, GTError, STATE_E4M3
from gotensor.backend import Context, CudaStorage


@pytest.fixture
def contexts(monkeypatch):
    made = [SimpleNamespace(lib=_lib.cuda_lib(), ptr=None, index=i) for i in range(2)]
    monkeypatch.setattr(Context, "get", classmethod(lambda cls, index=0: made[index]))
    return made


class Places:
    def __init__(self, contexts):
        self.contexts, self.next = contexts, 1 << 32

    def __call__(self, n, dt=FLOAT32, device=0):
        s = CudaStorage.__new__(CudaStorage)
        s.ctx, s.n, s.dt, s.ptr = self.contexts[device], n, dt, self.next
        self.next += 1 << 24
        return s


@pytest.fixture
def place(contexts):
    return Places(contexts)


def head(place, device=0, **kw):
    a = dict(x=place(32), w=place(128), bias=place(16), labels=place(4), loss=place(1), rows=place(4), dx=place(32),
             dw=place(128), db=place(16), bad_label=place(1))
    a.update(kw)
    args = [a.pop(k) for k in ("x", "w", "bias", "labels")]
    loss.linear_cross_entropy(*args, 4, 8, 16, device=device, **a)


def test_head_storages_that_fit(place):
    with pytest.raises(GTError, match="null context"):
        head(place)
    with pytest.raises(GTError, match="null context"):
        head(place, labels=place(2, FLOAT64))


@pytest.mark.parametrize("name", ["x", "w", "bias", "labels", "loss", "rows", "dx", "dw", "db", "bad_label"])
def test_head_storages_of_another_device(place, name):
    n = {"x": 32, "w": 128, "bias": 16, "labels": 4, "loss": 1, "rows": 4, "dx": 32, "dw": 128, "db": 16, "bad_label": 1}
    with pytest.raises(TypeError, match="not on cuda:0"):
        head(place, **{name: place(n[name], device=1)})


@pytest.mark.parametrize("name,n", [("x", 31), ("w", 127), ("bias", 15), ("labels", 3), ("loss", 0), ("rows", 3),
                                    ("dx", 31), ("dw", 127), ("db", 15), ("bad_label", 0)])
def test_head_storages_too_short(place, name, n):
    with pytest.raises(ValueError, match=name):
        head(place, **{name: place(n)})


def adamw(place, n=300, state=0, step=0x8000, **kw):
    held = -(-n // 4) if state == STATE_E4M3 else n
    t = dict(p=place(n), g=place(n), m=place(held), v=place(held), m_scale=place(2), v_scale=place(2), n=n)
    t.update(kw)
    optim.AdamW([optim.Tensor(**t)], step=step, state=state)


@pytest.mark.parametrize("state", [0, STATE_E4M3])
def test_adamw_storages_that_fit(place, state):
    with pytest.raises(GTError, match="null context"):
        adamw(place, state=state)


@pytest.mark.parametrize("state", [0, STATE_E4M3])
@pytest.mark.parametrize("name,n", [("p", 299), ("g", 299), ("m", 74), ("v", 74), ("m_scale", 1), ("v_scale", 1)])
def test_adamw_storages_too_short(place, state, name, n):
    """Codes are a byte each: 300 of them need 75 float32."""
    with pytest.raises(ValueError, match=name):
        adamw(place, state=state, **{name: place(n)})


@pytest.mark.parametrize("name", ["p", "g", "m", "v", "m_scale", "v_scale", "step"])
def test_adamw_storages_of_another_device(place, name):
    other = place(300, FLOAT32, device=1)
    with pytest.raises(TypeError, match="not on cuda:0"):
        adamw(place, **{name: other})


class Calls:
    """A library that refuses what `refuse` names and counts the rest."""

    def __init__(self):
        self.refuse, self.seen = set(), []

    def __getattr__(self, name):
        def call(*args):
            self.seen.append((name, args))
            if name not in self.refuse:
                return None
            lib = _lib.cuda_lib()
            return lib.gt_adamw_free(None) or lib.gt_adamw_clip(None, 1.0, 16)
        return call


def test_a_refused_call_changes_nothing(place, contexts):
    contexts[0].lib = lib = Calls()
    t = optim.Tensor(p=place(300), g=place(300), m=place(300), v=place(300), n=300)
    opt = optim.AdamW([t], step=0x8000, lr=0.5)
    opt.ptr = 7
    clip = place(2, FLOAT64)
    opt.clip_grad_norm(1.0, clip)
    lib.refuse = {"gt_adamw_step"}
    with pytest.raises(GTError):
        opt.step(lr=0.25)
    lib.refuse = set()
    opt.step()
    name, args = lib.seen[-1]
    assert name == "gt_adamw_step" and args[2] == clip.ptr and args[1]._obj.lr == 0.5
    opt.step(lr=0.125)
    assert lib.seen[-1][1][2] is None and lib.seen[-1][1][1]._obj.lr == 0.125
    lib.refuse = {"gt_adamw_free"}
    with pytest.raises(GTError):
        opt.close()
    lib.refuse = set()
    opt.close()
    assert lib.seen[-1] == ("gt_adamw_free", (7,)) and opt.ptr is None


X, W, B, Y, LOSS, ROWS, DX, DW, DB, BAD, OVER = (0x10000000 * (i + 1) for i in range(11))


@pytest.mark.parametrize("kw,message", [
    ({}, "null context"), ({"over": None}, "over: null"), ({"over": OVER + 4}, "over: a pointer is not aligned"),
    ({"over": LOSS}, "over: an output overlaps an input"), ({"over": DW + 8}, "overlaps an input"),
    ({"x": None}, "over: null"), ({"M": 0}, "over: M, K and V")])
def test_head_over_refuses(kw, message):
    a = dict(x=X, M=4, over=OVER)
    a.update(kw)
    with pytest.raises(GTError, match=message):
        _lib.check(_lib.cuda_lib().gt_linear_xent_fwd_bwd_over(None, 0, a["x"], W, B, Y, a["M"], 8, 16, -100, 0,
                                                               a["over"], LOSS, ROWS, DX, DW, DB, BAD))


@pytest.mark.parametrize("labels,n,count,message", [(Y, 4, LOSS, "null context"), (None, 4, LOSS, "null"),
                                                    (Y, 4, None, "null"), (Y, -1, LOSS, "negative"),
                                                    (Y + 2, 4, LOSS, "aligned"), (Y, 4, LOSS + 4, "aligned")])
def test_count_labels_refuses(labels, n, count, message):
    with pytest.raises(GTError, match=message):
        _lib.check(_lib.cuda_lib().gt_count_labels(None, labels, n, -100, count))


def test_over_has_to_be_a_double_of_this_device(place):
    with pytest.raises(TypeError, match="over"):
        head(place, over=place(1, FLOAT32))
    with pytest.raises(TypeError, match="not on"):
        head(place, over=place(1, FLOAT64, device=1))
    with pytest.raises(GTError, match="null context"):
        head(place, over=place(1, FLOAT64))
