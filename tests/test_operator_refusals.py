"""What the head-loss and AdamW entry points refuse, before any device is
touched: the argument checks come first, and a call that passes them all then
misses its context (no GPU needed; the addresses are never read)."""
import ctypes

import pytest

from gotensor import _lib
from gotensor._lib import AdamCfg, AdamwTensor, GTError, check

X, W, B, Y, LOSS, ROWS, DX, DW, DB, BAD = (0x10000000 * (i + 1) for i in range(10))


def head(dtype=0, x=X, w=W, bias=B, labels=Y, M=4, K=8, V=16, ignore=-100, ws=0, loss=LOSS, rows=ROWS, dx=DX, dw=DW,
         db=DB, bad=BAD, ctx=None):
    check(_lib.cuda_lib().gt_linear_xent_fwd_bwd(ctx, dtype, x, w, bias, labels, M, K, V, ignore, ws, loss, rows, dx,
                                                 dw, db, bad))


def test_head_valid_arguments_reach_the_context_check():
    for kw in ({}, {"bias": None}, {"rows": None}, {"dx": None, "dw": None, "db": None}, {"bad": None},
               {"dtype": 1}, {"ws": 1}, {"M": 2 ** 30 - 1, "K": 1, "V": 1, "dx": 10 ** 11, "rows": 10 ** 12, "x": 10 ** 13, "labels": 10 ** 14}):
        with pytest.raises(GTError, match="null context"):
            head(**kw)


@pytest.mark.parametrize("kw,message", [
    ({"dtype": 2}, "dtype"), ({"dtype": -1}, "dtype"), ({"x": None}, "null"), ({"w": None}, "null"),
    ({"labels": None}, "null"), ({"loss": None}, "null"), ({"M": 0}, "positive"), ({"K": 0}, "positive"),
    ({"V": 0}, "positive"), ({"M": -1}, "positive"), ({"V": 2 ** 30}, "2\\^30"), ({"M": 2 ** 40}, "2\\^30"),
    ({"M": 2 ** 29, "K": 2 ** 29}, "2\\^56"), ({"V": 2 ** 29, "K": 2 ** 29, "dtype": 1}, "2\\^56"),
    ({"ws": -1}, "negative"), ({"x": X + 2}, "aligned"), ({"labels": Y + 1}, "aligned"),
    ({"dtype": 1, "dw": DW + 4}, "aligned"), ({"dx": X}, "overlaps"), ({"dw": W + 4}, "overlaps"),
    ({"db": B}, "overlaps"), ({"loss": Y}, "overlaps"), ({"rows": LOSS}, "two outputs"),
    ({"dx": DW + 4 * 16 * 8 - 4}, "two outputs"), ({"dw": DX + 4 * 4 * 8 - 4}, "two outputs"),
    ({"bad": LOSS}, "two outputs"),
])
def test_head_refuses(kw, message):
    with pytest.raises(GTError, match=message):
        head(**kw)


def tensor(i, n=300, size=4, **kw):
    at = 0x100000000 * (i + 1)
    t = dict(p=at, g=at + 0x10000000, m=at + 0x20000000, v=at + 0x30000000, m_scale=at + 0x40000000,
             v_scale=at + 0x50000000, n=n, lr_mul=1.0, wd_mul=1.0)
    t.update(kw)
    return AdamwTensor(**t)


def new(*tensors, dtype=0, state=0, step=0x8000, count=None):
    arr = (AdamwTensor * max(1, len(tensors)))(*tensors)
    out = ctypes.c_void_p()
    check(_lib.cuda_lib().gt_adamw_new(None, dtype, state, arr, len(tensors) if count is None else count, step, 7,
                                       ctypes.byref(out)))


def test_adamw_valid_arguments_reach_the_context_check():
    a = tensor(0)
    end = a.p + 300 * 4
    for ts, kw in ((( ), {}), ((a, tensor(1)), {}), ((a,), {"dtype": 1}), ((a,), {"state": 1}),
                   ((a, tensor(1, n=0, p=None, g=None, m=None, v=None)), {}), ((a, tensor(1, p=end)), {}),
                   ((a, tensor(1, g=a.g)), {}), ((tensor(0, m_scale=None, v_scale=None),), {})):
        with pytest.raises(GTError, match="null context"):
            new(*ts, **kw)


@pytest.mark.parametrize("ts,kw,message", [
    ((tensor(0),), {"dtype": 3}, "dtype"), ((tensor(0),), {"state": 2}, "state format"),
    ((tensor(0),), {"state": 1, "dtype": 1}, "float32 only"), ((tensor(0),), {"count": -1}, "negative"),
    ((tensor(0),), {"step": None}, "null"), ((tensor(0),), {"step": 0x8004}, "aligned"),
    ((tensor(0, n=-1),), {}, "length"), ((tensor(0, p=None),), {}, "null pointer"),
    ((tensor(0, g=None),), {}, "null pointer"), ((tensor(0, v=None),), {}, "null pointer"),
    ((tensor(0, p=0x100000002),), {}, "aligned"), ((tensor(0, m=0x120000004),), {"dtype": 1}, "aligned"),
    ((tensor(0, m_scale=None),), {"state": 1}, "without scales"),
    ((tensor(0, v_scale=0x150000002),), {"state": 1}, "aligned"),
    ((tensor(0, lr_mul=float("nan")),), {}, "multiplier"), ((tensor(0, wd_mul=float("inf")),), {}, "multiplier"),
    ((tensor(0), tensor(0)), {}, "overlaps"), ((tensor(0), tensor(1, p=tensor(0).p + 299 * 4)), {}, "overlaps"),
    ((tensor(0), tensor(1, g=tensor(0).p)), {}, "overlaps"), ((tensor(0, m=tensor(0).g),), {}, "overlaps"),
    ((tensor(0), tensor(1, v=tensor(0).m_scale)), {"state": 1}, "overlaps"),
    ((tensor(0, v_scale=tensor(0).m_scale + 4),), {"state": 1}, "overlaps"),
    ((tensor(0, p=0x7ff8),), {}, "overlaps"),
])
def test_adamw_refuses(ts, kw, message):
    with pytest.raises(GTError, match=message):
        new(*ts, **kw)


def test_adamw_null_handles():
    lib = _lib.cuda_lib()
    cfg = AdamCfg(1e-3, 0.9, 0.999, 1e-8, 0.0)
    with pytest.raises(GTError, match="null"):
        check(lib.gt_adamw_step(None, ctypes.byref(cfg), None, None))
    with pytest.raises(GTError, match="null"):
        check(lib.gt_adamw_clip(None, 1.0, 16))
    with pytest.raises(GTError, match="null"):
        check(lib.gt_adamw_set_grads(None, (ctypes.c_void_p * 1)(), 1))
    check(lib.gt_adamw_free(None))
