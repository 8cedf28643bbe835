"""gt_adamw_* against AdamW in float64 (numpy), and against float32 numpy bit by bit.

Every operation of the kernel is one correctly rounded operation of the dtype
in a fixed order, so numpy's float32 arithmetic in that order gives the same
bits, 8-bit codes included. The float64 comparison bounds the roundings: m is
two products and a sum of terms with one rounding each (3 u of the terms'
magnitudes, u = eps / 2), v four, sqrt and its scaling 2 u more, and the update
is off by at most 10 u of itself plus what m's error contributes.
"""
import ctypes
import math

import numpy as np
import pytest

from gotensor import _lib, optim
from gotensor._lib import GTError, check
from gpu_common import cuda_backend

pytestmark = pytest.mark.gpu

NP = {0: np.float32, 1: np.float64}
HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


class Raw:
    """Bytes on the device, readable as any type, starting `shift` bytes into the allocation."""

    def __init__(self, a, shift=0):
        self.ctx = cuda_backend().ctx
        self.a = np.ascontiguousarray(a)
        self.base = self.ctx.alloc(self.a.nbytes + 256)
        self.ptr = self.base + shift
        self.set(self.a)

    def set(self, a):
        a = np.ascontiguousarray(a)
        check(self.ctx.lib.gt_upload(self.ctx.ptr, self.ptr, a.ctypes.data, a.nbytes))

    def host(self):
        out = np.empty_like(self.a)
        check(self.ctx.lib.gt_download(self.ctx.ptr, out.ctypes.data, self.ptr, out.nbytes))
        return out

    def __del__(self):
        self.ctx.release(self.base)


def mix(x):
    x = np.asarray(x, dtype=np.uint64) & 0xFFFFFFFF
    x ^= x >> 16
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x ^= x >> 15
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def bits32(seed, t, block0, n):
    key = mix(mix(mix(mix(seed & 0xFFFFFFFF) ^ np.uint64(seed >> 32)) ^ np.uint64(t & 0xFFFFFFFF)) ^ np.uint64(t >> 32))
    blocks = -(-n // 256)
    b = np.arange(block0, block0 + blocks, dtype=np.uint64)
    kb = mix(mix(key ^ (b & np.uint64(0xFFFFFFFF))) ^ (b >> np.uint64(32)))
    return mix(kb[:, None] + np.arange(256, dtype=np.uint64)).reshape(-1)[:n]


#: the values of the 256 codes: sign, 4 bits of exponent with bias 7, 3 of mantissa; 0x7f and 0xff are NaN
CODES = np.array([(-1.0) ** (c >> 7) * (np.nan if c & 127 == 127 else (c & 7) * 2.0 ** -9 if c & 120 == 0 else
                                        (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10)) for c in range(256)], np.float32)


def per_block(a, fn):
    return np.array([fn(a[i:i + 256]) for i in range(0, len(a), 256)], dtype=np.float32)


def encode(x, r16, positive):
    """float32, the kernel's order of roundings."""
    f = np.float32
    fine = np.isfinite(x)
    top = per_block(np.where(fine, np.abs(x), 0), np.max)
    some = top >= f(2.0 ** -100)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        scale = np.where(some, top * f(1 / 448), 0).astype(f)
        inv = np.where(some, f(448) / np.where(some, top, 1), 0).astype(f)
        y = np.minimum(np.abs(x) * np.repeat(inv, 256)[:len(x)], f(448))
    y = np.where(fine, y, 0).astype(f)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(y, 2.0 ** -30).astype(np.float64))), -6) - 3)
    yq = np.where(y < 2.0 ** -6, (y + f(2.0 ** -6)).astype(f).astype(np.float64) - 2.0 ** -6, y.astype(np.float64))
    value = np.floor(yq / step + r16 / 65536.0) * step
    table = CODES[:127].astype(np.float64)
    code = np.searchsorted(table, value)
    assert (table[code] == value).all()
    if positive:
        code = np.where((code == 0) & (y > 0), 1, code)
    return np.where(fine, code + 128 * (x < 0), 127).astype(np.uint8), scale


def step32(s, i, t, coef, seed, block0, state, dt, lr_mul, wd_mul, hyper):
    """One AdamW step of tensor s in numpy of the dtype, in the kernel's order; new p, m, v (codes and scales too)."""
    f = NP[dt]
    lr, b1, b2, eps, wd = (hyper[k] for k in ("lr", "beta1", "beta2", "eps", "weight_decay"))
    p, g = s["p"], s["g"]
    n = len(p)
    if state:
        m = CODES[s["m"]] * np.repeat(s["m_scale"], 256)[:n]
        r = CODES[s["v"]] * np.repeat(s["v_scale"], 256)[:n]
        v = r * r
    else:
        m, v = s["m"], s["v"]
    with np.errstate(invalid="ignore", over="ignore"):
        g = g * f(coef)
        m = m * f(b1) + g * f(1 - b1)
        v = v * f(b2) + (g * g) * f(1 - b2)
        r = np.sqrt(v)
        decay = f(1.0 - lr * lr_mul * (wd * wd_mul))
        upd = (m * f(lr / (1 - b1 ** t) * lr_mul)) / (r * f(1 / math.sqrt(1 - b2 ** t)) + f(eps))
        p = p * decay - upd
    out = {"p": p.astype(f)}
    if state:
        h = bits32(seed, t, block0, n)
        out["m"], out["m_scale"] = encode(m.astype(f), (h & np.uint64(0xFFFF)).astype(np.float64), False)
        out["v"], out["v_scale"] = encode(r.astype(f), (h >> np.uint64(16)).astype(np.float64), True)
    else:
        out["m"], out["v"] = m.astype(f), v.astype(f)
    return out


class Many:
    """A list of tensors on the device, mirrored on the host."""

    def __init__(self, sizes, dt=0, state=0, seed=5, shift=0, lr_mul=None, wd_mul=None, t=0, hyper=HYPER, scale=1e-3):
        rng = np.random.default_rng(sum(sizes) + len(sizes))
        f = NP[dt]
        self.dt, self.state, self.seed, self.t, self.hyper = dt, state, seed, t, hyper
        self.lr_mul, self.wd_mul = lr_mul or [1.0] * len(sizes), wd_mul or [1.0] * len(sizes)
        self.h, self.d, block = [], [], 0
        self.block0 = []
        shifts = shift if isinstance(shift, dict) else dict.fromkeys("pgmv", shift)
        for n in sizes:
            s = {"p": rng.standard_normal(n).astype(f), "g": (rng.standard_normal(n) * scale * np.exp(rng.standard_normal(n))).astype(f)}
            m, r = (rng.standard_normal(n) * 3e-4).astype(f), np.abs(rng.standard_normal(n) * 1e-3).astype(f)
            if state:
                s["m"], s["m_scale"] = encode(m, np.full(n, 32768.0), False)
                s["v"], s["v_scale"] = encode(r, np.full(n, 32768.0), True)
            else:
                s["m"], s["v"] = m, r * r
            self.h.append(s)
            self.d.append({k: Raw(a, shifts.get(k, 0)) for k, a in s.items()})
            self.block0.append(block)
            block += -(-n // 256)
        self.step = Raw(np.array([t], dtype=np.int64))
        self.clip = Raw(np.zeros(2))
        self.opt = optim.AdamW([optim.Tensor(n=n, lr_mul=a, wd_mul=b, **{k: r.ptr for k, r in d.items()})
                                for n, a, b, d in zip(sizes, self.lr_mul, self.wd_mul, self.d)],
                               step=self.step.ptr, state=state, seed=seed, dtype=dt, **hyper)

    def host_step(self, max_norm=None):
        self.t += 1
        coef = 1.0
        if max_norm is not None:
            norm = math.sqrt(sum(float((s["g"].astype(np.float64) ** 2).sum()) for s in self.h))
            coef = min(1.0, max_norm / norm)
        for i, s in enumerate(self.h):
            s.update(step32(s, i, self.t, coef, self.seed, self.block0[i], self.state, self.dt, self.lr_mul[i],
                            self.wd_mul[i], self.hyper))

    def same(self):
        for i, (s, d) in enumerate(zip(self.h, self.d)):
            for k, a in s.items():
                got = d[k].host()
                assert got.dtype == a.dtype
                nan = np.isnan(got) & np.isnan(a) if a.dtype.kind == "f" else np.zeros(len(a), bool)
                bad = (got != a) & ~nan
                assert not bad.any(), (i, k, int(bad.sum()), len(a), np.argwhere(bad)[:3].ravel().tolist(), got[bad][:3],
                                       a[bad][:3])
        assert self.step.host()[0] == self.t


SIZES = [[1], [3], [255], [256], [257], [4095, 1, 4096, 4097, 2], [5, 12289, 300, 0, 70001, 1, 8192], [31] * 40]


@pytest.mark.parametrize("state,dt", [(0, 0), (0, 1), (1, 0)])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_bits_against_numpy(state, dt, sizes):
    """Three steps; lr and decay factors of their own for each tensor."""
    k = len(sizes)
    a = Many(sizes, dt, state, lr_mul=[1.0 if i % 3 else 0.5 for i in range(k)], wd_mul=[float(i % 2) for i in range(k)])
    for _ in range(3):
        a.opt.step()
        a.host_step()
        a.same()


def test_bits_of_many_values():
    """A million and a half values with 8-bit states: the packed square roots and quotients are the rounded ones."""
    a = Many([1500007, 300000], 0, 1)
    for _ in range(3):
        a.opt.step()
        a.host_step()
        a.same()


@pytest.mark.parametrize("state,dt,shift", [(0, 0, 4), (0, 0, 12), (0, 1, 8), (1, 0, 4), (0, 0, {"g": 4}), (0, 0, {"m": 8}),
                                            (0, 1, {"p": 8}), (1, 0, {"m": 1}), (1, 0, {"v": 3, "m": 7}), (1, 0, {"g": 8})])
def test_any_alignment(state, dt, shift):
    a = Many([1, 2, 5, 4099, 8200, 300], dt, state, shift=shift)
    for _ in range(2):
        a.opt.step()
        a.host_step()
        a.same()


@pytest.mark.parametrize("dt", [0, 1])
def test_against_float64(dt):
    """From zero states over ten steps, the bound of the module's comment times the steps (errors add up)."""
    sizes, u = [1000, 33, 5000], 2.0 ** -53 if dt else 2.0 ** -24
    a = Many(sizes, dt)
    for s, d in zip(a.h, a.d):
        for k in "mv":
            s[k] = np.zeros_like(s[k])
            d[k].set(s[k])
    ref = [{k: v.astype(np.float64) for k, v in s.items()} for s in a.h]
    lr, b1, b2, eps, wd = (HYPER[k] for k in ("lr", "beta1", "beta2", "eps", "weight_decay"))
    for t in range(1, 11):
        a.opt.step()
        for s in ref:
            s["m"] = b1 * s["m"] + (1 - b1) * s["g"]
            s["v"] = b2 * s["v"] + (1 - b2) * s["g"] ** 2
            s["p"] = s["p"] * (1 - lr * wd) - lr * (s["m"] / (1 - b1 ** t)) / (np.sqrt(s["v"] / (1 - b2 ** t)) + eps)
    for s, d in zip(ref, a.d):
        for k, tol in (("m", 10 * 4 * u * np.abs(s["m"])), ("v", 10 * 6 * u * s["v"]),
                       ("p", 10 * (2 * u * np.abs(s["p"]) + 60 * u * lr * 3.2))):
            assert (np.abs(d[k].host() - s[k]) <= tol).all(), k


def test_zero_gradients_and_states():
    for state in (0, 1):
        a = Many([700, 3], 0, state)
        for s, d in zip(a.h, a.d):
            for k in s:
                if k != "p":
                    s[k] = np.zeros_like(s[k])
                    d[k].set(s[k])
        for _ in range(2):
            a.opt.step()
            a.host_step()
            a.same()
        assert all((d["m"].host() == 0).all() and (d["v"].host() == 0).all() for d in a.d)


@pytest.mark.parametrize("state", [0, 1])
def test_not_finite_gradients_stay_where_they_are(state):
    a = Many([600], 0, state)
    g = a.h[0]["g"]
    g[5], g[300], g[599] = np.nan, np.inf, -np.inf
    a.d[0]["g"].set(g)
    a.opt.step()
    a.host_step()
    a.same()
    p = a.d[0]["p"].host()
    assert np.isnan(p[[5, 300, 599]]).all() and np.isfinite(np.delete(p, [5, 300, 599])).all()
    if state:
        assert (a.d[0]["m"].host()[[5, 300, 599]] == 127).all() and np.isfinite(a.d[0]["m_scale"].host()).all()


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e18])
@pytest.mark.parametrize("state", [0, 1])
def test_extreme_gradients(state, scale):
    a = Many([1000, 257], 0, state, scale=scale)
    for _ in range(2):
        a.opt.step()
        a.host_step()
        a.same()


def test_stochastic_rounding_is_unbiased():
    """r = sqrt(v) with b2 = 0 and g = value: a code's mean over many steps is the value. The mean of n roundings between
    codes a step d apart has a standard deviation of at most d / 2 / sqrt(n), and the 16 random bits add d 2^-16."""
    n, steps = 256, 4000
    hyper = dict(lr=0.0, beta1=0.0, beta2=0.0, eps=1e-8, weight_decay=0.0)
    a = Many([n], 0, 1, hyper=hyper)
    g = np.linspace(-1, 1, n).astype(np.float32) ** 3
    a.d[0]["g"].set(g)
    sums = np.zeros(n), np.zeros(n)
    for _ in range(steps):
        a.opt.step()
        for total, k in zip(sums, "mv"):
            total += CODES[a.d[0][k].host()].astype(np.float64) * a.d[0][k + "_scale"].host()[0]
    y = np.abs(g).astype(np.float64) * 448
    gap = np.exp2(np.maximum(np.floor(np.log2(np.maximum(y, 1e-9))), -6) - 3) / 448
    for total, want in zip(sums, (g.astype(np.float64), np.abs(g).astype(np.float64))):
        ok = np.abs(total / steps - want) <= 5 * gap / 2 / math.sqrt(steps) + gap * 2.0 ** -15 + 2.0 ** -22 * np.abs(want)
        ok |= (want > 0) & (y < 2.0 ** -9) & (want == np.abs(g))  # a positive r is never stored as zero
        assert ok.all(), np.argwhere(~ok).ravel()


def test_seeds_and_steps_give_other_bits():
    codes = []
    for seed, t in ((1, 0), (2, 0), (1, 1), (1 << 32 | 1, 0), (1, 1 << 32)):
        a = Many([2000], 0, 1, seed=seed, t=t)
        a.opt.step()
        codes.append(a.d[0]["m"].host())
    for i in range(5):
        for j in range(i):
            assert (codes[i] != codes[j]).mean() > 0.05, (i, j)


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("sizes,max_norm", [([1], 1.0), ([70001, 3, 0, 4096 * 9], 1e-2), ([500, 500], 1e9), ([31] * 300, 0.0)])
def test_clipping(dt, sizes, max_norm):
    """The norm to the last bits of float64 (n terms in any order: n 2^-53), then the clipped step's bits."""
    a = Many(sizes, dt)
    a.opt.clip_grad_norm(max_norm, a.clip.ptr)
    a.opt.step()
    norm = math.sqrt(sum(float((s["g"].astype(np.float64) ** 2).sum()) for s in a.h))
    got = a.clip.host()
    assert abs(got[0] - norm) <= (sum(sizes) + 4) * 2.0 ** -53 * norm
    assert got[1] == min(1.0, max_norm / got[0])
    if dt == 0:  # (in float64 the last bits of the norm reach the states)
        a.host_step(max_norm)
        a.same()
    a.opt.step()  # the coefficient serves one step
    if dt == 0:
        a.host_step()
        a.same()


@pytest.mark.parametrize("state", [0, 1])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_norm_that_is_not_finite_skips_the_step(state, value):
    a = Many([300, 5000], 0, state)
    good = a.h[1]["g"].copy()
    bad = good.copy()
    bad[4500] = value
    a.d[1]["g"].set(bad)
    a.opt.clip_grad_norm(1.0, a.clip.ptr)
    a.opt.step()
    a.h[1]["g"] = bad
    a.same()  # nothing moved, the counter neither
    assert not np.isfinite(a.clip.host()[0]) and np.isnan(a.clip.host()[1])
    a.d[1]["g"].set(good)
    a.h[1]["g"] = good
    a.opt.clip_grad_norm(1.0, a.clip.ptr)
    a.opt.step()
    a.host_step(1.0)
    a.same()


def test_no_tensors():
    a = Many([])
    a.opt.clip_grad_norm(1.0, a.clip.ptr)
    a.opt.step()
    assert a.clip.host().tolist() == [0.0, 1.0] and a.step.host()[0] == 1


def test_new_gradient_addresses():
    a = Many([300, 4100])
    a.opt.step()
    a.host_step()
    other = [Raw(-s["g"], 4) for s in a.h]
    for s in a.h:
        s["g"] = -s["g"]
    a.opt.set_grads([r.ptr for r in other])
    for d, r in zip(a.d, other):
        d["g"] = r
    a.opt.step()
    a.host_step()
    a.same()
    with pytest.raises(GTError, match="overlaps"):
        a.opt.set_grads([a.d[0]["p"].ptr, other[1].ptr])
    with pytest.raises(ValueError, match="gradients"):
        a.opt.set_grads([other[0].ptr])
    a.opt.step()  # the refused addresses were not taken
    a.host_step()
    a.same()


@pytest.mark.parametrize("state", [0, 1])
def test_captured_and_replayed(state):
    """Each replay is a further step; the learning rate comes from the device."""
    be = cuda_backend()
    a = Many([300, 5000, 7], 0, state)
    lr = Raw(np.array([1e-3]))
    be.Sync()
    check(be.lib.gt_capture_begin(be.ctx.ptr))
    a.opt.clip_grad_norm(0.05, a.clip.ptr)
    a.opt.step(lr_device=lr.ptr)
    with pytest.raises(GTError, match="captured"):
        a.opt.set_grads([d["g"].ptr for d in a.d])
    with pytest.raises(GTError, match="captured"):
        optim.AdamW(a.opt.tensors, step=a.step.ptr, state=state)
    graph = ctypes.c_void_p()
    check(be.lib.gt_capture_end(be.ctx.ptr, ctypes.byref(graph)))
    for value in (1e-3, 5e-4, 0.0):
        lr.set(np.array([value]))
        check(be.lib.gt_graph_launch(be.ctx.ptr, graph))
        a.hyper = {**HYPER, "lr": value}
        a.host_step(0.05)
        a.same()
    be.lib.gt_graph_free(graph)


def test_values_behind_the_tensors_stay():
    """What lies before and behind each tensor in memory is not touched."""
    for state, shift in ((0, 16), (0, 20), (1, 16), (1, 20)):
        n, be = 4300, cuda_backend()
        f = np.random.default_rng(0).standard_normal(n + 64).astype(np.float32)
        c = np.random.default_rng(0).integers(0, 120, n + 64).astype(np.uint8)
        held = {k: Raw(f) for k in ("p", "g", "ms", "vs")} | {k: Raw(c if state else np.abs(f)) for k in "mv"}
        first = 32
        es = 1 if state else 4
        off = first * 4 + (shift - 16)
        step = Raw(np.zeros(1, np.int64))
        opt = optim.AdamW([optim.Tensor(p=held["p"].ptr + off, g=held["g"].ptr + off, m=held["m"].ptr + first * es,
                                        v=held["v"].ptr + first * es, n=n, m_scale=held["ms"].ptr + 128,
                                        v_scale=held["vs"].ptr + 128)], step=step.ptr, state=state)
        before = {k: r.host() for k, r in held.items()}
        opt.step()
        be.Sync()
        for k, lo, count in (("p", off // 4, n), ("m", first, n), ("v", first, n), ("ms", 32, 17 if state else 0),
                             ("vs", 32, 17 if state else 0), ("g", 0, 0)):
            after = held[k].host()
            same = after == before[k]
            same[lo:lo + count] = True
            assert same.all(), (state, shift, k, np.argwhere(~same).ravel()[:5])


@pytest.mark.parametrize("kw", [dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(eps=float("nan")),
                                dict(lr=float("inf")), dict(weight_decay=float("nan"))])
def test_refused_hyperparameters(kw):
    a = Many([10], hyper={**HYPER, **kw})
    with pytest.raises(GTError, match="must"):
        a.opt.step()
    with pytest.raises(GTError, match="max_norm"):
        a.opt.clip_grad_norm(-1.0, a.clip.ptr)
    with pytest.raises(GTError, match="aligned"):
        a.opt.clip_grad_norm(1.0, a.clip.ptr + 4)
    a.same()
