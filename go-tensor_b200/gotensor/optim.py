"""AdamW over many tensors in one launch (``gt_adamw_*``, include/gt_cuda.h)."""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Any

from . import _lib
from ._lib import FLOAT32, STATE_E4M3, STATE_NATIVE, AdamCfg, AdamwTensor, check
from .backend import Context
from .loss import address

BLOCK = 256  # values that share a scale of an 8-bit state


@dataclass
class Tensor:
    """One parameter tensor of ``n`` values: device addresses or storages of the parameters, gradients and states
    (codes and scales for 8-bit states), and its factors on the learning rate and the weight decay."""
    p: Any
    g: Any
    m: Any
    v: Any
    n: int
    m_scale: Any = None
    v_scale: Any = None
    lr_mul: float = 1.0
    wd_mul: float = 1.0


class AdamW:
    """``step`` is the address of the device's int64 step counter; ``state`` STATE_NATIVE or STATE_E4M3 (8 bits, with
    stochastic rounding from ``seed``). The buffers stay the caller's and have to outlive the optimizer's use."""

    def __init__(self, tensors, *, step, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01,
                 state=STATE_NATIVE, seed=0, dtype=FLOAT32, device=0):
        self.ptr = None
        self.ctx = Context.get(device)
        self.lib = self.ctx.lib
        self.cfg = AdamCfg(lr, beta1, beta2, eps, weight_decay)
        self.tensors = list(tensors)  # keeps the storages alive
        arr = (AdamwTensor * max(1, len(self.tensors)))()
        for a, t in zip(arr, self.tensors):
            a.p, a.g = self._at(t.p, t.n, dtype, "p"), self._at(t.g, t.n, dtype, "g")
            if state == STATE_E4M3:  # codes: a byte each, in a storage of any dtype
                a.m, a.v = self._at(t.m, t.n, None, "m", size=1), self._at(t.v, t.n, None, "v", size=1)
            else:
                a.m, a.v = self._at(t.m, t.n, dtype, "m"), self._at(t.v, t.n, dtype, "v")
            a.m_scale = self._at(t.m_scale, -(-t.n // BLOCK), FLOAT32, "m_scale")
            a.v_scale = self._at(t.v_scale, -(-t.n // BLOCK), FLOAT32, "v_scale")
            a.n, a.lr_mul, a.wd_mul = t.n, t.lr_mul, t.wd_mul
        self._step = step
        self.dtype = dtype
        self._clip = None
        p = ctypes.c_void_p()
        check(self.lib.gt_adamw_new(self.ctx.ptr, dtype, state, arr, len(self.tensors),
                                    self._at(step, 1, None, "step", size=8), seed, ctypes.byref(p)))
        self.ptr = p

    def _at(self, buf, n, dt, what, size=None):
        return address(buf, self.ctx, n, dt, what, size)

    def close(self):
        """Frees the handle (not while the stream is captured)."""
        if self.ptr:
            check(self.lib.gt_adamw_free(self.ptr))
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter shutdown
            pass

    def set_grads(self, grads):
        """New gradient buffers, one per tensor, for every later call."""
        grads = list(grads)
        if len(grads) != len(self.tensors):
            raise ValueError(f"{len(grads)} gradients for {len(self.tensors)} tensors")
        arr = (ctypes.c_void_p * max(1, len(grads)))(
            *[self._at(g, t.n, self.dtype, "g") for g, t in zip(grads, self.tensors)])
        check(self.lib.gt_adamw_set_grads(self.ptr, arr, len(grads)))
        for t, g in zip(self.tensors, grads):
            t.g = g

    def clip_grad_norm(self, max_norm, out):
        """Writes the gradients' global norm and the coefficient min(1, max_norm / norm) to the two doubles at the
        device address ``out``; the next ``step`` multiplies the gradients by it."""
        check(self.lib.gt_adamw_clip(self.ptr, max_norm, self._at(out, 2, _lib.FLOAT64, "out")))
        self._clip = out  # (a storage stays alive until the step)

    def step(self, lr=None, lr_device=None):
        """One update; ``lr`` replaces the learning rate from here on, ``lr_device`` is a device double that
        replaces it for this call (and for the replays of a graph that captured it). A refused call changes
        nothing: the clipping before it goes to the next."""
        cfg = self.cfg
        if lr is not None:
            cfg = AdamCfg(lr, cfg.beta1, cfg.beta2, cfg.eps, cfg.weight_decay)
        check(self.lib.gt_adamw_step(self.ptr, ctypes.byref(cfg), self._at(self._clip, 2, _lib.FLOAT64, "out"),
                                     self._at(lr_device, 1, _lib.FLOAT64, "lr_device")))
        self.cfg, self._clip = cfg, None
