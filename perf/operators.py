"""Cases of the training-tail operators for language-model-sized problems:

* ``head``: the classifier head's loss. A Linear over a large vocabulary, its
  softmax cross-entropy and all gradients, without keeping the logits.
* ``adamw``: one AdamW step over many tensors at once, the states in the
  parameters' type or in 8 bits with a scale per 256 values, optionally with
  the gradients clipped by their global norm.

``run`` computes a case in its plain form (elementary torch operations), or,
with ``own`` set, through gotensor's own operators.
"""
import math
import random

import torch

own = False

LR, BETA1, BETA2, EPS, DECAY, MAX_NORM = 1e-3, 0.9, 0.95, 1e-8, 0.1, 1.0
BLOCK = 256  # values that share one scale of an 8-bit state
START = 100  # steps already taken
IGNORE = -100
MASK32 = 0xFFFFFFFF
TYPES = {"float32": torch.float32, "float64": torch.float64}


def listed():
    return [
        # a handful of short sequences' last hidden rows: latency counts
        {"name": "head_tiny", "op": "head", "dtype": "float32", "M": 7, "K": 96, "V": 517, "bias": True, "grad": True,
         "ignored": 0.0, "masked": 0},
        # the wide MLP's own head: 8192 rows, 4096 features, 1000 classes
        {"name": "head_wide_mlp", "op": "head", "dtype": "float32", "M": 8192, "K": 4096, "V": 1000, "bias": True,
         "grad": True, "ignored": 0.0, "masked": 0},
        # an ordinary training batch of tokens, no bias
        {"name": "head_mid", "op": "head", "dtype": "float32", "M": 2048, "K": 1024, "V": 32000, "bias": False,
         "grad": True, "ignored": 0.0, "masked": 0},
        # a padded batch of odd sizes: a third of the rows is padding, and some classes are masked out
        {"name": "head_ragged", "op": "head", "dtype": "float32", "M": 1999, "K": 1111, "V": 50021, "bias": True,
         "grad": True, "ignored": 0.35, "masked": 21},
        # a long batch over a large vocabulary
        {"name": "head_large", "op": "head", "dtype": "float32", "M": 8192, "K": 2048, "V": 98304, "bias": False,
         "grad": True, "ignored": 0.05, "masked": 0},
        # evaluation: the loss and every token's loss, no gradient
        {"name": "head_eval", "op": "head", "dtype": "float32", "M": 4096, "K": 1024, "V": 65536, "bias": True,
         "grad": False, "ignored": 0.1, "masked": 0},
        # double precision, as the fp64 MLP trains
        {"name": "head_f64", "op": "head", "dtype": "float64", "M": 512, "K": 512, "V": 8192, "bias": True,
         "grad": True, "ignored": 0.1, "masked": 0},
        # a small model: ten tensors, one launch's latency
        {"name": "adamw_tiny", "op": "adamw", "dtype": "float32", "state": "native", "tensors": 10, "total": 120000,
         "packed": True, "clip": False},
        # the wide MLP's parameter count over many tensors, clipped by the global norm
        {"name": "adamw_mid_clip", "op": "adamw", "dtype": "float32", "state": "native", "tensors": 96,
         "total": 37659624, "packed": False, "clip": True},
        # a large model: a few hundred packed tensors, most of them not 16-byte aligned
        {"name": "adamw_large", "op": "adamw", "dtype": "float32", "state": "native", "tensors": 291,
         "total": 400000000, "packed": True, "clip": False},
        # the same with 8-bit states
        {"name": "adamw_large_8bit", "op": "adamw", "dtype": "float32", "state": "e4m3", "tensors": 291,
         "total": 400000000, "packed": False, "clip": False},
        # double precision
        {"name": "adamw_f64", "op": "adamw", "dtype": "float64", "state": "native", "tensors": 37, "total": 20000003,
         "packed": True, "clip": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.55:
        f64 = rng.random() < 0.15
        while True:
            M, K, V = _log(rng, 1, 8192), _log(rng, 16, 4096), _log(rng, 200, 100000)
            if M * K * V <= (2 ** 31 if f64 else 2 ** 41):
                break
        return {"op": "head", "dtype": "float64" if f64 else "float32", "M": M, "K": K, "V": V,
                "bias": rng.random() < 0.5, "grad": rng.random() < 0.8,
                "ignored": rng.choice([0.0, 0.0, 0.1, 0.5]), "masked": rng.choice([0, 0, 1, V // 50])}
    state = "e4m3" if rng.random() < 0.4 else "native"
    f64 = state == "native" and rng.random() < 0.2
    total = _log(rng, 2000, 20_000_000 if f64 else 400_000_000)
    return {"op": "adamw", "dtype": "float64" if f64 else "float32", "state": state,
            "tensors": min(_log(rng, 1, 400), max(1, total // 100)), "total": total,
            "packed": state == "native" and rng.random() < 0.5, "clip": state == "native" and rng.random() < 0.5}


def _sizes(case):
    """The tensors' lengths: vectors and matrices of a model, `total` values in all."""
    rng = random.Random(case["tensors"] * 1000003 + case["total"])
    share = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    scale = case["total"] / sum(share)
    sizes = [max(1, int(s * scale)) for s in share]
    sizes[-1] += max(0, case["total"] - sum(sizes))
    return sizes


def _layout(case):
    """(length, start) of every tensor in the flat buffers, and the buffers' length."""
    at, found = 0, []
    for n in _sizes(case):
        found.append((n, at))
        at += n if case["packed"] else -(-n // BLOCK) * BLOCK
    return found, -(-at // BLOCK) * BLOCK


# ---- inputs -------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    return (_prepare_head if case["op"] == "head" else _prepare_adamw)(case, seed, gen)


def _prepare_head(case, seed, gen):
    M, K, V, t = case["M"], case["K"], case["V"], TYPES[case["dtype"]]
    new = lambda *shape: torch.randn(*shape, generator=gen, device="cuda", dtype=t)  # noqa: E731
    # hidden rows after a norm; weights that give logits of a few units; frequent and rare labels
    s = {"case": case, "x": new(M, K), "w": new(V, K).mul_(2.0 / math.sqrt(K)), "bias": None}
    u = torch.rand(M, generator=gen, device="cuda", dtype=torch.float64)
    labels = (torch.exp(u * math.log(V + 1.0)) - 1.0).to(torch.int64).clamp_(0, V - 1)
    if case["bias"]:
        s["bias"] = new(V).mul_(0.5)
        if case["masked"]:  # classes that may not be chosen: the last ones, never a label
            s["bias"][V - case["masked"]:] = -math.inf
    if case["masked"]:
        labels.clamp_(max=V - case["masked"] - 1)
    if case["ignored"]:
        drop = torch.rand(M, generator=gen, device="cuda") < case["ignored"]
        drop[0] = False
        labels = torch.where(drop, IGNORE, labels)
    s["labels"] = labels.to(torch.int32)
    s["loss"], s["rows"] = torch.zeros(1, device="cuda", dtype=t), torch.zeros(M, device="cuda", dtype=t)
    if case["grad"]:
        s["dx"], s["dw"] = torch.zeros_like(s["x"]), torch.zeros_like(s["w"])
        s["db"] = torch.zeros(V, device="cuda", dtype=t) if case["bias"] else None
    return s


def _prepare_adamw(case, seed, gen):
    t = TYPES[case["dtype"]]
    tensors, total = _layout(case)
    new = lambda: torch.randn(total, generator=gen, device="cuda", dtype=t)  # noqa: E731
    here = torch.zeros(total, device="cuda", dtype=torch.bool)  # values of a tensor, not of the gaps between them
    decays = torch.zeros(total, device="cuda", dtype=torch.bool)
    for n, at in tensors:
        here[at:at + n] = True
        decays[at:at + n] = n > 8192  # vectors are not decayed
    g = new().mul_(1e-3).mul_(torch.exp(new()))
    s = {"case": case, "tensors": tensors, "seed": seed, "t": START, "decays": decays,
         "p": new().mul_(0.02).mul_(here), "g": g.mul_(here), "step": torch.full((1,), START, device="cuda", dtype=torch.int64),
         "norm": torch.zeros(2, device="cuda", dtype=torch.float64)}
    del g
    m = new().mul_(3e-4).mul_(here)
    v = new().mul_(1e-3).mul_(torch.exp(new())).square_().mul_(here)
    if case["state"] == "e4m3":
        h = _hash(total // BLOCK, seed + 1, 0, "cuda")
        s["m"], s["m_scale"] = _encode(m, h & 0xFFFF, False)
        s["v"], s["v_scale"] = _encode(v.sqrt(), h >> 16, True)
    else:
        s["m"], s["v"] = m, v
    if own:
        s["opt"] = _optimizer(s)
    return s


# ---- one pass -----------------------------------------------------------------


def run(s):
    if own:
        return _own_head(s) if s["case"]["op"] == "head" else _own_adamw(s)
    return _head(s) if s["case"]["op"] == "head" else _adamw(s)


def _package():
    import os
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-tensor_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from gotensor import _lib, loss, optim
    return _lib, loss, optim


def _own_head(s):
    _lib, loss, _ = _package()
    c = s["case"]
    loss.linear_cross_entropy(
        s["x"].data_ptr(), s["w"].data_ptr(), s["bias"].data_ptr() if c["bias"] else None, s["labels"].data_ptr(),
        c["M"], c["K"], c["V"], loss=s["loss"].data_ptr(), rows=s["rows"].data_ptr(),
        dx=s["dx"].data_ptr() if c["grad"] else None, dw=s["dw"].data_ptr() if c["grad"] else None,
        db=s["db"].data_ptr() if c["grad"] and c["bias"] else None, ignore_label=IGNORE,
        dtype=_lib.FLOAT64 if c["dtype"] == "float64" else _lib.FLOAT32)
    return _outputs_head(s)


def _outputs_head(s):
    out = {"loss": s["loss"], "rows": s["rows"]}
    if s["case"]["grad"]:
        out["dx"], out["dw"] = s["dx"], s["dw"]
        if s["case"]["bias"]:
            out["db"] = s["db"]
    return out


def _head(s):
    c = s["case"]
    keep = s["labels"] != IGNORE
    y = torch.where(keep, s["labels"], 0).to(torch.int64)
    x = torch.where(keep[:, None], s["x"], 0)
    z = x @ s["w"].T
    if c["bias"]:
        z = z + s["bias"]
    top = z.amax(1, keepdim=True)
    picked = z.gather(1, y[:, None])
    e = torch.exp(z.sub_(top))
    total = e.sum(1, keepdim=True)
    rows = torch.where(keep, (torch.log(total) + (top - picked))[:, 0], 0)
    count = keep.sum()
    out = {"loss": (rows.double().sum() / count).to(rows.dtype)[None], "rows": rows}
    if c["grad"]:
        grad = e.mul_(torch.where(keep, 1.0 / count.to(rows.dtype), 0)[:, None] / total)
        at = torch.arange(c["M"], device=z.device)
        grad[at, y] -= torch.where(keep, 1.0 / count.to(rows.dtype), 0)
        out["dx"], out["dw"] = grad @ s["w"], grad.T @ x
        if c["bias"]:
            out["db"] = grad.sum(0)
    return out


def _optimizer(s):
    _lib, _, optim = _package()
    c = s["case"]
    size = 8 if c["dtype"] == "float64" else 4
    low = c["state"] == "e4m3"
    held = 1 if low else size
    tensors = [optim.Tensor(
        p=s["p"].data_ptr() + at * size, g=s["g"].data_ptr() + at * size, m=s["m"].data_ptr() + at * held,
        v=s["v"].data_ptr() + at * held, n=n, wd_mul=1.0 if n > 8192 else 0.0,
        m_scale=s["m_scale"].data_ptr() + at // BLOCK * 4 if low else None,
        v_scale=s["v_scale"].data_ptr() + at // BLOCK * 4 if low else None) for n, at in s["tensors"]]
    return optim.AdamW(tensors, step=s["step"].data_ptr(), lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS,
                       weight_decay=DECAY, state=optim.STATE_E4M3 if low else optim.STATE_NATIVE, seed=s["seed"],
                       dtype=_lib.FLOAT64 if c["dtype"] == "float64" else _lib.FLOAT32)


def _own_adamw(s):
    if s["case"]["clip"]:
        s["opt"].clip_grad_norm(MAX_NORM, s["norm"].data_ptr())
    s["opt"].step()
    return _outputs_adamw(s)


def _outputs_adamw(s):
    out = {"p": s["p"], "m": s["m"], "v": s["v"]}
    if s["case"]["state"] == "e4m3":  # the values that the codes stand for, in units of their blocks' scales
        out["m"], out["v"] = s["m"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn)
        out["m_scale"], out["v_scale"] = s["m_scale"], s["v_scale"]
    if s["case"]["clip"]:
        out["norm"] = s["norm"][:1]
    return out


def _mix(x):
    """A mix of the bits of 32-bit words (held in int64)."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & MASK32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & MASK32
    return x ^ (x >> 16)


def _hash(blocks, seed, t, device):
    """32 random bits for each value of `blocks` blocks at step t."""
    words = torch.tensor([seed & MASK32, (seed >> 32) & MASK32, t & MASK32, (t >> 32) & MASK32], dtype=torch.int64)
    key = _mix(_mix(_mix(_mix(words[0]) ^ words[1]) ^ words[2]) ^ words[3]).to(device)
    b = torch.arange(blocks, device=device)
    b = _mix(_mix(key ^ (b & MASK32)) ^ (b >> 32))
    return _mix((b[:, None] + torch.arange(BLOCK, device=device)) & MASK32).view(-1)


def _encode(x, r16, positive):
    """Codes (a sign, 4 bits of exponent, 3 of mantissa) of x in units of its blocks' scales, rounded up or down at
    random by r16 / 65536, and the scales. What is above zero in a `positive` state stays above zero."""
    x = x.view(-1, BLOCK)
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), 0).amax(1, keepdim=True)
    some = top >= 2.0 ** -100
    scale = torch.where(some, top * (1.0 / 448.0), 0)
    y = torch.clamp(x.abs() * torch.where(some, torch.full_like(top, 448.0) / top, 0), max=448.0)
    small = y < 2.0 ** -6
    bits = torch.where(small, y + 2.0 ** -6, y).view(torch.int32).to(torch.int64)
    code = ((bits + (r16.view(-1, BLOCK) << 4)) >> 20) - (120 << 3) - torch.where(small, 8, 0)
    if positive:
        code = torch.where((code == 0) & (y > 0), 1, code)
    code = torch.where(fine, code + torch.where(x < 0, 128, 0), 127)
    return code.to(torch.uint8).view(-1), scale.view(-1)


def _decode(codes, scale):
    return (codes.view(torch.float8_e4m3fn).to(torch.float32).view(-1, BLOCK) * scale[:, None]).view(-1)


def _adamw(s):
    c, low = s["case"], s["case"]["state"] == "e4m3"
    s["t"] += 1
    t, g = s["t"], s["g"]
    if c["clip"]:
        norm = g.double().square().sum().sqrt()
        s["norm"][0] = norm
        g = g * torch.clamp(MAX_NORM / norm, max=1.0).to(g.dtype)
    m = _decode(s["m"], s["m_scale"]) if low else s["m"]
    v = _decode(s["v"], s["v_scale"]).square() if low else s["v"]
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    root = v.sqrt()
    p = torch.where(s["decays"], s["p"] * (1.0 - LR * DECAY), s["p"])
    s["p"].copy_(p - (m * (LR / (1.0 - BETA1 ** t))) / (root * (1.0 / math.sqrt(1.0 - BETA2 ** t)) + EPS))
    if low:
        h = _hash(m.numel() // BLOCK, s["seed"], t, m.device)
        for name, x, r16, positive in (("m", m, h & 0xFFFF, False), ("v", root, h >> 16, True)):
            codes, scale = _encode(x, r16, positive)
            s[name].copy_(codes)
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _outputs_adamw(s)


# ---- the work, and the outputs in 64 bits -----------------------------------------


def work(case):
    if case["op"] == "head":
        M, K, V = case["M"], case["K"], case["V"]
        e = 8 if case["dtype"] == "float64" else 4
        once = M * K + V * K + (V if case["bias"] else 0)
        return {"bytes": e * (once * (2 if case["grad"] else 1) + M + 1) + 4 * M,
                "flops": (6 if case["grad"] else 2) * M * K * V}
    n = sum(_sizes(case))
    if case["state"] == "e4m3":
        return {"bytes": n * (4 * 3 + 2 * 2) + 16 * (n / BLOCK), "flops": 14 * n}
    e = 8 if case["dtype"] == "float64" else 4
    return {"bytes": n * e * 7, "flops": (14 + (2 if case["clip"] else 0)) * n}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_head(case, s) if case["op"] == "head" else _exact_adamw(case, s)


def _exact_head(case, s):
    M, K, V = case["M"], case["K"], case["V"]
    kept = torch.nonzero(s["labels"] != IGNORE)[:, 0]
    w, bias = s["w"].double(), s["bias"].double() if case["bias"] else None
    rows = torch.zeros(M, device="cuda", dtype=torch.float64)
    dx = torch.zeros(M, K, device="cuda", dtype=torch.float64)
    dw = torch.zeros(V, K, device="cuda", dtype=torch.float64) if case["grad"] else None
    db = torch.zeros(V, device="cuda", dtype=torch.float64)
    for part in torch.split(kept, 1024):
        x, y = s["x"][part].double(), s["labels"][part].long()
        z = torch.mm(x, w.t())
        if bias is not None:
            z += bias
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        rows[part] = -logp.gather(1, y[:, None])[:, 0]
        if case["grad"]:
            g = logp.exp_()
            g.scatter_add_(1, y[:, None], torch.full((len(part), 1), -1.0, device="cuda", dtype=torch.float64))
            g /= len(kept)
            dx[part] = torch.mm(g, w)
            dw.addmm_(g.t(), x)
            db += g.sum(0)
    out = {"loss": rows.sum()[None] / len(kept), "rows": rows}
    if case["grad"]:
        out["dx"], out["dw"] = dx, dw
        if case["bias"]:
            out["db"] = db
    return out


def _exact_adamw(case, s):
    low, t = case["state"] == "e4m3", START + 1
    g, p = s["g"].double(), s["p"].double()
    norm = torch.linalg.vector_norm(g)
    if case["clip"] and norm > MAX_NORM:
        g *= MAX_NORM / norm
    if low:
        m, root = (s[k].view(torch.float8_e4m3fn).double() * s[k + "_scale"].double().repeat_interleave(BLOCK)
                   for k in ("m", "v"))
        v = root ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    p -= LR * DECAY * p * s["decays"]
    p -= LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out = {"p": p, "m": m, "v": v}
    if low:
        h = _hash(m.numel() // BLOCK, s["seed"], t, m.device)
        for k, value, bits in (("m", m, h % 65536), ("v", v.sqrt(), h // 65536)):
            blocks = value.view(-1, BLOCK)
            scale = blocks.abs().amax(1) / 448
            out[k + "_scale"] = scale
            y = (blocks / torch.where(scale > 0, scale, 1.0)[:, None]).abs()
            # the step of the number format at y: 8 steps from each power of two to the next, no finer than 2^-9
            step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6, max=448.0))) - 3)
            steps = torch.floor(y / step + bits.view(-1, BLOCK) / 65536.0)
            if k == "v":
                steps = torch.where((steps == 0) & (y > 0), 1.0, steps)
            out[k] = (steps * step * torch.sign(blocks)).view(-1)
    if case["clip"]:
        out["norm"] = norm[None]
    return out
