"""Measured cases of the training operators beyond the render path: a gated linear recurrence along a
long axis (forward and backward), the softmax cross entropy of a linear head (forward and backward) and
an AdamW step over many tensors with 32-bit or 8-bit states.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the
end) while ``own`` is false, and through ``nerf_kinematics_amd`` while it is true.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"

BLOCK = 256                      # elements that share a scale in an 8-bit optimiser state
BETA1, BETA2, EPS, LR, DECAY, STEP = 0.9, 0.999, 1e-8, 5e-4, 0.01, 1000


def listed():
    return [
        # ---- recurrence: h_t = a_t * h_(t-1) + x_t -------------------------------------------------
        # one step of 64 running sequences, the state carried over from the step before: latency counts
        dict(name="scan_step", op="scan", B=64, T=1, C=2048, gates=2048, dt="bf16", gate_dt="f32", reverse=False, ragged=False, train=False),
        # feature compositing along rays: 64 + 128 samples, 64 features, one transmittance per sample shared
        # by the features, far sample first, rays cut short at different depths; one training step
        dict(name="scan_rays", op="scan", B=4096, T=192, C=64, gates=1, dt="bf16", gate_dt="f32", reverse=True, ragged=True, train=True),
        # a few long sequences of a gated layer in training, a gate for each channel
        dict(name="scan_long", op="scan", B=2, T=32768, C=1024, gates=1024, dt="bf16", gate_dt="bf16", reverse=False, ragged=False, train=True),
        # one long odd sequence in 32 bits, heads of 20 channels that share a gate: forward only
        dict(name="scan_odd", op="scan", B=1, T=50021, C=300, gates=15, dt="f32", gate_dt="f32", reverse=False, ragged=False, train=False),
        # ---- softmax cross entropy of a linear head ------------------------------------------------
        # scoring a handful of positions against a large vocabulary
        dict(name="xent_score", op="xent", N=16, D=1024, V=50000, dt="bf16", mean=False, train=False),
        # label head of a rendered view: a batch of rays against a small set of classes, 32-bit features
        dict(name="xent_labels", op="xent", N=1024, D=256, V=1000, dt="f32", mean=True, train=True),
        # ordinary training batch, an odd vocabulary
        dict(name="xent_train", op="xent", N=4096, D=1024, V=32003, dt="bf16", mean=True, train=True),
        # large training batch and vocabulary
        dict(name="xent_large", op="xent", N=8192, D=2048, V=65536, dt="bf16", mean=True, train=True),
        # ---- AdamW over many tensors ----------------------------------------------------------------
        # the weights and biases of the coarse and the fine 8x256 network, 32-bit states
        dict(name="adamw_pair", op="adamw", tensors=48, total=1191688, dt="f32", grad_dt="f32", bits=32),
        # the same with 8-bit states
        dict(name="adamw_pair_8bit", op="adamw", tensors=48, total=1191688, dt="f32", grad_dt="f32", bits=8),
        # a large model in 32 bits
        dict(name="adamw_large", op="adamw", tensors=150, total=200000000, dt="f32", grad_dt="f32", bits=32),
        # a large model held in bf16 with bf16 gradients and 8-bit states
        dict(name="adamw_large_8bit", op="adamw", tensors=150, total=200000000, dt="bf16", grad_dt="bf16", bits=8),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["scan", "scan", "xent", "xent", "adamw"])
    if op == "scan":
        while True:
            B, T, C = log(1, 4096), log(1, 50000), log(1, 2048)
            if B * T * C <= 64000000:
                break
        d = rng.choice([1, 1, C] + [k for k in range(2, 65) if C % k == 0])
        dt = rng.choice(["bf16", "bf16", "f16", "f32"])
        return dict(op="scan", B=B, T=T, C=C, gates=C // d, dt=dt, gate_dt=rng.choice([dt, "f32"]), reverse=rng.random() < 0.5,
                    ragged=rng.random() < 0.4, train=rng.random() < 0.7)
    if op == "xent":
        dt = rng.choice(["bf16", "bf16", "f16", "f32"])
        while True:
            N, D, V = log(1, 8192), log(16, 2048), log(2, 65536)
            if N * D * V <= (2 ** 40 if dt != "f32" else 2 ** 37):
                break
        D = D if rng.random() < 0.3 else max(16, D // 16 * 16)
        return dict(op="xent", N=N, D=D, V=V, dt=dt, mean=rng.random() < 0.7, train=rng.random() < 0.7)
    dt = rng.choice(["f32", "f32", "bf16", "f16"])
    return dict(op="adamw", tensors=rng.randint(1, 150), total=log(1000, 150000000), dt=dt, grad_dt=rng.choice([dt, "f32"]),
                bits=rng.choice([32, 8]))


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"case": case, **{"scan": _prepare_scan, "xent": _prepare_xent, "adamw": _prepare_adamw}[case["op"]](case, seed, g)}


def _prepare_scan(c, seed, g):
    B, T, C, dt = c["B"], c["T"], c["C"], DTYPES[c["dt"]]
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    s = {"a": torch.sigmoid(rn(B, T, c["gates"]) * 1.5 + 2.0).to(DTYPES[c["gate_dt"]]), "x": rn(B, T, C).to(dt), "h0": rn(B, C),
         "lengths": None}
    if c["ragged"]:
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    if c["train"]:
        s["d_h"], s["d_last"] = rn(B, T, C).to(dt), rn(B, C)
        for k in ("a", "x", "h0"):
            s[k].requires_grad_(True)
    return s


def _prepare_xent(c, seed, g):
    N, D, V, dt = c["N"], c["D"], c["V"], DTYPES[c["dt"]]
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    s = {"hidden": rn(N, D).to(dt), "weight": (rn(V, D) * (2.5 / math.sqrt(D))).to(dt)}
    t = torch.randint(0, V, (N,), generator=g, device=DEV)
    drop = torch.rand(N, generator=g, device=DEV) < 0.1
    s["target"] = torch.where(drop, torch.full_like(t, -100), t)
    if c["train"]:
        s["hidden"].requires_grad_(True)
        s["weight"].requires_grad_(True)
        s["d_loss"] = torch.rand((), generator=g, device=DEV) + 0.5 if c["mean"] else rn(N)
    return s


def _sizes(c):
    """Element counts of the tensors: weights with a bias behind each, as in a stack of linear layers."""
    n, total = c["tensors"], c["total"]
    rest, out = total, []
    for i in range(n):
        if i == n - 1:
            k = rest
        elif i % 2:
            k = max(1, int(math.isqrt(out[-1])))
        else:
            k = max(1, 2 * total // (n + 1) + 37 * (i % 5) - 74)
        k = max(1, min(k, rest - (n - 1 - i)))
        out.append(k)
        rest -= k
    return out


def _prepare_adamw(c, seed, g):
    sizes = _sizes(c)
    starts = [0]
    for n in sizes:         # every tensor starts on a block of its own inside the flat buffers
        starts.append(starts[-1] + -(-n // BLOCK) * BLOCK)
    F = starts[-1]
    rn = lambda: torch.randn(F, generator=g, device=DEV)  # noqa: E731
    inside = torch.zeros(F, dtype=torch.bool, device=DEV)
    index = torch.empty(F, dtype=torch.int32, device=DEV)       # place of an element inside its tensor
    for a, n in zip(starts, sizes):
        inside[a:a + n] = True
    for a, b in zip(starts, starts[1:]):
        index[a:b] = torch.arange(b - a, device=DEV, dtype=torch.int32)
    p, grad = (rn() * 0.05) * inside, (rn() * 1e-3) * inside
    m, v = (rn() * 3e-4) * inside, (rn() * 1e-3).square() * inside
    cut = lambda t, unit=1: [t[a // unit:(a + n + unit - 1) // unit] for a, n in zip(starts, sizes)]  # noqa: E731
    s = {"p": p.to(DTYPES[c["dt"]]), "g": grad.to(DTYPES[c["grad_dt"]]), "index": index, "inside": inside, "sizes": sizes,
         "master": p.clone() if c["dt"] != "f32" else None, "seed": seed & 0x7FFFFFFF}
    if c["bits"] == 8:
        s["m"], s["m_scale"] = _nearest(m, torch.float8_e4m3fn, 8)
        s["v"], s["v_scale"] = _nearest(v, torch.float8_e5m2, 15)
    else:
        s["m"], s["v"], s["m_scale"], s["v_scale"] = m, v, None, None
    s["lists"] = {k: cut(s[k]) for k in ("p", "g", "m", "v")}
    s["lists"]["master"] = cut(s["master"]) if s["master"] is not None else None
    s["lists"]["scales"] = ([t for t in zip(cut(s["m_scale"], BLOCK), cut(s["v_scale"], BLOCK))] if c["bits"] == 8 else None)
    return s


def _nearest(x, fmt, top):
    """Blocks of x in an 8-bit format: codes and power-of-two scales, the block's largest value in (2^(top-1), 2^top]."""
    b = x.view(-1, BLOCK)
    e = torch.ceil(torch.log2(b.abs().amax(1, keepdim=True).clamp_min(2.0 ** -80))) - top
    scale = torch.exp2(e)
    return (b / scale).to(fmt).reshape(-1), scale.reshape(-1)


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"scan": _own_scan, "xent": _own_xent, "adamw": _own_adamw}[op](state)
    with torch.no_grad():
        return {"scan": _plain_scan, "xent": _plain_xent, "adamw": _plain_adamw}[op](state)


def _own_scan(s):
    import nerf_kinematics_amd as nk
    c = s["case"]
    h, last = nk.gated_scan(s["a"], s["x"], s["h0"], lengths=s["lengths"], reverse=c["reverse"])
    if not c["train"]:
        return {"h": h, "last": last}
    d_a, d_x, d_h0 = torch.autograd.grad((h, last), (s["a"], s["x"], s["h0"]), (s["d_h"], s["d_last"]))
    return {"h": h.detach(), "last": last.detach(), "d_a": d_a, "d_x": d_x, "d_h0": d_h0}


def _own_xent(s):
    import nerf_kinematics_amd as nk
    c = s["case"]
    loss = nk.linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=-100, reduction="mean" if c["mean"] else "none")
    if not c["train"]:
        return {"loss": loss}
    d_hidden, d_weight = torch.autograd.grad(loss, (s["hidden"], s["weight"]), s["d_loss"])
    return {"loss": loss.detach(), "d_hidden": d_hidden, "d_weight": d_weight}


def _own_adamw(s):
    import nerf_kinematics_amd as nk
    if "optimizer" not in s:        # a program makes it once, before its first step
        l = s["lists"]
        s["optimizer"] = nk.AdamW(l["p"], betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, masters=l["master"],
                                  state=(l["m"], l["v"], l["scales"]))
    s["optimizer"].step(s["lists"]["g"], lr=LR, step=STEP, seed=s["seed"])
    return _adamw_outputs(s)


def _adamw_outputs(s):
    """The flat buffers; an 8-bit moment is its codes as the 8-bit floats they are, and the scales of their blocks."""
    return {k: s[k] for k in ("p", "m", "v", "m_scale", "v_scale", "master")}


def _affine_scan(A, H):
    """Inclusive scan of h -> A h + H along dim 1 by doubling: the state after each step from a zero start, and the product of A."""
    T, k = A.shape[1], 1
    while k < T:
        H = torch.cat((H[:, :k], H[:, k:] + A[:, k:] * H[:, :-k]), 1)
        A = torch.cat((A[:, :k], A[:, k:] * A[:, :-k]), 1)
        k *= 2
    return A, H


def _plain_scan(s):
    c = s["case"]
    B, T, C = c["B"], c["T"], c["C"]
    G, J = C // c["gates"], c["gates"]
    order = (lambda t: t.flip(1)) if c["reverse"] else (lambda t: t)
    a = order(s["a"].float())
    x = order(s["x"].float())
    h0 = s["h0"].float()
    if s["lengths"] is None:
        live = None
    else:       # steps behind a sequence's length pass the state on unchanged, and their outputs are zero
        live = order((torch.arange(T, device=DEV)[None, :] < s["lengths"][:, None])[:, :, None])
        a, x = torch.where(live, a, torch.ones_like(a)), torch.where(live, x, torch.zeros_like(x))
    av = a.repeat_interleave(G, 2)
    A, H = _affine_scan(av, x)
    h = H + A * h0[:, None]
    last = h[:, -1].clone()
    shown = h if live is None else torch.where(live, h, torch.zeros_like(h))
    out = {"h": order(shown).to(s["x"].dtype), "last": last}
    if not c["train"]:
        return out
    g = order(s["d_h"].float())
    if live is not None:
        g = torch.where(live, g, torch.zeros_like(g))
    g = torch.cat((g[:, :-1], g[:, -1:] + s["d_last"].float()[:, None]), 1)
    nxt = torch.cat((av[:, 1:], torch.zeros_like(av[:, :1])), 1)
    d = _affine_scan(nxt.flip(1), g.flip(1))[1].flip(1)
    before = torch.cat((h0[:, None], h[:, :-1]), 1)
    d_a = (d * before).view(B, T, J, G).sum(3)
    d_x = d
    if live is not None:
        d_a, d_x = torch.where(live, d_a, torch.zeros_like(d_a)), torch.where(live, d_x, torch.zeros_like(d_x))
    out["d_a"] = order(d_a).to(s["a"].dtype)
    out["d_x"] = order(d_x).to(s["x"].dtype)
    out["d_h0"] = av[:, 0] * d[:, 0]
    return out


def _plain_xent(s):
    c = s["case"]
    h, w, t = s["hidden"].float(), s["weight"].float(), s["target"]
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    lse = (logits - top).exp().sum(1, keepdim=True).log() + top
    keep = t != -100
    at = torch.where(keep, t, torch.zeros_like(t))[:, None]
    loss = torch.where(keep, (lse - logits.gather(1, at))[:, 0], torch.zeros_like(lse[:, 0]))
    count = keep.sum().clamp_min(1)
    out = {"loss": loss.sum() / count if c["mean"] else loss}
    if not c["train"]:
        return out
    d = (logits - lse).exp()
    d.scatter_add_(1, at, torch.full_like(at, -1, dtype=d.dtype))
    coef = s["d_loss"] / count if c["mean"] else s["d_loss"]
    d = d * torch.where(keep, coef, torch.zeros_like(coef))[:, None]
    out["d_hidden"] = (d @ w).to(s["hidden"].dtype)
    out["d_weight"] = (d.t() @ h).to(s["weight"].dtype)
    return out


def _bits(seed, index, u=torch.int64):
    """32 random bits for each element: a finaliser over (seed, index of the element in its tensor)."""
    m = 0xFFFFFFFF

    def mix(x):
        x = x ^ (x >> 16)
        x = (x * 0x7FEB352D) & m
        x = x ^ (x >> 15)
        x = (x * 0x846CA68B) & m
        return x ^ (x >> 16)

    key = mix(torch.tensor((seed ^ (5 * 0x85EBCA6B)) & m, dtype=u, device=index.device))
    return mix((index.to(u) * 0x9E3779B9 + key) & m)


def _stochastic(x, r16, mant, bias, top):
    """Blocks of x >= 0 in an 8-bit float of `mant` fraction bits, rounded up with the probability of the part cut off (r16: 16 random bits)."""
    b = x.view(-1, BLOCK)
    big = b.amax(1, keepdim=True)
    bits = big.view(torch.int32)
    e = (bits >> 23) - 127 + ((bits & 0x7FFFFF) != 0).to(torch.int32) - top      # ceil(log2(largest)) - top
    e = e.clamp_min(-100)
    y = (b * torch.exp2(-e.float())).reshape(-1)
    cut = 23 - mant
    normal = ((y.view(torch.int32) + (r16.to(torch.int32) << (cut - 16))) >> cut) - ((127 - bias) << mant)
    tiny = (y * 2.0 ** (bias - 1 + mant) + r16.float() * 2.0 ** -16).floor().to(torch.int32)
    return torch.where(y < 2.0 ** (1 - bias), tiny, normal), torch.exp2(e.float()).reshape(-1)


def _plain_adamw(s):
    c = s["case"]
    eight = c["bits"] == 8
    g = s["g"].float()
    if eight:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).reshape(-1)
        v = (s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]).reshape(-1)
    else:
        m, v = s["m"], s["v"]
    p = s["master"] if s["master"] is not None else s["p"]
    m = m + (g - m) * float(np.float32(1.0 - BETA1))
    v = v * float(np.float32(BETA2)) + (g * g) * float(np.float32(1.0 - BETA2))
    step_size = float(np.float32(LR / (1.0 - BETA1 ** STEP)))
    root = float(np.float32(math.sqrt(1.0 - BETA2 ** STEP)))
    p = p * float(np.float32(1.0 - LR * DECAY)) - (m / (v.sqrt() / root + EPS)) * step_size
    if s["master"] is not None:
        s["master"].copy_(p)
    s["p"].copy_(p)
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return _adamw_outputs(s)
    r = _bits(s["seed"], s["index"])
    code, scale = _stochastic(m.abs(), r & 0xFFFF, 3, 7, 8)
    code = torch.where(m < 0, code + 128, code).to(torch.uint8)
    s["m"].view(torch.uint8).copy_(code)
    s["m_scale"].copy_(scale)
    code, scale = _stochastic(v, r >> 16, 2, 15, 15)
    code = torch.where((v > 0) & (code == 0), torch.ones_like(code), code).to(torch.uint8)
    s["v"].view(torch.uint8).copy_(code)
    s["v_scale"].copy_(scale)
    return _adamw_outputs(s)


# ------------------------------------------------------------------------------------------------
# cost, and the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "scan":
        n, ng, b, gb = c["B"] * c["T"] * c["C"], c["B"] * c["T"] * c["gates"], BYTES[c["dt"]], BYTES[c["gate_dt"]]
        ends = c["B"] * c["C"] * 4
        if not c["train"]:
            return {"bytes": ng * gb + 2 * n * b + 2 * ends, "flops": 2 * n}
        return {"bytes": 2 * ng * gb + 4 * n * b + 4 * ends, "flops": 6 * n}
    if c["op"] == "xent":
        N, D, V, b = c["N"], c["D"], c["V"], BYTES[c["dt"]]
        one = (N + V) * D * b
        return {"bytes": (2 if c["train"] else 1) * one + 12 * N, "flops": (6 if c["train"] else 2) * N * D * V}
    n = c["total"]
    p, g = BYTES[c["dt"]], BYTES[c["grad_dt"]]
    state = 2 * 8 if c["bits"] == 32 else 2 * (2 + 8 / BLOCK)
    params = 2 * p if c["dt"] == "f32" else p + 8            # a 32-bit master is read and written, its copy written
    return {"bytes": n * (params + g + state), "flops": 14 * n}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"scan": _exact_scan, "xent": _exact_xent, "adamw": _exact_adamw}[case["op"]](case, s)


def _exact_scan(c, s):
    B, T, C, G = c["B"], c["T"], c["C"], c["C"] // c["gates"]
    a64 = lambda t: s["a"][:, t].double().repeat_interleave(G, 1)  # noqa: E731
    n = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), T, device=DEV)
    live = torch.arange(T, device=DEV)[:, None] < n[None, :]             # [T, B]
    steps = range(T - 1, -1, -1) if c["reverse"] else range(T)
    h = s["h0"].double().clone()
    hs = torch.zeros(B, T, C, dtype=torch.float64, device=DEV)
    whole = s["lengths"] is None
    for t in steps:
        new = a64(t) * h + s["x"][:, t].double()
        if whole:
            h = new
            hs[:, t] = new
        else:
            on = live[t][:, None]
            h = torch.where(on, new, h)
            hs[:, t] = torch.where(on, new, torch.zeros_like(new))
    out = {"h": hs, "last": h}
    if not c["train"]:
        return out
    d = s["d_last"].double().clone()
    d_a = torch.zeros(B, T, c["gates"], dtype=torch.float64, device=DEV)
    d_x = torch.zeros_like(hs)
    back = 1 if c["reverse"] else -1
    zero = torch.zeros_like(d)
    for t in reversed(steps):
        q = t + back
        prev = s["h0"].double() if not 0 <= q < T else hs[:, q]
        if not whole and c["reverse"] and 0 <= q < T:      # the first step of a reversed sequence starts from h0
            prev = torch.where(live[q][:, None], prev, s["h0"].double())
        full = d + s["d_h"][:, t].double()
        on = live[t][:, None]
        d_x[:, t] = torch.where(on, full, zero)
        d_a[:, t] = torch.where(on, full * prev, zero).view(B, -1, G).sum(2)
        d = torch.where(on, a64(t) * full, d)
    out.update(d_a=d_a, d_x=d_x, d_h0=d)
    return out


def _exact_xent(c, s):
    N, D, V = c["N"], c["D"], c["V"]
    h, w, t = s["hidden"].detach().double(), s["weight"].detach().double(), s["target"]
    if N * D * V > 2 ** 41:
        return None
    rows = max(1, min(N, 2 ** 27 // V))
    keep = (t != -100).double()
    count = keep.sum().clamp_min(1)
    coef = None
    if c["train"]:
        coef = keep * (s["d_loss"].double() / count if c["mean"] else s["d_loss"].double())
    loss = torch.zeros(N, dtype=torch.float64, device=DEV)
    d_h, d_w = torch.zeros_like(h), torch.zeros_like(w)
    for a in range(0, N, rows):
        b = min(N, a + rows)
        z = h[a:b] @ w.t()
        logp = torch.log_softmax(z, 1)
        at = t[a:b].clamp_min(0)[:, None]
        loss[a:b] = -logp.gather(1, at)[:, 0] * keep[a:b]
        if c["train"]:
            d = logp.exp()
            d.scatter_add_(1, at, torch.full((b - a, 1), -1.0, dtype=torch.float64, device=DEV))
            d *= coef[a:b, None]
            d_h[a:b] = d @ w
            d_w += d.t() @ h[a:b]
    out = {"loss": loss.sum() / count if c["mean"] else loss}
    if c["train"]:
        out.update(d_hidden=d_h, d_weight=d_w)
    return out


def _exact_adamw(c, s):
    f = torch.float64
    g = s["g"].to(f)
    scale = lambda k: s[k + "_scale"].to(f).repeat_interleave(BLOCK) if c["bits"] == 8 else 1.0  # noqa: E731
    m = BETA1 * s["m"].to(f) * scale("m") + (1 - BETA1) * g
    v = BETA2 * s["v"].to(f) * scale("v") + (1 - BETA2) * g ** 2
    p = (s["master"] if s["master"] is not None else s["p"]).to(f)
    p = (1 - LR * DECAY) * p - LR * (m / (1 - BETA1 ** STEP)) / ((v / (1 - BETA2 ** STEP)).sqrt() + EPS)
    out = {"p": p, "master": p if s["master"] is not None else None}
    if c["bits"] == 32:
        return {**out, "m": m, "v": v, "m_scale": None, "v_scale": None}
    r = _bits(s["seed"], s["index"]).to(f)
    low, high = r % 65536, torch.div(r, 65536, rounding_mode="floor")
    for k, x, part, mant, least, top in (("m", m, low, 3, -6, 8), ("v", v, high, 2, -14, 15)):
        peak = x.abs().view(-1, BLOCK).amax(1)
        frac, e = torch.frexp(peak)
        e = (e.to(f) - (frac == 0.5).to(f) - top)
        e = torch.where(peak == 0, torch.full_like(e, -100), e).clamp_min(-100)
        unit = torch.exp2(e)
        y = x.abs() / unit.repeat_interleave(BLOCK)
        grid = torch.exp2((torch.frexp(y)[1].to(f) - 1).clamp_min(least) - mant)         # distance of the values around y
        q = torch.floor(y / grid + part / 65536) * grid
        if k == "v":
            q = torch.where((y > 0) & (q == 0), grid, q)
        out[k], out[k + "_scale"] = torch.where(x < 0, -q, q), unit
    return out
