"""Gated linear recurrence (nk_gated_scan_fwd / _bwd) against a step-by-step loop in 64 bits.

Tolerances.  u = 2^-24.  A result is a sum of terms x_i * (gates between); however the terms are grouped, a gate
enters one product of gates and one multiply-add (2 roundings), a term takes one further addition per step
and at most 40 more in the compositions of runs, wavefronts and stretches.  With hbar the same recurrence on
absolute values and E_s = |a_s| E_(s-1) + 3 hbar_s, the fp32 state is within u (E + 40 hbar); the output adds
half a step of its type.  The backward pass is the same recurrence on gradients, times the state before
(with its own bound) and summed over the G channels of a gate: at most G additions."""
import pytest
import torch

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}        # half a step of fp16's subnormals
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

SHAPES = [(1, 1, 1, 1), (3, 1, 5, 5), (2, 7, 4, 4), (2, 9, 12, 3), (1, 129, 64, 64), (5, 130, 20, 4), (2, 300, 6, 2),
          (3, 257, 200, 2), (1, 4000, 33, 33), (1, 5001, 300, 15), (2, 1000, 1000, 1), (70, 17, 3, 1), (300, 40, 8, 1),
          (1, 600, 7, 7), (4, 8, 512, 1), (4, 8, 1200, 1), (1, 3000, 1, 1), (2, 33, 40, 8), (600, 3, 68, 68), (64, 1, 2048, 2048)]


def order(t, lengths, reverse):
    """Rows in the order of processing (an involution): the first lengths[b] rows flipped if reverse."""
    if not reverse:
        return t
    T = t.shape[1]
    i = torch.arange(T, device=t.device)[None, :]
    n = lengths[:, None]
    at = torch.where(i < n, n - 1 - i, i)
    return t.gather(1, at[:, :, None].expand_as(t))


def loop(a, x, h0, live):
    """h, last, bound of the fp32 error: a, x [B,T,C] in the order of processing, 64 bits."""
    h, hb = h0.clone(), h0.abs()
    E = torch.zeros_like(h)
    hs, bound = [], []
    for t in range(x.shape[1]):
        on = live[:, t, None]
        A, X = a[:, t].abs(), x[:, t].abs()
        hb2 = A * hb + X
        E2 = A * E + 3 * hb2
        h = torch.where(on, a[:, t] * h + x[:, t], h)
        hb, E = torch.where(on, hb2, hb), torch.where(on, E2, E)
        hs.append(torch.where(on, h, 0 * h)); bound.append(U * (E + 40 * hb))
    return torch.stack(hs, 1), h, torch.stack(bound, 1), U * (E + 40 * hb)


def clean(t, live):
    return torch.where(live[:, :, None], t.double(), torch.zeros((), dtype=torch.float64, device=t.device))


def within(got, want, bound, dtype, what):
    tol = bound + HALF[dtype] * want.abs() + TINY[dtype]
    over = (got.double() - want).abs() - tol
    assert bool((over <= 0).all()), f"{what}: {float(over.max()):.3e} over the tolerance"


def check(a, x, h0, lengths, reverse, d_h, d_last):
    import nerf_kinematics_amd as nk
    B, T, C = x.shape
    G, J = C // a.shape[2], a.shape[2]
    n = lengths.long().clamp(0, T) if lengths is not None else torch.full((B,), T, device=x.device)
    live = torch.arange(T, device=x.device)[None, :] < n[:, None]
    leaves = [t.detach().requires_grad_(True) for t in (a, x)] + ([h0.clone().requires_grad_(True)] if h0 is not None else [])
    h, last = nk.gated_scan(leaves[0], leaves[1], leaves[2] if h0 is not None else None, lengths=lengths, reverse=reverse)
    assert h.dtype == x.dtype and last.dtype == F32 and h.shape == x.shape
    outs, gs = [h, last], [d_h, d_last]
    outs, gs = zip(*[(o, g) for o, g in zip(outs, gs) if g is not None])
    grads = torch.autograd.grad(outs, leaves, gs)
    f = lambda t: order(clean(t, live), n, reverse)
    av, xv = f(a).repeat_interleave(G, 2), f(x)
    z = h0.double() if h0 is not None else torch.zeros(B, C, dtype=torch.float64, device=x.device)
    rh, rl, bh, bl = loop(av, xv, z, live)
    within(order(h, n, reverse), rh, bh, x.dtype, "h")
    assert not h[~live].any()
    within(last, rl, bl, F32, "last")
    # backward: e_s = a_s (g_s + e_(s+1)), i.e. d_s = g_s + a_(s+1) d_(s+1), as the loop on flipped rows
    g = f(d_h) if d_h is not None else torch.zeros_like(xv)
    e = d_last.double() if d_last is not None else torch.zeros_like(z)
    d, E, db = torch.zeros_like(xv), torch.zeros_like(e), e.abs()
    bd = torch.zeros_like(xv)
    for s in range(T - 1, -1, -1):
        on = live[:, s, None]
        cur, cb = g[:, s] + e, g[:, s].abs() + db
        ce = E + 3 * cb
        d[:, s] = torch.where(on, cur, 0 * cur); bd[:, s] = torch.where(on, U * (ce + 40 * cb), 0 * cb)
        A = av[:, s]
        e, db, E = torch.where(on, A * cur, e), torch.where(on, A.abs() * cb, db), torch.where(on, A.abs() * ce, E)
    prev, bprev = torch.cat((z[:, None], rh[:, :-1]), 1), torch.cat((0 * z[:, None], bh[:, :-1]), 1)
    da = (d * prev).view(B, T, J, G).sum(3)
    bda = (bd * (prev.abs() + bprev) + bprev * d.abs() + (G + 2) * U * (d * prev).abs()).view(B, T, J, G).sum(3)
    within(order(grads[0], n, reverse), da, bda, a.dtype, "d_a")
    within(order(grads[1], n, reverse), d, bd, x.dtype, "d_x")
    assert not grads[0][~live].any() and not grads[1][~live].any()
    if h0 is not None:
        within(grads[2], e, U * (E + 43 * db), F32, "d_h0")


def inputs(B, T, C, J, dt, gdt, seed, ragged):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)
    a, x, h0 = torch.sigmoid(r(B, T, J) * 1.5 + 2).to(gdt), r(B, T, C).to(dt), r(B, C)
    d_h, d_last, lengths = r(B, T, C).to(dt), r(B, C), None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
        lengths[0] = (0, T, T + 5, -3)[seed % 4]
        dead = torch.arange(T, device=dev)[None, :] >= lengths[:, None]
        for t in (a, x, d_h):
            t[dead] = float("nan")         # nothing behind a sequence is read
    return a, x, h0, lengths, d_h, d_last


@gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shapes(shape, ragged, reverse):
    k = SHAPES.index(shape)
    dt, gdt = [(BF16, BF16), (F32, F32), (F16, F16), (BF16, F32), (F16, F32)][k % 5]
    a, x, h0, lengths, d_h, d_last = inputs(*shape, dt, gdt, k, ragged)
    check(a, x, h0 if k % 3 else None, lengths, reverse, d_h, d_last)


@gpu
@pytest.mark.parametrize("shape", [(2, 259, 48, 48), (2, 259, 48, 4), (3, 50, 9, 3), (1, 2100, 12, 12)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dt,gdt", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_types(shape, dt, gdt):
    a, x, h0, _, d_h, d_last = inputs(*shape, dt, gdt, 9, False)
    check(a, x, h0, None, False, d_h, d_last)


@gpu
@pytest.mark.parametrize("shape", [(2, 300, 129, 1), (2, 70, 255, 3), (3, 40, 127, 127), (2, 1100, 2, 1), (1, 2100, 3, 3)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dt,gdt", [(F32, F32), (BF16, F32), (F16, F16)])
def test_odd_widths(shape, dt, gdt):
    """Columns of two channels over an odd number of them, gates wider than a wavefront among them."""
    a, x, h0, lengths, d_h, d_last = inputs(*shape, dt, gdt, 31, True)
    check(a, x, h0, lengths, True, d_h, d_last)


@gpu
@pytest.mark.parametrize("which", ["sliced", "odd address", "gates shared by sequences", "one gate expanded", "sum", "last only", "h only"])
def test_layouts(which):
    a, x, h0, _, d_h, d_last = inputs(3, 150, 24, 24, BF16, F32, 3, False)
    if which == "sliced":
        x = torch.cat((x, x), 2)[:, ::1, 24:]
        a = a.repeat_interleave(2, 1)[:, ::2]
        d_h = d_h.transpose(0, 1).contiguous().transpose(0, 1)
    elif which == "odd address":
        mv = lambda t: torch.cat((t.reshape(-1)[:1], t.reshape(-1)))[1:].view(t.shape)
        a, x, d_h = mv(a), mv(x), mv(d_h)
    elif which == "gates shared by sequences":
        a = a[:1].expand(3, -1, -1)
    elif which == "one gate expanded":
        a = a[:, :, :1].expand(-1, -1, 24)
    elif which == "sum":
        d_h = torch.ones((), dtype=BF16, device=x.device).expand(3, 150, 24)
    elif which == "last only":
        d_h = None
    elif which == "h only":
        d_last = None
    check(a, x, h0, None, False, d_h, d_last)


@gpu
def test_gradients_against_differences():
    """The loss is linear in each single element of a, x and h0, so a central difference is exact but for the
    rounding of the two losses: their bound (2 u E-type terms summed, below 2e-5 here) over the step of 1."""
    import nerf_kinematics_amd as nk
    a, x, h0, _, w, wl = inputs(2, 13, 6, 2, F32, F32, 5, False)
    ts = [t.clone().requires_grad_(True) for t in (a, x, h0)]
    f = lambda a, x, h0: sum(((o.double() * q.double()).sum()) for o, q in zip(nk.gated_scan(a, x, h0, reverse=True), (w, wl)))
    grads = torch.autograd.grad(f(*ts), ts)
    with torch.no_grad():
        for k, g in enumerate(grads):
            for i in range(0, g.numel(), max(1, g.numel() // 17)):
                up, dn = [t.detach().clone() for t in ts], [t.detach().clone() for t in ts]
                up[k].view(-1)[i] += 0.5; dn[k].view(-1)[i] -= 0.5
                d = float(f(*up) - f(*dn))
                step = float(up[k].view(-1)[i]) - float(dn[k].view(-1)[i])
                assert abs(d / step - float(g.reshape(-1)[i])) < 1e-4 * (1 + abs(d)), (k, i)


@gpu
def test_edges_of_the_values():
    """Zero gates restart a sequence; an untouched zero state stays zero under growing gates; NaN and infinities run on
    from where they are, in their channel, and a step behind the sequence never sees them."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    a, x = torch.full((1, 1000, 8), 0.5, device=dev), torch.ones(1, 1000, 8, device=dev)
    a[0, 500] = 0.0
    h, _ = nk.gated_scan(a, x, torch.full((1, 8), 3.0, device=dev))
    assert torch.equal(h[0, 500], x[0, 500])
    big = torch.full((1, 1000, 8), 2.0, device=dev)
    h, last = nk.gated_scan(big, torch.zeros_like(x))
    assert not h.any() and not last.any()
    x[0, 300, 3], x[0, 400, 5] = float("nan"), float("inf")
    h, last = nk.gated_scan(torch.full_like(a, 0.5), x)
    assert torch.isnan(h[0, 300:, 3]).all() and torch.isinf(h[0, 400:, 5]).all()
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.isfinite(h[0][:, keep]).all() and torch.isfinite(h[0, :300]).all()
    n = torch.tensor([300], dtype=torch.int32, device=dev)
    h, last = nk.gated_scan(torch.full_like(a, 0.5), x, lengths=n)
    assert torch.isfinite(h).all() and torch.isfinite(last).all()


@gpu
def test_empty_batches_and_sequences():
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    for B, T in ((0, 5), (3, 0), (0, 0)):
        a, x = torch.ones(B, T, 4, device=dev, requires_grad=True), torch.ones(B, T, 4, device=dev, requires_grad=True)
        h0 = torch.randn(B, 4, device=dev, requires_grad=True)
        h, last = nk.gated_scan(a, x, h0)
        assert h.shape == (B, T, 4) and torch.equal(last, h0)
        g = torch.autograd.grad(last.sum(), (a, x, h0))
        assert g[0].shape == a.shape and torch.equal(g[2], torch.ones_like(h0))


@gpu
def test_one_step_at_a_time_equals_the_whole():
    """200 calls of one step, the state handed on, against one call: two groupings of the same fp32 sums."""
    import nerf_kinematics_amd as nk
    a, x, h0, _, _, _ = inputs(3, 200, 20, 4, F32, F32, 11, False)
    whole, last = nk.gated_scan(a, x, h0)
    s, rows = h0, []
    for t in range(200):
        h, s = nk.gated_scan(a[:, t:t + 1], x[:, t:t + 1], s)
        rows.append(h)
    av = a.double().repeat_interleave(5, 2)
    live = torch.ones(3, 200, dtype=torch.bool, device=x.device)
    ref, _, bound, _ = loop(av, x.double(), h0.double(), live)
    within(torch.cat(rows, 1), ref, bound, F32, "steps")
    within(whole, ref, bound, F32, "whole")


@gpu
def test_other_stream_repeat_and_graph_replay():
    """The same bits on every run, on a side stream, and from replays of a captured forward and backward pass."""
    import nerf_kinematics_amd as nk
    a, x, h0, lengths, d_h, d_last = inputs(2, 3000, 40, 2, BF16, F32, 14, True)

    def both(a, x, h0):
        h, last = nk.gated_scan(a, x, h0, lengths=lengths, reverse=True)
        return (h, last) + torch.autograd.grad((h, last), (a, x, h0), (d_h, d_last))
    leaves = lambda: [t.detach().clone().requires_grad_(True) for t in (a, x, h0)]
    first = [t.detach().clone() for t in both(*leaves())]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        again = both(*leaves())
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    inp = leaves()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = both(*inp)
    for k in range(3):
        with torch.no_grad():
            inp[1].copy_(x * (k + 1))
        graph.replay()
        eager_in = leaves()
        with torch.no_grad():
            eager_in[1].copy_(x * (k + 1))
        eager = both(*eager_in)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), k


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last steps behind a zero gate equal the same steps on their own."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    T, C, tail = (1 << 21) + 77, 1024, 100
    x = torch.zeros(1, T, C, dtype=BF16, device=dev)
    a = torch.full((1, T, 1), 0.9, device=dev)
    a[0, T - tail] = 0.0
    x[0, T - tail:] = torch.randn(tail, C, device=dev).to(BF16)
    x.requires_grad_(True); a.requires_grad_(True)
    h, last = nk.gated_scan(a, x)
    xs, as_ = x.detach()[:, T - tail:].clone().requires_grad_(True), a.detach()[:, T - tail:].clone().requires_grad_(True)
    hs, ls = nk.gated_scan(as_, xs)
    assert torch.allclose(h[:, T - tail:].float(), hs.float(), rtol=2.0 ** -7, atol=1e-5) and torch.allclose(last, ls, rtol=1e-5, atol=1e-5)
    g = torch.autograd.grad(last.sum(), (a, x)); gs = torch.autograd.grad(ls.sum(), (as_, xs))
    assert torch.allclose(g[1][:, T - tail:].float(), gs[1].float(), rtol=2.0 ** -7, atol=1e-6)
    assert not g[1][:, :T - tail].any()
    assert torch.allclose(g[0][:, T - tail:], gs[0], rtol=1e-2, atol=0.1)


def test_refusals_on_the_host():
    import nerf_kinematics_amd as nk
    from nerf_kinematics_amd import lib as nklib
    z = torch.zeros
    for a, x, msg in ((z(2, 3, 4), z(2, 3, 4), "GPU"), (z(2, 3, 3), z(2, 3, 4), "divisor"), (z(2, 4, 4), z(2, 3, 4), "a:"),
                      (z(2, 3, 4), z(3, 4), "x:"), (z(2, 3, 4), z(2, 3, 4, dtype=torch.float64), "x:"),
                      (z(2, 3, 4, dtype=F16), z(2, 3, 4, dtype=BF16), "a:")):
        with pytest.raises(ValueError, match=msg):
            nk.gated_scan(a, x)
    L = nk.load()
    opts = lambda **k: nklib.NkScanOpts(**{**dict(B=2, T=3, C=4, gates=4, a_stride_b=12, a_stride_t=4, x_stride_b=12, x_stride_t=4), **k})
    assert L.nk_gated_scan_fwd(opts(), *[None] * 7, 0, None) == -1
    assert L.nk_gated_scan_bwd(opts(), *[None] * 10, 0, None) == -1
    for bad, rc in ((dict(gates=3), -1), (dict(gates=0), -1), (dict(B=-1), -1), (dict(T=-1), -1), (dict(dtype=5), -2), (dict(gate_dtype=1), -2),
                    (dict(x_stride_t=-4), -1), (dict(C=1 << 30, gates=1), -2)):
        assert L.nk_gated_scan_workspace_bytes(opts(**bad), 1) == rc, bad
        assert L.nk_gated_scan_fwd(opts(**bad), 8, 8, None, 8, None, None, None, 0, None) == rc, bad
    assert L.nk_gated_scan_fwd(opts(B=1 << 29, T=1, C=16, gates=16), 8, 8, None, 8, None, None, None, 0, None) == -2     # a launch has 2^32 threads
    long = opts(B=1, T=100000)
    need = L.nk_gated_scan_workspace_bytes(long, 0)
    assert need > 0
    assert L.nk_gated_scan_fwd(long, 4096, 4096, None, 4096, None, None, None, 0, None) == -4
    assert L.nk_gated_scan_fwd(long, 4096, 4096, None, 4096, None, None, 4096 + 8, need, None) == -4
    assert L.nk_gated_scan_fwd(opts(T=0), 8, 8, None, 8, None, None, None, 0, None) == -1
    assert L.nk_gated_scan_fwd(opts(B=0), 8, 8, None, 8, None, None, None, 0, None) == 0
