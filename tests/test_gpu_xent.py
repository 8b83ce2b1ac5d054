"""Softmax cross entropy of a linear head (nk_linear_xent_fwd / _bwd) against the definition in 64 bits.

Tolerances.  u = 2^-24, H = half a step of the operands' type (2^-24, 2^-8, 2^-11).
A logit is a sum of D products, exact (16-bit operands) or rounded once (fp32), added in fp32: off by at most
bz = 2 (D + 2) u sum |h w|.  The log-sum-exp adds the rounding of the exponentials (v_exp_f32: 1 unit in the last
place, its argument one product) and of at most 100 + V / 64 additions in sequence, each u relative, so
  b_loss = 2 max bz + u (100 + V / 64 + 4 |lse| + 4 |z_t|).
dz = c (p - onehot): p is off by p (bz + b_loss + 16 u), the result is rounded once to the operands' type (H, and for
fp16 at most half of 2^-24 2^-14 absolute); then K products in fp32 (2 (K + 8) u of the sum of magnitudes) and one
rounding of the result (H)."""
import pytest
import torch

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(N, D, V, dt, seed, ignored=0.15, spread=2.5):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    h = torch.randn(N, D, generator=g, device=dev).to(dt)
    w = (torch.randn(V, D, generator=g, device=dev) * (spread / D ** 0.5)).to(dt)
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    t[torch.rand(N, generator=g, device=dev) < ignored] = -100
    if N > 2:
        t[0], t[1] = V - 1, 0
    return h, w, t, g


def check(h, w, t, reduction, g, piece=0, ignore=-100, h64=None):
    """Losses and gradients; h64: what the reference takes for hidden (rows that must not count replaced)."""
    import nerf_kinematics_amd as nk
    N, D = h.shape
    V, dt, dev = w.shape[0], h.dtype, h.device
    h_, w_ = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = nk.linear_cross_entropy(h_, w_, t, ignore_index=ignore, reduction=reduction, piece=piece)
    d_loss = torch.randn(N, generator=g, device=dev) if reduction == "none" else torch.rand((), generator=g, device=dev) + 0.5
    dh, dw = torch.autograd.grad(loss, (h_, w_), d_loss)
    a, b = (h if h64 is None else h64).detach().double(), w.detach().double()
    keep = t != ignore
    at = torch.where(keep, t, 0 * t)[:, None]
    z = a @ b.t()
    lse = torch.logsumexp(z, 1)
    zt = z.gather(1, at)[:, 0]
    bz = (2 * (D + 2) * U * (a.abs() @ b.abs().t())).amax(1)
    bl = 2 * bz + U * (100 + V / 64 + 4 * lse.abs() + 4 * zt.abs())
    ref = torch.where(keep, lse - zt, 0 * lse)
    bl = torch.where(keep, bl, 0 * bl)
    count = max(1, int(keep.sum()))
    if reduction == "none":
        c, total, btotal = d_loss.double() * keep, ref, bl
    else:
        f = count if reduction == "mean" else 1
        c, total, btotal = keep.double() * (d_loss.double() / f), ref.sum() / f, bl.sum() / f
    err = (loss.detach().double() - total).abs()
    assert bool((err <= btotal + 2 * U * total.abs()).all()), f"loss: {float((err - btotal).max()):.3e} over"
    p = (z - lse[:, None]).exp()
    dz = p.clone()
    dz.scatter_add_(1, at, torch.full_like(at, -1, dtype=dz.dtype))
    dz = dz * c[:, None]
    bd = c.abs()[:, None] * p * (bz + bl + 16 * U)[:, None] + dz.abs() * (HALF[dt] + 8 * U)
    if dt == F16:
        bd = bd + 2.0 ** -39 * 2 * c.abs().max()
    bd = bd * keep[:, None]
    for name, got, want, bound in (("d_hidden", dh, dz @ b, bd @ b.abs() + 2 * (V + 8) * U * (dz.abs() @ b.abs())),
                                   ("d_weight", dw, dz.t() @ a, bd.t() @ a.abs() + 2 * (N + 8) * U * (dz.abs().t() @ a.abs()))):
        assert got.dtype == dt and got.shape == want.shape
        tol = bound + HALF[dt] * want.abs() + (2.0 ** -25 if dt == F16 else 0.0)
        over = (got.double() - want).abs() - tol
        assert bool((over <= 0).all()), f"{name}: {float(over.max()):.3e} over the tolerance"
    assert not dh[~keep].any()
    return loss.detach(), dh, dw


SHAPES = [(1, 1, 1), (1, 8, 2), (3, 16, 7), (33, 24, 129), (64, 64, 256), (5, 100, 1000), (130, 72, 257), (31, 40, 300), (300, 200, 3000),
          (257, 128, 5003), (1000, 64, 130), (129, 333, 511), (16, 256, 9001)]


@gpu
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shapes(shape, dt):
    k = SHAPES.index(shape)
    h, w, t, g = make(*shape, dt, k)
    check(h, w, t, ("mean", "sum", "none")[k % 3], g)


@gpu
@pytest.mark.parametrize("shape", [(2048, 512, 8192), (200, 2048, 8192), (7168, 2048, 300), (33, 1056, 2500)], ids=lambda s: "x".join(map(str, s)))
def test_large_tiles(shape):
    h, w, t, g = make(*shape, BF16, 1)
    check(h, w, t, "none", g)


@gpu
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(20000, 64, 16), (9001, 50, 150), (16385, 24, 2), (8193, 33, 65)], ids=lambda s: "x".join(map(str, s)))
def test_many_tokens_few_labels(shape, dt):
    """d_weight's long sum is cut into stretches, and the tokens are counted by many workgroups."""
    h, w, t, g = make(*shape, dt, 14)
    check(h, w, t, "none" if shape[1] == 64 else "mean", g)
    check(h, w, t, "sum", g, piece=256)


@gpu
@pytest.mark.parametrize("piece", [1, 256, 300, 512, 5000])
@pytest.mark.parametrize("D", [64, 50])
def test_pieces(piece, D):
    """The vocabulary in pieces of any size; d_hidden's sums run over the pieces."""
    h, w, t, g = make(70, D, 1111, BF16, 3)
    check(h, w, t, "mean", g, piece=piece)


@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions_and_ignored_rows(reduction):
    h, w, t, g = make(90, 48, 400, BF16, 4)
    check(h, w, t, reduction, g)
    h, w, t, g = make(90, 48, 400, BF16, 4, ignored=0.0)
    t[5] = 7
    check(h, w, t, reduction, g, ignore=7)
    # rows that do not count may hold anything
    h, w, t, g = make(90, 48, 400, BF16, 5)
    clean = h.clone()
    h[t == -100] = float("nan")
    check(h, w, t, reduction, g, h64=clean)
    h[t == -100] = float("inf")
    check(h, w, t, reduction, g, h64=clean)


@gpu
def test_no_row_counts_and_no_rows():
    import nerf_kinematics_amd as nk
    h, w, t, _ = make(20, 16, 50, F32, 6)
    t[:] = -100
    for N in (20, 0):
        a, b = h[:N].clone().requires_grad_(True), w.clone().requires_grad_(True)
        for reduction in ("mean", "sum", "none"):
            loss = nk.linear_cross_entropy(a, b, t[:N], reduction=reduction)
            assert loss.shape == ((N,) if reduction == "none" else ()) and not loss.any()
            da, db = torch.autograd.grad(loss.sum(), (a, b))
            assert da.shape == a.shape and not da.any() and not db.any()


@gpu
@pytest.mark.parametrize("bad", [50, -1, 1 << 40, -(1 << 40)])
def test_targets_out_of_range(bad):
    import nerf_kinematics_amd as nk
    h, w, t, _ = make(20, 16, 50, F32, 7)
    t[3] = bad
    loss = nk.linear_cross_entropy(h, w, t, reduction="none")
    assert torch.isnan(loss[3]) and int(torch.isnan(loss).sum()) == 1
    assert torch.isnan(nk.linear_cross_entropy(h, w, t))
    a = h.clone().requires_grad_(True)
    nk.linear_cross_entropy(a, w, t, reduction="sum").backward()
    assert torch.isnan(a.grad[3]).all() and int(torch.isnan(a.grad).any(1).sum()) == 1


@gpu
def test_large_logits():
    """Logits of +-1000 and a column that never wins: no overflow, and a certain answer has loss 0."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    h = torch.eye(16, device=dev) * 100.0
    w = torch.zeros(40, 16, device=dev)
    w[:16] = torch.eye(16, device=dev) * 10.0
    w[20:] = -10.0
    t = torch.arange(16, device=dev)
    loss = nk.linear_cross_entropy(h, w, t, reduction="none")
    assert not loss.any()
    loss = nk.linear_cross_entropy(h, w, (t + 1) % 16, reduction="none")
    assert torch.allclose(loss, torch.full_like(loss, 1000.0), rtol=2 ** -22, atol=0)
    a = h.clone().requires_grad_(True)
    nk.linear_cross_entropy(a, w, (t + 1) % 16, reduction="sum").backward()
    want = w[:16] - w[(t + 1) % 16]
    assert torch.allclose(a.grad, want, rtol=2 ** -20, atol=0)


@gpu
@pytest.mark.parametrize("which", ["columns of a wider tensor", "odd address", "transposed", "overlapping rows", "expanded loss"])
def test_layouts(which):
    h, w, t, g = make(65, 64, 333, BF16, 8)
    if which == "columns of a wider tensor":
        h, w = torch.cat((h, h), 1)[:, 64:], torch.cat((w, w, w), 1)[:, 64:128]
    elif which == "odd address":
        mv = lambda x: torch.cat((x.reshape(-1)[:1], x.reshape(-1)))[1:].view(x.shape)
        h, w = mv(h), mv(w)
    elif which == "transposed":
        h, w = h.t().contiguous().t(), w.t().contiguous().t()
    elif which == "overlapping rows":
        h = h[:1].expand(65, 64)
    check(h, w, t, "none", g)


@gpu
def test_millions_of_tokens():
    """Row offsets of the logit gradients far beyond 2^22 bytes times a tile's rows."""
    h, w, t, g = make(4200003, 16, 3, BF16, 15)
    check(h, w, t, "mean", g)


@gpu
def test_single_rows_of_any_stride():
    """One token and one label: torch gives a dimension of size one any stride, zero among them."""
    h, w, t, g = make(1, 24, 1, BF16, 12, ignored=0.0)
    one = h[0].as_strided((1, 24), (0, 1))
    check(one, w, t, "none", g)
    check(h, w[0].as_strided((1, 24), (3, 1)), t, "mean", g)
    h, w, t, g = make(1, 24, 700, BF16, 13, ignored=0.0)
    check(h[0].as_strided((1, 24), (0, 1)), w, t, "sum", g, piece=2 ** 62)


@gpu
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_the_loss_may_be_changed_in_place(reduction):
    import nerf_kinematics_amd as nk
    h, w, t, _ = make(40, 24, 50, F32, 16)
    a, b = h.clone().requires_grad_(True), h.clone().requires_grad_(True)
    x, y = nk.linear_cross_entropy(a, w, t, reduction=reduction), nk.linear_cross_entropy(b, w, t, reduction=reduction)
    x *= 2.0
    (got,), (want,) = torch.autograd.grad(x.sum(), a), torch.autograd.grad((y * 2.0).sum(), b)
    assert torch.equal(got, want) and bool(got.any())


@gpu
def test_only_one_gradient():
    import nerf_kinematics_amd as nk
    h, w, t, g = make(100, 64, 500, BF16, 9)
    _, dh, dw = check(h, w, t, "mean", torch.Generator(device=h.device).manual_seed(1))
    d = torch.rand((), generator=torch.Generator(device=h.device).manual_seed(1), device=h.device) + 0.5
    a = h.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(nk.linear_cross_entropy(a, w, t), a, d)[0], dh)
    b = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(nk.linear_cross_entropy(h, b, t), b, d)[0], dw)


@gpu
def test_gradients_against_differences():
    """Central differences of the fp32 losses (summed in 64 bits): a step of 2^-6 leaves a truncation of at most
    2^-12 |w|^3 / 6 and a rounding of N b_loss / 2^-6, both far below the 2e-3 allowed."""
    import nerf_kinematics_amd as nk
    h, w, t, _ = make(6, 8, 30, F32, 10, spread=1.0)
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    f = lambda x, y: nk.linear_cross_entropy(x, y, t, reduction="none").double().sum()
    ga, gb = torch.autograd.grad(f(a, b), (a, b))
    e = 2.0 ** -6
    with torch.no_grad():
        for k, grad in ((0, ga), (1, gb)):
            for i in range(0, grad.numel(), 5):
                up, dn = [h.clone(), w.clone()], [h.clone(), w.clone()]
                up[k].view(-1)[i] += e; dn[k].view(-1)[i] -= e
                d = float(f(*up) - f(*dn)) / float(up[k].view(-1)[i] - dn[k].view(-1)[i])
                assert abs(d - float(grad.reshape(-1)[i])) < 2e-3 * (1 + abs(d))


@gpu
def test_repeat_other_stream_and_graph_replay():
    import nerf_kinematics_amd as nk
    h, w, t, g = make(200, 96, 3000, BF16, 11)

    def both(a, b):
        loss = nk.linear_cross_entropy(a, b, t, piece=1024)
        return (loss,) + torch.autograd.grad(loss, (a, b))
    leaves = lambda: (h.clone().requires_grad_(True), w.clone().requires_grad_(True))
    first = [x.detach().clone() for x in both(*leaves())]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        again = both(*leaves())
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, again))
    inp = leaves()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = both(*inp)
    for k in range(3):
        new = h * (1 + 0.25 * k)
        with torch.no_grad():
            inp[0].copy_(new)
        graph.replay()
        eager = both(new.clone().requires_grad_(True), w.clone().requires_grad_(True))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, eager)), k


def test_refusals_on_the_host():
    import nerf_kinematics_amd as nk
    from nerf_kinematics_amd import lib as nklib
    z = torch.zeros
    i64 = lambda n: z(n, dtype=torch.int64)
    for h, w, t, kw, msg in ((z(4, 8), z(5, 8), i64(4), {}, "GPU"), (z(4, 8), z(5, 7), i64(4), {}, "weight"), (z(4, 8), z(5, 8), z(4), {}, "target"),
                             (z(4, 8), z(5, 8), i64(3), {}, "target"), (z(4), z(5, 8), i64(4), {}, "hidden"), (z(4, 8), z(0, 8), i64(4), {}, "weight"),
                             (z(4, 8), z(5, 8, dtype=BF16), i64(4), {}, "weight"), (z(4, 8).double(), z(5, 8).double(), i64(4), {}, "hidden"),
                             (z(4, 8), z(5, 8), i64(4), dict(reduction="max"), "reduction"), (z(4, 8), z(5, 8), i64(4), dict(piece=-1), "piece")):
        with pytest.raises(ValueError, match=msg):
            nk.linear_cross_entropy(h, w, t, **kw)
    L = nk.load()
    o = lambda **k: nklib.NkXentOpts(**{**dict(N=4, D=8, V=5, hidden_stride=8, weight_stride=8, ignore_index=-100, dtype=1, reduction=1), **k})
    for bad, rc in ((dict(N=-1), -1), (dict(D=0), -1), (dict(V=0), -1), (dict(dtype=3), -1), (dict(reduction=4), -1), (dict(hidden_stride=7), -1),
                    (dict(weight_stride=7), -1), (dict(piece=-1), -1), (dict(V=1 << 27), -2), (dict(D=1 << 21, hidden_stride=1 << 21, weight_stride=1 << 21), -2)):
        assert L.nk_linear_xent_workspace_bytes(o(**bad), 1024, 1024, 1) == rc, bad
        assert L.nk_linear_xent_fwd(o(**bad), 1024, 1024, 1024, 1024, 1024, 1024, 1024, 1 << 40, None) == rc, bad
    assert L.nk_linear_xent_bwd(o(N=(1 << 20) + 1, dtype=0), 1024, 1024, 1024, 1024, 1024, 1024, 1024, 1024, 1 << 40, None) == -2
    assert L.nk_linear_xent_workspace_bytes(o(N=64, D=8, V=1 << 26, piece=1 << 26), 1024, 1024, 1) < 64 * (1 << 22) + (1 << 20)     # a row of dz: 2^22 bytes
    assert L.nk_linear_xent_fwd(o(), None, 1024, 1024, 1024, 1024, 1024, 1024, 1 << 40, None) == -1
    assert L.nk_linear_xent_fwd(o(), 1024, 1024, 1024, 1024, 1024, None, 1024, 1 << 40, None) == -1
    assert L.nk_linear_xent_fwd(o(), 1024, 1024, 1024, 1024, 1024, 1024, 1024, 0, None) == -4
    assert L.nk_linear_xent_bwd(o(), 1024, 1024, 1024, 1024, 1024, None, None, 1024, 1 << 40, None) == -1
    assert L.nk_linear_xent_bwd(o(), 1024, 1024, 1024, 1024, 1024, 1024, 1024, 1024 + 8, 1 << 40, None) == -4
    assert L.nk_linear_xent_bwd(o(N=0), 1024, 1024, 1024, 1024, 1024, 1024, 1024, 1024, 1 << 40, None) == -1
