"""Saved-tensor hooks may hand a backward pass its tensors in another layout (``save_on_cpu`` returns dense copies of strided ones).

On the CPU the launch is replaced by a recorder: the addresses and strides that a call would have been made with have to
describe the values that were saved, inside the memory that the hook gave.  On the GPU the gradients have to be the same bits as
without hooks: the same values in the same order, whatever the rows' distance."""
import ctypes

import pytest
import torch

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def scattered(t):
    """The same values where no two neighbours along the last axis are neighbours in memory."""
    if t.dim() < 2:
        return torch.stack((t, t), t.dim())[..., 0]
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)


HOOKS = {"dense copies": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
         "scattered copies": lambda: torch.autograd.graph.saved_tensors_hooks(scattered, lambda t: t)}
GPU_HOOKS = {**HOOKS, "save_on_cpu": lambda: torch.autograd.graph.save_on_cpu()}        # on the CPU it copies nothing


@pytest.fixture
def calls(monkeypatch):
    """What the operators launch, as (name, arguments) in order; nothing runs."""
    from nerf_kinematics_amd import lib
    got = []
    monkeypatch.setattr(lib, "launch", lambda dev, fn, *args: got.append((fn.__name__, args)))
    return got


def reading(address, shape, strides):
    """The float32 values that a kernel reads at `address` with `strides` (elements), row by row."""
    out = torch.empty(shape)
    rows = out.view(-1, shape[-1])
    for i in range(rows.shape[0]):
        at, k = address, i
        for n, s in zip(reversed(shape[:-1]), reversed(strides)):
            at += 4 * (k % n) * s
            k //= n
        rows[i] = torch.tensor((ctypes.c_float * shape[-1]).from_address(at)[:])
    return out


@pytest.mark.parametrize("hook", sorted(HOOKS))
def test_cross_entropy_reads_what_the_hook_returned(calls, hook):
    from nerf_kinematics_amd.xent import _LinearCrossEntropy
    features = torch.arange(8 * 128.0).view(8, 128)
    hidden, weight = features[:, 64:].requires_grad_(True), features.clone()[:5, :64].requires_grad_(True)
    target = torch.arange(8) % 5
    given, back = hidden.detach().clone(), []
    with HOOKS[hook]():
        loss = _LinearCrossEntropy.apply(hidden, weight, target, -100, 0, 0)
    d_hidden, d_weight = torch.autograd.grad(loss, (hidden, weight), torch.ones(8))
    assert [c[0] for c in calls] == ["nk_linear_xent_fwd", "nk_linear_xent_bwd"]
    o, h, w, t = calls[0][1][:4]
    assert (o.hidden_stride, o.weight_stride, h) == (128, 128, hidden.data_ptr())
    o = calls[1][1][0]
    assert (o.N, o.D, o.V) == (8, 64, 5) and (o.hidden_stride, o.weight_stride) == (64, 64)     # the copies are dense
    assert d_hidden.shape == hidden.shape and d_weight.shape == weight.shape


def test_cross_entropy_values_behind_the_addresses(monkeypatch):
    """The same, read out while the call would run."""
    from nerf_kinematics_amd import lib
    from nerf_kinematics_amd.xent import _LinearCrossEntropy
    wide = torch.randn(9, 96)
    hidden, weight = wide[:, 32:].requires_grad_(True), torch.randn(7, 64).requires_grad_(True)
    target, seen = torch.arange(18)[::2] % 7, []

    def launch(dev, fn, o, h, w, t, *rest):
        seen.append((reading(h, (o.N, o.D), (o.hidden_stride,)), reading(w, (o.V, o.D), (o.weight_stride,)), (ctypes.c_int64 * o.N).from_address(t)[:]))
    monkeypatch.setattr(lib, "launch", launch)
    for hook in sorted(HOOKS):
        del seen[:]
        with HOOKS[hook]():
            loss = _LinearCrossEntropy.apply(hidden, weight, target.contiguous(), -100, 0, 0)
        torch.autograd.grad(loss, (hidden, weight), torch.ones(9))
        assert len(seen) == 2
        for h, w, t in seen:
            assert torch.equal(h, hidden.detach()) and torch.equal(w, weight.detach()) and t == target.tolist()


def test_cross_entropy_refuses_other_tensors(calls):
    """A hook that changes more than the layout is refused, not read."""
    from nerf_kinematics_amd.xent import _LinearCrossEntropy
    hidden, weight = torch.randn(8, 64, requires_grad=True), torch.randn(5, 64, requires_grad=True)
    for change in (lambda t: t[:4], lambda t: t.half() if t.is_floating_point() else t.int(), lambda t: t.half() if t.dim() == 2 and len(t) == 8 else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            loss = _LinearCrossEntropy.apply(hidden, weight, torch.zeros(8, dtype=torch.int64), -100, 0, 0)
        with pytest.raises(RuntimeError, match="saved"):
            torch.autograd.grad(loss, (hidden, weight), torch.ones(8))
    assert all(c[0] == "nk_linear_xent_fwd" for c in calls)


def test_scan_values_behind_the_addresses(monkeypatch):
    from nerf_kinematics_amd import lib
    from nerf_kinematics_amd.scan import _GatedScan
    B, T, C, J = 3, 5, 8, 4
    a, x, h0 = torch.rand(B, T, J, requires_grad=True), torch.randn(B, 2 * T, C)[:, ::2].requires_grad_(True), torch.randn(B, C, requires_grad=True)
    lengths, seen = torch.tensor([5, 0, 3], dtype=torch.int32), []
    kept = torch.arange(float(B * C))           # states [B][1][C]

    def launch(dev, fn, o, *args):
        pa, px = args[:2]
        p0 = args[2] if fn.__name__ == "nk_gated_scan_fwd" else args[3]
        seen.append((reading(pa, (B, T, J), (o.a_stride_b, o.a_stride_t)), reading(px, (B, T, C), (o.x_stride_b, o.x_stride_t)),
                     reading(p0, (B, C), (C,)), (ctypes.c_int32 * B).from_address(o.lengths)[:]))
        if fn.__name__ == "nk_gated_scan_fwd":
            ctypes.memmove(args[5], kept.data_ptr(), 4 * B * C)
        else:
            seen.append(reading(args[2], (B * C,), ()))
    monkeypatch.setattr(lib, "launch", launch)
    for hook in sorted(HOOKS):
        del seen[:]
        with HOOKS[hook]():
            h, last = _GatedScan.apply(a, x, h0, lengths, 0)
        torch.autograd.grad((h, last), (a, x, h0), (torch.ones_like(h), torch.ones_like(last)))
        assert len(seen) == 3
        for pa, px, p0, n in seen[:2]:
            assert torch.equal(pa, a.detach()) and torch.equal(px, x.detach()) and torch.equal(p0, h0.detach()) and n == lengths.tolist(), hook
        assert torch.equal(seen[2], kept)


def test_scan_refuses_other_tensors(calls):
    from nerf_kinematics_amd.scan import _GatedScan
    a, x, h0 = torch.rand(3, 5, 4, requires_grad=True), torch.randn(3, 5, 8, requires_grad=True), torch.randn(3, 8, requires_grad=True)
    for change in (lambda t: t[:2], lambda t: t.half(), lambda t: t.bfloat16() if t.shape == x.shape else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            h, last = _GatedScan.apply(a, x, h0, None, 0)
        with pytest.raises(RuntimeError, match="saved"):
            torch.autograd.grad(h, (a, x, h0), torch.ones_like(h))
    assert all(c[0] == "nk_gated_scan_fwd" for c in calls)


@gpu
@pytest.mark.parametrize("hook", sorted(GPU_HOOKS))
@pytest.mark.parametrize("dt", [F32, BF16])
def test_cross_entropy_gradients_under_hooks(dt, hook):
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(2)
    wide, head = torch.randn(130, 192, generator=g, device=dev).to(dt), (torch.randn(700, 192, generator=g, device=dev) / 8).to(dt)
    target = torch.randint(0, 700, (130,), generator=g, device=dev)
    d = torch.randn(130, generator=g, device=dev)

    def run():
        a, b = wide.clone().requires_grad_(True), head.clone().requires_grad_(True)
        loss = nk.linear_cross_entropy(a[:, 64:], b[:, 64:], target, reduction="none")
        return a, b, loss
    a, b, loss = run()
    want = torch.autograd.grad(loss, (a, b), d)
    with GPU_HOOKS[hook]():
        a, b, loss = run()
    got = torch.autograd.grad(loss, (a, b), d)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and bool(want[0].any())


@gpu
@pytest.mark.parametrize("hook", sorted(GPU_HOOKS))
@pytest.mark.parametrize("J", [1, 4, 24])
def test_scan_gradients_under_hooks(J, hook):
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    a0, x0, h0, d, dl = torch.sigmoid(r(3, 200, J)), r(3, 200, 48), r(3, 24), r(3, 200, 24), r(3, 24)
    lengths = torch.tensor([200, 0, 77], dtype=torch.int32, device=dev)

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (a0, x0, h0)]
        return leaves, nk.gated_scan(leaves[0], leaves[1][:, :, 24:], leaves[2], lengths=lengths, reverse=True)
    leaves, out = run()
    want = torch.autograd.grad(out, leaves, (d, dl))
    with GPU_HOOKS[hook]():
        leaves, out = run()
    got = torch.autograd.grad(out, leaves, (d, dl))
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and all(bool(p.any()) for p in want)


@gpu
def test_gradients_under_recomputation():
    """torch's checkpoint hands a backward pass the tensors of a second forward pass."""
    import nerf_kinematics_amd as nk
    from torch.utils.checkpoint import checkpoint
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    alpha, feats, head, labels = torch.sigmoid(r(60, 70, 1)), r(60, 70, 96), r(300, 48) / 7, torch.randint(0, 300, (60,), generator=g, device=dev)

    def loss(a, x, w):
        return nk.linear_cross_entropy(nk.gated_scan(1 - a, a * x[:, :, 48:], reverse=True)[1], w, labels)

    def run(f):
        leaves = [t.clone().requires_grad_(True) for t in (alpha, feats, head)]
        return torch.autograd.grad(f(*leaves), leaves)
    want, got = run(loss), run(lambda *t: checkpoint(loss, *t, use_reentrant=False))
    assert all(torch.equal(p, q) for p, q in zip(want, got)) and all(bool(p.any()) for p in want)
