"""The operators have first-order gradients only: an input with a forward-mode tangent is refused, whatever else requires a
gradient.  A result without a tangent would be read as a derivative of zero."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_scan_refuses_tangents(which, requires_grad):
    import nerf_kinematics_amd as nk
    args = [torch.rand(2, 3, 4), torch.randn(2, 3, 8), torch.randn(2, 8)]
    for t in args:
        t.requires_grad_(requires_grad)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="GPU"):         # none of them has a tangent
            nk.gated_scan(*args)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nk.gated_scan(*args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            nk.gated_scan(*args)


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("which", [0, 1])
def test_cross_entropy_refuses_tangents(which, requires_grad):
    import nerf_kinematics_amd as nk
    args = [torch.randn(4, 8), torch.randn(5, 8), torch.zeros(4, dtype=torch.int64)]
    for t in args[:2]:
        t.requires_grad_(requires_grad)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="GPU"):
            nk.linear_cross_entropy(*args)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nk.linear_cross_entropy(*args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            nk.linear_cross_entropy(*args)


def test_functional_jvp_is_refused():
    import nerf_kinematics_amd as nk
    a, x, w, t = torch.rand(2, 3, 4), torch.randn(2, 3, 4), torch.randn(5, 4), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda y: nk.gated_scan(a, y)[0], (x,), (x,))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda y: nk.linear_cross_entropy(y, w, t), (x[:, 0],), (x[:, 0],))


def test_second_derivatives_are_refused(monkeypatch):
    """create_graph=True gives first gradients that cannot be differentiated again."""
    from nerf_kinematics_amd import lib
    from nerf_kinematics_amd.scan import _GatedScan
    from nerf_kinematics_amd.xent import _LinearCrossEntropy
    monkeypatch.setattr(lib, "launch", lambda *args: None)
    a, x = torch.rand(2, 3, 4, requires_grad=True), torch.randn(2, 3, 4, requires_grad=True)
    h, w = torch.randn(4, 8, requires_grad=True), torch.randn(5, 8, requires_grad=True)
    for out, inp in ((_GatedScan.apply(a, x, None, None, 0)[0], x), (_LinearCrossEntropy.apply(h, w, torch.zeros(4, dtype=torch.int64), -100, 0, 0), h)):
        weight = torch.ones_like(out, requires_grad=True)
        (g,) = torch.autograd.grad(out, inp, weight, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            g.sum().backward()
