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
