"""Gradients of single losses (``reduction="none"``) where one of them is not finite."""
import pytest
import torch

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("N", [20, 9001])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_one_gradient_that_is_not_finite(dt, N, bad):
    """It makes its own row and the whole of d_weight what 0 * inf and NaN make them, and leaves the other rows of d_hidden alone: their
    common factor is the power of two above the largest finite |d_loss|, so they are the same bits as with 0 in its place."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(N)
    h = torch.randn(N, 64, generator=g, device=dev).to(dt)
    w = (torch.randn(300, 64, generator=g, device=dev) / 8).to(dt)
    t = torch.randint(0, 300, (N,), generator=g, device=dev)
    d = torch.rand(N, generator=g, device=dev) + 0.5

    def run(at):
        a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        x = d.clone()
        x[7] = at
        return torch.autograd.grad(nk.linear_cross_entropy(a, b, t, reduction="none"), (a, b), x)
    (want, _), (got, got_w) = run(0.0), run(bad)
    rest = torch.arange(N, device=dev) != 7
    assert torch.equal(got[rest], want[rest]) and bool(want[rest].any(1).all())
    assert not torch.isfinite(got[7].float()).any() and not torch.isfinite(got_w.float()).any()
    assert not want[7].any()
