"""What an AdamW object reads at each step, and what it tells autograd."""
import pytest
import torch

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_settings_changed_between_steps(bits):
    """lr, betas, eps and weight_decay assigned between two steps are those of the next one: the same bits as an object that was
    made with them and given the state."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(1)
    r = lambda: [torch.randn(n, generator=gen, device=dev) for n in (300, 7)]
    p, g1, g2 = r(), r(), r()
    opt = nk.AdamW(p, 1e-2, (0.9, 0.999), 1e-8, 0.01, state_bits=bits, seed=3)
    opt.step(g1)
    copy = lambda ts: [t.clone() for t in ts]
    q, scales = copy(p), None if bits == 32 else [tuple(copy(s)) for s in opt.scales]
    other = nk.AdamW(q, 2e-2, (0.5, 0.9), 1e-3, 0.1, state=(copy(opt.exp_avgs), copy(opt.exp_avg_sqs), scales), seed=3)
    same, s2 = copy(p), None if bits == 32 else [tuple(copy(s)) for s in opt.scales]
    before = nk.AdamW(same, 1e-2, (0.9, 0.999), 1e-8, 0.01, state=(copy(opt.exp_avgs), copy(opt.exp_avg_sqs), s2), seed=3)
    opt.lr, opt.betas, opt.eps, opt.weight_decay = 2e-2, (0.5, 0.9), 1e-3, 0.1
    opt.step(g2); other.step(g2, step=2); before.step(g2, step=2)
    for a, b, c in zip(p, q, same):
        assert torch.equal(a, b) and not torch.equal(a, c)
    for a, b in zip(opt.exp_avgs + opt.exp_avg_sqs, other.exp_avgs + other.exp_avg_sqs):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for name, bad in (("betas", (1.0, 0.9)), ("betas", (0.9, -0.1)), ("eps", -1.0)):
        keep, was = getattr(opt, name), copy(p)
        setattr(opt, name, bad)
        with pytest.raises(ValueError):
            opt.step(g2)
        setattr(opt, name, keep)
        assert all(torch.equal(a, b) for a, b in zip(p, was)) and opt.steps == 2


@gpu
def test_autograd_notices_that_masters_changed():
    """A master is updated in place as a parameter is: what autograd saved of either must not be used afterwards."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    w = torch.randn(40, device=dev, requires_grad=True)
    p = w.detach().bfloat16()
    opt = nk.AdamW([p], 1e-2, masters=[w])
    loss = (w * w).sum()
    opt.step([torch.ones(40, device=dev)])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def lazily(t):
    """`t` as the imaginary part of a conjugate: the same values, negated lazily."""
    out = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert out.is_neg()
    return out


@gpu
@pytest.mark.parametrize("shape", [(), (1,), (1, 1)])
def test_gradients_that_torch_negates_lazily(shape):
    """Only a tensor of one element can be both such a view and contiguous; autograd leaves such a .grad behind a complex loss."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    start = lambda: [torch.ones(5, device=dev), torch.full(shape, 2.0, device=dev, requires_grad=True)]
    p, q = start(), start()
    torch.complex(torch.full(shape, 3.0, device=dev), p[1]).conj().abs().sum().backward()
    assert p[1].grad.is_neg() and float(p[1].grad) > 0
    p[0].grad = torch.ones(5, device=dev)
    nk.AdamW(p, 1e-2).step()
    nk.AdamW(q, 1e-2).step([torch.ones(5, device=dev), p[1].grad.clone().resolve_neg()])
    assert all(torch.equal(a, b) for a, b in zip(p, q)) and float(p[1].detach()) < 2.0


def test_parameters_that_torch_negates_lazily_are_refused():
    from nerf_kinematics_amd.optim import _check_list
    for t in (lazily(torch.ones(())), lazily(torch.ones(1))):
        with pytest.raises(ValueError, match="resolve_neg"):
            _check_list("params", [torch.ones(3), t], [3, 1], torch.float32, t.device, [])
