"""The training operators together, as a field of labels uses them: features composited along rays by the gated
recurrence, classified by the linear cross entropy, updated by AdamW -- and AdamW as the trainer's optimiser.

Tolerances are those of the single operators (half a step of a type per rounding), carried through the chain by the
reference in 64 bits where a bound is given, or equality of bits where two routes run the same kernels."""
import math
import os

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def nk():
    import nerf_kinematics_amd as m
    return m


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def teacher(dev):
    from nerf_kinematics_amd.datasets import teacher_scene
    return teacher_scene(None, 4, 1, 64, dev)


@gpu
def test_compositing_is_the_reversed_recurrence(nk, dev):
    """h_i = (1 - alpha_i) h_(i+1) + alpha_i c_i from the far sample on gives raw2outputs' colour.  raw2outputs
    multiplies its transmittance with 1 - alpha + 1e-10 and takes 192 products and sums in fp32: both are within
    192 x 4 x 2^-24 + 192 x 1e-10 < 5e-5 of the sum of colours of at most 1."""
    R, n = 301, 192
    g = torch.Generator(device=dev).manual_seed(0)
    raw = torch.randn(R, n, 4, generator=g, device=dev)
    raw[..., 3] *= 3
    z = torch.linspace(2, 6, n, device=dev).expand(R, n).contiguous()
    rays = torch.randn(R, 11, generator=g, device=dev)
    want = nk.raw2outputs(raw, z, rays, nk.make_opts(64, 128))
    dist = torch.cat((z[:, 1:] - z[:, :-1], torch.full((R, 1), 1e10, device=dev)), 1) * rays[:, 3:6].norm(dim=1, keepdim=True)
    alpha = 1 - torch.exp(-torch.relu(raw[..., 3]) * dist)
    rgb = torch.sigmoid(raw[..., :3])
    _, got = nk.gated_scan((1 - alpha)[:, :, None], alpha[:, :, None] * rgb, reverse=True)
    assert float((got - want["rgb"]).abs().max()) < 5e-5


def _chain_reference(feats, alpha, lengths, head, labels):
    """Loss and gradients in 64 bits by autograd."""
    f, w = feats.detach().double().requires_grad_(True), head.detach().double().requires_grad_(True)
    R, n, C = f.shape
    live = (torch.arange(n, device=f.device)[None] < lengths[:, None])[..., None]
    a = torch.where(live, 1 - alpha.double()[..., None], torch.ones((), dtype=torch.float64, device=f.device))
    x = torch.where(live, alpha.double()[..., None] * f, torch.zeros((), dtype=torch.float64, device=f.device))
    h = torch.zeros(R, C, dtype=torch.float64, device=f.device)
    for i in range(n - 1, -1, -1):
        h = a[:, i] * h + x[:, i]
    loss = torch.nn.functional.cross_entropy(h @ w.t(), labels, ignore_index=-100)
    return (loss.detach(),) + torch.autograd.grad(loss, (f, w))


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_label_field_step(nk, dev, bits):
    """One whole step against 64 bits, then twenty steps twice: the same bits, and every value finite.

    The composited features are rounded to bf16 before the head (2^-8 relative) and the head's bf16 gradients once
    more; with logits of size ~1 that moves the loss by less than 2 x 2^-8 and a gradient by less than 4 x 2^-8 of the
    largest magnitude it sums."""
    R, n, C, V = 513, 65, 48, 701
    g = torch.Generator(device=dev).manual_seed(1)
    feats0 = torch.randn(R, n, C, generator=g, device=dev)
    head0 = (torch.randn(V, C, generator=g, device=dev) / C ** 0.5).to(BF16)
    alpha = torch.rand(R, n, generator=g, device=dev) * 0.3
    lengths = torch.randint(0, n + 1, (R,), generator=g, device=dev, dtype=torch.int32)
    labels = torch.randint(0, V, (R,), generator=g, device=dev)
    labels[::7] = -100

    def run(steps):
        feats, head = feats0.clone().requires_grad_(True), head0.clone().requires_grad_(True)
        masters = [head.detach().float()]
        opt_f = nk.AdamW([feats], 1e-2, state_bits=bits)
        opt_h = nk.AdamW([head], 1e-2, masters=masters, state_bits=bits)
        losses = []
        for _ in range(steps):
            _, pixel = nk.gated_scan((1 - alpha)[..., None], alpha[..., None] * feats, lengths=lengths, reverse=True)
            loss = nk.linear_cross_entropy(pixel.to(BF16), head, labels)
            gf, gh = torch.autograd.grad(loss, (feats, head))
            opt_f.step([gf]); opt_h.step([gh])
            losses.append((loss.detach(), gf, gh))
        return feats.detach(), head.detach(), losses
    feats, head, first = run(1)
    loss, gf, gh = first[0]
    rl, rf, rh = _chain_reference(feats0, alpha, lengths, head0, labels)
    assert abs(float(loss) - float(rl)) < 2 * 2.0 ** -8
    assert float((gf.double() - rf).abs().max()) <= 4 * 2.0 ** -8 * float(rf.abs().max())
    assert float((gh.double() - rh).abs().max()) <= 4 * 2.0 ** -8 * float(rh.abs().max())
    # first step of Adam: every element with a gradient moves by lr (1 +- eps / |g| ...), against its gradient
    moved = feats - feats0 * (1 - 1e-2 * 1e-2)
    big = gf.abs() > 1e-6
    assert bool((torch.sign(moved[big]) == -torch.sign(gf[big])).all())
    assert float((moved[big].abs() - 1e-2).abs().max()) < 1.2e-4
    assert float(moved[~big & (gf == 0)].abs().max()) < 1e-6
    a, b = run(20), run(20)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.isfinite(a[0]).all() and torch.isfinite(a[1].float()).all()


def _trainer(nk, dev, bits, rays=512, seed=42, arch=None):
    from nerf_kinematics_amd.trainer import Trainer, TrainOpts
    arch = arch or nk.ARCH_LEGO_CKPT
    return Trainer(arch, arch, TrainOpts(num_coarse=32, num_fine=32, num_random_rays=rays, seed=seed, optimizer="AdamW", weight_decay=0.05,
                                         state_bits=bits), dev)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_with_adamw_graph_equals_eager(nk, dev, teacher, bits):
    from nerf_kinematics_amd.datasets import RaySampler
    from nerf_kinematics_amd.trainer import GraphedStep
    ref, tr = _trainer(nk, dev, bits), _trainer(nk, dev, bits)
    gs, smp = GraphedStep(tr, RaySampler(teacher, 512, seed=3)), RaySampler(teacher, 512, seed=3)
    for i in range(6):
        ref.step(*smp.next(i))
        gs.step()
        torch.zeros(10, device=dev).add_(1).sum().item()        # the program's own work between replays
        for a, b in zip(ref.optimizer_tensors(), tr.optimizer_tensors()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert float(ref.grad.abs().sum()) > 0


@gpu
def test_trainer_adamw_follows_torch(nk, dev, teacher):
    """32-bit moments against torch.optim.AdamW in 64 bits on the same gradients: m and v round 4 times a step
    (2^-24 each), the update 6 times, six steps."""
    from nerf_kinematics_amd.datasets import RaySampler
    from nerf_kinematics_amd.trainer import lr_at
    tr, smp = _trainer(nk, dev, 32), RaySampler(teacher, 512, seed=3)
    p = tr.params.double().requires_grad_(True)
    opt = torch.optim.AdamW([p], lr=tr.opts.lr, betas=tr.opts.betas, eps=tr.opts.eps, weight_decay=0.05)
    for i in range(6):
        opt.param_groups[0]["lr"] = lr_at(tr.iteration, tr.opts)
        tr.step(*smp.next(i))
        p.grad = tr.grad.double()
        opt.step()
    # an element whose gradient cancels to a few units of rounding moves by up to lr in either direction: the bound
    # is relative to the steps taken, 6 x lr x 60 x 2^-24, where the moments themselves are not tiny
    err = (tr.params.double() - p.detach()).abs()
    assert float(err.max()) <= 6 * tr.opts.lr * 60 * 2.0 ** -24 + 4 * 2.0 ** -24 * float(tr.params.abs().max())


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_adamw_resumes_exactly(nk, dev, teacher, tmp_path, bits):
    """A checkpoint holds the moments as fp32; 8-bit ones come back as the values they stood for."""
    from nerf_kinematics_amd import checkpoint as ckpt
    from nerf_kinematics_amd.datasets import RaySampler
    a, smp = _trainer(nk, dev, bits), RaySampler(teacher, 512, seed=3)
    for i in range(5):
        a.step(*smp.next(i))
    path = str(tmp_path / ckpt.checkpoint_name(a.iteration))
    ckpt.save_checkpoint(path, a.export_state(0.1, 10.0), nk.ARCH_LEGO_CKPT, nk.ARCH_LEGO_CKPT, weight_decay=0.05)
    raw = ckpt.load_checkpoint(path)
    assert raw["optimizer_state_dict"]["param_groups"][0]["weight_decay"] == 0.05
    b = _trainer(nk, dev, bits, seed=7)
    b.import_state(ckpt.state_from_checkpoint(raw, nk.ARCH_LEGO_CKPT, nk.ARCH_LEGO_CKPT))
    b.opts.seed = a.opts.seed
    for x, y in zip(a._moments(), b._moments()):
        assert torch.equal(x, y)
    for i in range(5, 8):
        rb, tgt = smp.next(i)
        a.step(rb, tgt); b.step(rb, tgt)
    assert torch.equal(a.params, b.params)
    for x, y in zip(a._moments(), b._moments()):
        assert torch.equal(x, y)


def test_config_keys(golden_dir, tmp_path):
    import yaml
    from nerf_kinematics_amd import config as config_mod
    from nerf_kinematics_amd.trainer import TrainOpts
    with open(os.path.join(golden_dir, "lego-lowres3_config.yml")) as fh:
        cfg = yaml.safe_load(fh)

    def load(**opt):
        c = dict(cfg, optimizer=dict(cfg["optimizer"], **opt))
        path = tmp_path / "c.yml"
        path.write_text(yaml.safe_dump(c))
        return config_mod.load_config(str(path))
    o = TrainOpts.from_config(load())
    assert o.optimizer == "Adam"
    o = TrainOpts.from_config(load(type="AdamW"))
    assert (o.optimizer, o.weight_decay, o.state_bits) == ("AdamW", 0.01, 32)
    o = TrainOpts.from_config(load(type="AdamW", weight_decay=0.1, state_bits=8))
    assert (o.weight_decay, o.state_bits) == (0.1, 8)
    assert TrainOpts.from_config(load(weight_decay=0.1)).optimizer == "Adam"      # read by AdamW alone
    for bad in (dict(type="AdamW", state_bits=16), dict(type="AdamW", weight_decay=-1.0), dict(type="Adamax")):
        with pytest.raises(config_mod.ConfigError, match="optimizer"):
            load(**bad)
