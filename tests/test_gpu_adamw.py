"""AdamW over many tensors (nk_adamw_step) against a plain implementation in 64 bits.

Tolerances.  One step in fp32 rounds each of m (3 operations), v (4) and the update (6) by at most 2^-24
relative to its largest operand, so the results are held to 8 x 2^-24 of the magnitudes that enter; a bf16 /
fp16 parameter is one rounding (2^-8 / 2^-11 relative, half a step) away from its fp32 value.  An 8-bit code is
one of the two neighbours of the exact value, chosen by the 16 random bits; the choice is recomputed here and may
differ only where the fp32 value lies within 2^-20 of the threshold."""
import math

import pytest
import torch

gpu = pytest.mark.gpu

B1, B2, EPS, LR, WD = 0.9, 0.999, 1e-8, 3e-3, 0.02
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZES = [1, 3, 4, 255, 256, 257, 1000, 4095, 4096, 4097, 20011]


def reference(p, g, m, v, step, grad_scale=1.0):
    g = g.double() * grad_scale
    m = B1 * m.double() + (1 - B1) * g
    v = B2 * v.double() + (1 - B2) * g * g
    up = LR * (m / (1 - B1 ** step)) / ((v / (1 - B2 ** step)).sqrt() + EPS)
    return p.double() * (1 - LR * WD) - up, m, v, up


def close(got, want, tol, slack):
    """|got - want| <= tol |want| + slack elementwise (NaN never passes)."""
    err = (got.double() - want).abs()
    bound = tol * want.abs() + slack
    assert bool((err <= bound).all()), f"worst excess {float((err - bound).max()):.3e}"


def make(sizes, dtype, gdtype, seed, offset=0):
    """Parameter and gradient lists cut out of flat buffers `offset` elements behind an aligned address."""
    gen = torch.Generator().manual_seed(seed)
    cut = lambda t: list(t[offset:].split(sizes))
    total = sum(sizes) + offset
    dev = torch.device("cuda:0")
    r = lambda s: torch.randn(total, generator=gen) * s
    return (cut(r(0.1).to(dev, dtype)), cut(r(1e-2).to(dev, gdtype)), cut(r(1e-3).to(dev)), cut((r(1e-2) ** 2).to(dev)))


@gpu
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32)])
def test_step_matches_the_formula(dtype, gdtype, offset):
    import nerf_kinematics_amd as nk
    p, g, m, v = make(SIZES, dtype, gdtype, 1, offset)
    before = [t.clone() for t in p], [t.clone() for t in m], [t.clone() for t in v]
    nk.adamw_step(p, g, m, v, 7, LR, (B1, B2), EPS, WD, grad_scale=0.5)
    for i in range(len(SIZES)):
        rp, rm, rv, up = reference(before[0][i], g[i], before[1][i], before[2][i], 7, 0.5)
        u = 2.0 ** -24
        close(m[i], rm, 0, 8 * u * (before[1][i].double().abs() + g[i].double().abs()))
        close(v[i], rv, 8 * u, 1e-40)
        close(p[i], rp, HALF[dtype], 8 * u * (before[0][i].double().abs() + 2 * up.abs()) + (2.0 ** -25 if dtype == torch.float16 else 0))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [32, 8])
def test_masters_are_updated_and_rounded_into_the_parameters(dtype, bits):
    import nerf_kinematics_amd as nk
    p, g, _, _ = make(SIZES, dtype, dtype, 2)
    w = [t.float() + 1e-4 for t in p]
    keep = [t.clone() for t in w]
    opt = nk.AdamW(p, LR, (B1, B2), EPS, WD, masters=w, state_bits=bits)
    opt.step(g)
    for i in range(len(SIZES)):
        z = torch.zeros_like(keep[i])
        rp, _, _, up = reference(keep[i], g[i], z, z, 1)
        close(w[i], rp, 2.0 ** -24, 8 * 2.0 ** -24 * (keep[i].double().abs() + 2 * up.abs()))
        assert torch.equal(p[i], w[i].to(dtype))


def codes_reference(x, part, mant, least, top):
    """(lower neighbour, upper neighbour, fraction) of every |x| on its block's grid, and the scales."""
    n = x.numel()
    b = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256)
    frac, e = torch.frexp(b.amax(1))
    e = torch.where(frac == 0, torch.full_like(e, -100), e - (frac == 0.5).to(e.dtype) - top).clamp_min(-100)
    unit = torch.exp2(e.double())
    y = x.abs() / unit.repeat_interleave(256)[:n]
    grid = torch.exp2((torch.frexp(y)[1].double() - 1).clamp_min(least) - mant)
    low = torch.floor(y / grid) * grid
    return y, low, grid, unit


def random_bits(seed, n):
    M = 0xFFFFFFFF

    def mix(x):
        x = x ^ (x >> 16); x = (x * 0x7FEB352D) & M
        x = x ^ (x >> 15); x = (x * 0x846CA68B) & M
        return x ^ (x >> 16)
    key = mix(torch.tensor((seed ^ (5 * 0x85EBCA6B)) & M))
    return mix((torch.arange(n) * 0x9E3779B9 + key) & M)


@gpu
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_eight_bit_moments(dtype, offset):
    import nerf_kinematics_amd as nk
    p, g, m32, v32 = make(SIZES, dtype, dtype, 3, offset)
    m, v, scales = [], [], []
    for a, b in zip(m32, v32):
        cm, sm = nk.encode_moment(a, torch.float8_e4m3fn)
        cv, sv = nk.encode_moment(b, torch.float8_e5m2)
        if offset:      # codes at an odd address
            cm, cv = (torch.cat((c[:1], c))[1:] for c in (cm.view(torch.uint8), cv.view(torch.uint8)))
            cm, cv = cm.view(torch.float8_e4m3fn), cv.view(torch.float8_e5m2)
        m.append(cm); v.append(cv); scales.append((sm, sv))
    dm, dv = [nk.decode_moment(a, s[0]) for a, s in zip(m, scales)], [nk.decode_moment(a, s[1]) for a, s in zip(v, scales)]
    keep = [t.clone() for t in p]
    seed = 12345
    nk.adamw_step(p, g, m, v, 9, LR, (B1, B2), EPS, WD, scales=scales, seed=seed)
    for i, n in enumerate(SIZES):
        rp, rm, rv, up = reference(keep[i], g[i], dm[i], dv[i], 9)
        u = 2.0 ** -24
        close(p[i], rp, HALF[dtype], 8 * u * (keep[i].double().abs() + 2 * up.abs()))
        r = random_bits(seed, n).to(p[i].device).double()
        for x, parts, code, scale, part, mant, least, top in (
                (rm, dm[i].double().abs() + g[i].double().abs(), m[i], scales[i][0], r % 65536, 3, -6, 8),
                (rv, rv, v[i], scales[i][1], torch.floor(r / 65536), 2, -14, 15)):
            y, low, grid, unit = codes_reference(x, part, mant, least, top)
            assert torch.equal(scale.double(), unit)
            got = code.double().abs()
            # the value before rounding is fp32: off by at most 8 u of the operands that made it
            near = 8 * u * (parts + x.abs()) / unit.repeat_interleave(256)[:n] / grid
            frac = (y - low) / grid + part / 65536
            up_wanted, sure = frac >= 1, (frac - 1).abs() > near + 2.0 ** -20
            want = torch.where(up_wanted, low + grid, low)
            if mant == 2:
                want = torch.where((y > 0) & (want == 0), grid, want)
            assert bool((got == want)[sure].all())
            assert bool(((got == low) | (got == low + grid)).all())
            assert int(sure.sum()) > 0.99 * n
        assert bool(((m[i].double() < 0) == (rm < 0))[m[i].double() != 0].all())


@gpu
def test_stochastic_rounding_lets_a_second_moment_decay():
    """With zero gradients v decays by b2 per step: rounding to nearest would keep it for ever.  The mean over n
    elements is within 5 standard deviations of b2^steps (per step variance <= value * spacing * drift)."""
    import nerf_kinematics_amd as nk
    n, steps = 1 << 16, 200
    dev = torch.device("cuda:0")
    p, g = [torch.zeros(n, device=dev)], [torch.zeros(n, device=dev)]
    cv, sv = nk.encode_moment(torch.ones(n, device=dev), torch.float8_e5m2)
    m, v, scales = nk.adamw_state(p, 8)
    v, scales = [cv], [(scales[0][0], sv)]
    opt = nk.AdamW(p, LR, (B1, B2), EPS, WD, state=(m, v, scales))
    for _ in range(steps):
        opt.step(g)
    got = float(nk.decode_moment(v[0], scales[0][1]).double().mean())
    want = B2 ** steps
    sd = math.sqrt(steps * 0.001 * 0.25 / n)
    assert abs(got - want) < 5 * sd + 1e-4, (got, want, sd)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_special_values(bits):
    """Zero gradients leave zero moments zero; infinities and NaN stay in their element (32 bits) or block (8)."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    n = 1000
    p, g = [torch.ones(n, device=dev)], [torch.zeros(n, device=dev)]
    opt = nk.AdamW(p, LR, (B1, B2), EPS, WD, state_bits=bits)
    opt.step(g)
    assert torch.allclose(p[0], torch.full_like(p[0], 1 - LR * WD), rtol=2 ** -23, atol=0)
    assert not opt.exp_avgs[0].float().any() and not opt.exp_avg_sqs[0].float().any()
    g[0][300], g[0][301], g[0][700] = float("inf"), float("nan"), 1e-30
    opt.step(g)
    bad = torch.zeros(n, dtype=torch.bool, device=dev)
    bad[300:302] = True
    assert torch.equal(torch.isnan(p[0]), bad)
    opt.step([torch.zeros(n, device=dev)])
    if bits == 32:
        assert torch.equal(~torch.isfinite(p[0]), bad)
    else:
        block = torch.zeros_like(bad); block[256:512] = True
        assert torch.equal(~torch.isfinite(p[0]), block)


@gpu
def test_many_tensors_empty_ones_and_chunks():
    """More tensors than one launch holds, empty ones between them: the same as one by one."""
    import nerf_kinematics_amd as nk
    sizes = [(37 * i) % 700 for i in range(131)]
    a, b = make(sizes, torch.float32, torch.float32, 4), make(sizes, torch.float32, torch.float32, 4)
    nk.adamw_step(*a, 3, LR, (B1, B2), EPS, WD)
    for k in range(len(sizes)):
        if sizes[k]:
            nk.adamw_step([b[0][k]], [b[1][k]], [b[2][k]], [b[3][k]], 3, LR, (B1, B2), EPS, WD)
    for x, y in zip(a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, y))


@gpu
def test_equals_adam_without_decay():
    """weight_decay = 0: AdamW is Adam; the existing flat update is within its own rounding (8 units of 2^-24)."""
    import nerf_kinematics_amd as nk
    p, g, m, v = (t[0] for t in make([5000], torch.float32, torch.float32, 5))
    q, mq, vq = p.clone(), m.clone(), v.clone()
    nk.adamw_step([p], [g], [m], [v], 4, LR, (B1, B2), EPS, 0.0)
    nk.adam_step(q, g, mq, vq, 4, LR, (B1, B2), EPS)
    close(p, q.double(), 8 * 2.0 ** -24, 8 * 2.0 ** -24 * LR * 10)
    close(v, vq.double(), 4 * 2.0 ** -24, 1e-40)


@gpu
def test_default_gradients_streams_and_graph_replay():
    import nerf_kinematics_amd as nk
    from nerf_kinematics_amd import lib as nklib
    import ctypes as C
    dev = torch.device("cuda:0")
    leaves = [torch.randn(300, device=dev, requires_grad=True), torch.randn(77, device=dev, requires_grad=True)]
    with pytest.raises(ValueError):
        nk.AdamW(leaves).step()
    sum((t ** 2).sum() for t in leaves).backward()
    side = torch.cuda.Stream(dev)
    copy = [t.detach().clone() for t in leaves]
    opt, other = nk.AdamW(leaves, 1e-2, state_bits=8), nk.AdamW(copy, 1e-2, state_bits=8)
    grads = [t.grad.clone() for t in leaves]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        opt.step()
    side.synchronize()
    other.step(grads)
    assert all(torch.equal(a.detach(), b) for a, b in zip(leaves, copy))
    # a captured step reads its scalars from device memory: three replays equal three eager steps
    state, host = torch.zeros(C.sizeof(nklib.NkStepState), dtype=torch.uint8, device=dev), nklib.NkStepState()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            opt.step(grads, step_state=state.data_ptr())
    L = nk.load()
    for step in (2, 3, 4):
        host.adam_step_size, host.adam_bc2_sqrt = 1e-2 / (1 - B1 ** step), math.sqrt(1 - B2 ** step)
        host.adamw_decay, host.render_seed = 1e-2 * 1e-2, 77 + step
        nklib.check(L.nk_set_step_state(host, state.data_ptr(), torch.cuda.current_stream(dev).cuda_stream))
        graph.replay()
        torch.zeros(1000, device=dev).add_(1).sum().item()      # the program's own eager work between the replays
        other.step(grads, step=step, seed=77 + step)
        torch.cuda.synchronize()
        assert torch.equal(opt.exp_avgs[0].view(torch.uint8), other.exp_avgs[0].view(torch.uint8))
        # 1 - float(lr wd) in fp32 against float(1 - lr wd): at most one rounding apart
        assert all(torch.allclose(a.detach(), b, rtol=2 ** -21, atol=1e-7) for a, b in zip(leaves, copy))


@gpu
def test_parameters_that_move():
    """A parameter or master whose storage is replaced is updated where it is now; the old storage is left alone."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    p = [torch.randn(n, device=dev) for n in (300, 5)]
    low = [t.bfloat16() for t in p]
    g = [torch.randn_like(t) for t in p]
    still, stay, moved = [t.clone() for t in p], [t.clone() for t in low], [t.clone() for t in p]
    a, b = nk.AdamW(stay, 1e-2, masters=still), nk.AdamW(low, 1e-2, masters=moved)
    a.step(g); b.step(g)
    old = low[0].data, moved[1].data
    kept = [t.clone() for t in old]
    low[0].data, moved[1].data = low[0].data.clone(), moved[1].data.clone()
    a.step(g); b.step(g)
    assert all(torch.equal(x, y) for x, y in zip(stay + still, low + moved))
    assert all(torch.equal(x, y) for x, y in zip(old, kept)) and not torch.equal(old[0], low[0])
    low[1].data = torch.zeros(6, device=dev, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="elements"):
        b.step(g)
    low[1].data = low[0].data[:5]
    with pytest.raises(ValueError, match="overlap"):
        b.step(g)


@gpu
def test_autograd_notices_the_step():
    import nerf_kinematics_amd as nk
    p = torch.randn(40, device="cuda:0", requires_grad=True)
    opt = nk.AdamW([p])
    loss = (p * p).sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with pytest.raises(ValueError, match="grads"):
        opt.step([None])
    with pytest.raises(ValueError, match="grads"):
        opt.step([p.detach()[::2]])


def test_moment_codec_round_trip():
    from nerf_kinematics_amd.optim import decode_moment, encode_moment
    gen = torch.Generator().manual_seed(0)
    for n in (1, 255, 256, 257, 3000):
        # below the smallest normal value codes are 2^-9 (e4m3) / 2^-16 (e5m2) apart and the block's largest is above
        # 2^7 / 2^14: half a spacing is 2^-17 of it for e4m3; a positive e5m2 value becomes at least one
        # whole spacing, 2^-30 of it
        x = torch.randn(n, generator=gen) * torch.exp2(torch.randint(-20, 20, (n,), generator=gen).float())
        for dt, val, half, low in ((torch.float8_e4m3fn, x, 2.0 ** -4, 2.0 ** -17), (torch.float8_e5m2, x * x, 2.0 ** -3, 2.0 ** -30)):
            c, s = encode_moment(val, dt)
            d = decode_moment(c, s)
            big = torch.nn.functional.pad(val.abs(), (0, -n % 256)).view(-1, 256).amax(1).repeat_interleave(256)[:n]
            assert bool(((d - val).abs() <= half * val.abs() + low * big).all())
            again = decode_moment(*encode_moment(d, dt))
            assert torch.equal(d, again)
            if dt == torch.float8_e5m2:
                assert bool((d > 0)[val > 0].all())
    assert not decode_moment(*encode_moment(torch.zeros(300), torch.float8_e5m2)).any()


def test_refusals_on_the_host():
    """Every refusal is raised by the host before anything is launched (no GPU here)."""
    import ctypes as C
    import nerf_kinematics_amd as nk
    from nerf_kinematics_amd import lib as nklib
    with pytest.raises(ValueError, match="GPU"):
        nk.AdamW([torch.zeros(4)])
    with pytest.raises(ValueError, match="no parameters"):
        nk.AdamW([])
    with pytest.raises(ValueError, match="dtype"):
        nk.AdamW([torch.zeros(4, dtype=torch.float64)])
    with pytest.raises(ValueError):
        nk.adamw_state([torch.zeros(3)], 16)
    L = nk.load()
    t = (nklib.NkAdamwTensor * 1)(nklib.NkAdamwTensor(0, 0, 0, 0, 0, 0, 0, 4))
    o = nklib.NkAdamwOpts(0, 0, 32, 0, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 0, None)
    assert L.nk_adamw_step(t, 1, o, None) == -1 and b"null pointer" in L.nk_last_error()
    assert L.nk_adamw_step(None, 1, o, None) == -1
    assert L.nk_adamw_step(t, -1, o, None) == -1
    for field, value, rc in (("state_bits", 16, -2), ("param_dtype", 7, -1), ("grad_dtype", 1, -2), ("step", 0, -1), ("beta1", 1.0, -1)):
        bad = nklib.NkAdamwOpts.from_buffer_copy(o)
        setattr(bad, field, value)
        assert L.nk_adamw_step(t, 1, bad, None) == rc, field
    far = (nklib.NkAdamwTensor * 1)(nklib.NkAdamwTensor(8, 8, 8, 8, 0, 0, 0, 1 << 34))
    assert L.nk_adamw_step(far, 1, o, None) == -2 and b"too large" in L.nk_last_error()
    t[0].n = -1
    assert L.nk_adamw_step(t, 1, o, None) == -1
    t[0].n = 0
    assert L.nk_adamw_step(t, 1, o, None) == 0 and L.nk_adamw_step(None, 0, o, None) == 0
