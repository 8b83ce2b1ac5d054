"""Tensors that torch negates lazily (the imaginary part of a conjugate, and gradients that come back through one): their memory
holds the opposite sign.  The launch is replaced by a recorder that reads what a call would have read."""
import ctypes

import pytest
import torch


def values(address, n):
    return list((ctypes.c_float * n).from_address(address)) if address else None


@pytest.fixture
def read(monkeypatch):
    """{call: [what lies behind each address of its first float32 operands]}"""
    from nerf_kinematics_amd import lib
    got = {}

    def launch(dev, fn, o, *args):
        name = fn.__name__
        if name.startswith("nk_gated_scan"):
            n = {"nk_gated_scan_fwd": (0, 1, 2), "nk_gated_scan_bwd": (0, 1, 3, 4, 5)}[name]
        else:
            n = {"nk_linear_xent_fwd": (0, 1), "nk_linear_xent_bwd": (0, 1, 4)}[name]
        got[name] = [values(args[i], 1) for i in n]
    monkeypatch.setattr(lib, "launch", launch)
    return got


def lazily(t):
    """`t` as the imaginary part of a conjugate: the same values, the sign bit set aside."""
    out = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert out.is_neg() and torch.equal(out, t)
    return out


def test_scan(read):
    from nerf_kinematics_amd import scan
    one = lambda v, *s: torch.full(s, float(v))
    a, x, h0 = lazily(one(0.5, 1, 1, 1)), lazily(one(2, 1, 1, 1)), lazily(one(3, 1, 1))
    for t in (a, x, h0):
        t.requires_grad_(True)
    h, last = scan._call(a, x, h0, None, 0)
    assert read["nk_gated_scan_fwd"] == [[0.5], [2.0], [3.0]]
    torch.autograd.grad((h, last), (a, x, h0), (lazily(one(5, 1, 1, 1)), lazily(one(7, 1, 1))))
    assert read["nk_gated_scan_bwd"] == [[0.5], [2.0], [3.0], [5.0], [7.0]]
    with torch.no_grad():
        read.clear()
        scan._call(a, x, h0, None, 0)
        assert read["nk_gated_scan_fwd"] == [[0.5], [2.0], [3.0]]


@pytest.mark.parametrize("reduction", [0, 1, 2])
def test_cross_entropy(read, reduction):
    from nerf_kinematics_amd import xent
    h, w, t = lazily(torch.full((1, 1), 2.0)), lazily(torch.full((1, 1), 3.0)), torch.zeros(1, dtype=torch.int64)
    h.requires_grad_(True); w.requires_grad_(True)
    loss = xent._call(h, w, t, -100, reduction, 0)
    assert read["nk_linear_xent_fwd"] == [[2.0], [3.0]]
    torch.autograd.grad(loss, (h, w), lazily(torch.full(loss.shape, 5.0)))
    assert read["nk_linear_xent_bwd"] == [[2.0], [3.0], [5.0]]


def test_a_loss_inside_a_complex_function(read):
    """Where such a gradient comes from: |conj(loss_1 + i loss_2)|."""
    from nerf_kinematics_amd import xent
    h, w, t = torch.full((1, 1), 2.0, requires_grad=True), torch.full((1, 1), 3.0, requires_grad=True), torch.zeros(1, dtype=torch.int64)
    loss = xent._call(h, w, t, -100, 2, 0)
    with torch.no_grad():
        loss.fill_(4.0)
    torch.complex(torch.tensor(3.0), loss).conj().abs().backward()
    assert read["nk_linear_xent_bwd"][2] == [pytest.approx(0.8)]
