"""Limits of the cross entropy's call surface: what the Python call takes and refuses, on the host."""
import pytest
import torch

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_rows_far_apart_are_copied(dt):
    """Rows up to 2^22 bytes apart are taken as they lie, others are copied: the library addresses 256 of them with 31 bits."""
    import nerf_kinematics_amd as nk
    from nerf_kinematics_amd.xent import _opts, _rows
    L, most = nk.load(), (1 << 22) // dt.itemsize
    near = torch.empty(2 * most + 16, dtype=dt)
    for step, copied in ((most, False), (most + 8, True), (2 * most, True)):
        t = near.as_strided((2, 16), (step, 1))
        got = _rows(t)
        assert (got is not t) == copied and got.stride() == ((16, 1) if copied else (step, 1))
        o = _opts(got, got, -100, 1, 0)
        for backward in (0, 1):
            assert L.nk_linear_xent_workspace_bytes(o, got.data_ptr(), got.data_ptr(), backward) > 0
    wide = torch.empty(1, 1 << 20, dtype=dt).expand(3, -1)          # as wide as rows may be
    assert L.nk_linear_xent_workspace_bytes(_opts(_rows(wide), _rows(wide), -100, 1, 0), 1024, 1024, 0) > 0


@gpu
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_last_positions_of_long_sequences(dt):
    """hidden = states[:, -1]: rows further apart than 2^22 bytes give the same bits as dense ones."""
    import nerf_kinematics_amd as nk
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(1)
    states = torch.randn(3, (1 << 22) // (64 * dt.itemsize) + 1, 64, generator=g, device=dev).to(dt)
    w, t = (torch.randn(500, 64, generator=g, device=dev) / 8).to(dt), torch.tensor([4, -100, 499], device=dev)
    s, b = states.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = nk.linear_cross_entropy(s[:, -1], b, t)
    ds, db = torch.autograd.grad(got, (s, b))
    h, c = states[:, -1].clone().requires_grad_(True), w.clone().requires_grad_(True)
    want = nk.linear_cross_entropy(h, c, t)
    dh, dc = torch.autograd.grad(want, (h, c))
    assert torch.equal(got, want) and torch.equal(ds[:, -1], dh) and torch.equal(db, dc) and not ds[:, :-1].any() and bool(dh[0].any())


def test_too_many_float32_tokens_are_refused_before_the_forward_pass():
    """float32 gradients: 2^20 tokens a call.  A training call of more is refused where it is made, not in backward(); one
    without gradients, and 16-bit types, get as far as the question of the device (there is none here)."""
    import nerf_kinematics_amd as nk
    N = (1 << 20) + 1
    h, w, t = torch.zeros(1, 8).expand(N, 8), torch.zeros(5, 8), torch.zeros(1, dtype=torch.int64).expand(N)
    leaf = lambda x: x.detach().requires_grad_(True)
    for a, b in ((leaf(h), w), (h, leaf(w)), (leaf(h), leaf(w))):
        with pytest.raises(ValueError, match="float32 gradients"):
            nk.linear_cross_entropy(a, b, t)
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            nk.linear_cross_entropy(a, b, t)
        with pytest.raises(ValueError, match="GPU"):
            nk.linear_cross_entropy(leaf(a.detach()[1:]), b, t[1:])
    with pytest.raises(ValueError, match="GPU"):
        nk.linear_cross_entropy(h, w, t)
    with pytest.raises(ValueError, match="GPU"):
        nk.linear_cross_entropy(leaf(h.to(BF16)), w.to(BF16), t)
    # the limit is the library's
    from nerf_kinematics_amd.xent import _opts
    L = nk.load()
    for n, rc in ((N, -2), (N - 1, 0)):
        got = L.nk_linear_xent_workspace_bytes(_opts(h[:1].expand(n, 8).contiguous(), w, -100, 1, 0), 1024, 1024, 1)
        assert (got == rc) if rc else got > 0


@pytest.mark.parametrize("dt,N,D,V", [(F32, 16, 4096, 131072), (F32, 16, 2048, 65536), (BF16, 16, 4095, 131072), (F16, 3, 8190, 200000), (F32, 1, 1, 1 << 26),
                                      (F32, 2000, 500, 100000), (F32, 8192, 2048, 65536), (BF16, 8192, 2048, 65536), (BF16, 300, 4099, 1 << 20), (F32, 5, 300, 7)])
def test_scratch_of_a_call_that_names_no_piece(dt, N, D, V):
    """Everything that grows with the piece stays within 256 MB (2048 rows at least), the eighth that saves one more piece, and the 256
    rows that a piece is rounded up by, twice: logit gradients (float32: in both orders, of whole steps of tokens), the transposed copy of the weight's rows (float32) and the
    copy of unaligned ones.  What does not grow with it: copies of hidden, and float32 sums of d_hidden (one, or partial ones:
    512 tiles of 64 x 64, of more than 32 tokens 512 of 256 x 256) and likewise of a d_weight that is cut."""
    import nerf_kinematics_amd as nk
    from nerf_kinematics_amd import lib as nklib
    L, es = nk.load(), dt.itemsize
    up = lambda a, b: -(-a // b) * b
    Dp, Np = up(D, 128 // es), up(N, 128 // es)
    o = nklib.NkXentOpts(N, D, V, D, D, -100, nklib.DTYPES[dt], 1, 0)
    unaligned = D * es % 16 != 0
    row = Np * es * (2 if dt == F32 else 1) + (D * es if dt == F32 else 0) + (Dp * es if unaligned else 0)
    fixed = N * Dp * es + D * Np * es + N * D * 4 + 2 * 512 * (256 * 256 if N > 32 else 64 * 64) * 4 + 16 * N + (1 << 16)
    got = L.nk_linear_xent_workspace_bytes(o, 1024, 1024, 1)
    assert 0 < got <= max(256 << 20, 2048 * row) * 9 / 8 + 2 * 256 * row + fixed, (got / 2**20, row, fixed / 2**20)
    got = L.nk_linear_xent_workspace_bytes(o, 1024, 1024, 0)
    assert 0 < got <= N * Dp * es + (V + 255) // 64 * N * 8 + 32 * N + (1 << 16) + (((288 << 20) + 512 * Dp * es) if unaligned else 0)
