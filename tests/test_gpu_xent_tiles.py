"""Every tile of the cross entropy's products, in every type, against the definition in 64 bits (tolerances: test_gpu_xent).

Which tile a shape takes is the library's answer (nk_linear_xent_cuts): a rule that changes makes the list of variants fail on the
host rather than leave one untested."""
import ctypes

import pytest
import torch

from test_gpu_xent import BF16, F16, F32, check, make

gpu = pytest.mark.gpu
TILES = ("256x256", "128x128", "128x32", "64x64")

#         N      D     V   piece
SHAPES = [(4100, 528, 3600, 0),         # logits and their gradients in large tiles, the last ones partly empty
          (19200, 72, 523, 0),
          (1664, 320, 2048, 0),         # in middle ones
          (70, 2048, 7300, 0),          # d_weight in large tiles
          (40, 1040, 3200, 0),          # in middle ones
          (10400, 1936, 1588, 0),       # cut into stretches of tokens: large
          (1760, 1764, 566, 0),         # middle
          (979, 16, 2, 0),              # few labels
          (19153, 528, 13, 0),          # d_hidden by itself in large tiles
          (3300, 1040, 300, 0),         # in middle ones
          (3937, 1878, 4126, 0),        # cut into stretches of the vocabulary: large
          (1088, 960, 2100, 0),         # middle
          (7700, 1968, 600, 256),       # summed over pieces: large
          (3300, 1040, 700, 256),       # middle
          (20, 80, 3000, 0), (20, 80, 3000, 256), (3, 24, 50, 0), (300, 33, 500, 0), (300, 64, 1300, 0), (300, 64, 1300, 512), (1100, 24, 40, 0), (50, 40, 12, 0)]


def variants(N, D, V, piece, dt):
    """(product, tile, form) of every product of a call with both gradients."""
    import nerf_kinematics_amd as nk
    from nerf_kinematics_amd import lib as nklib
    L, o, cuts, out, i, n = nk.load(), nklib.NkXentOpts(N, D, V, D, D, -100, nklib.DTYPES[dt], 1, piece), (ctypes.c_int32 * 4)(), set(), 0, 1
    while i < n:
        n = nklib.check(L.nk_linear_xent_cuts(o, 1024, 1024, i, cuts))
        tile, parts = [TILES[c % 16] for c in cuts], [c // 16 for c in cuts]
        out |= {("logits", tile[0], ""), ("logit gradients", tile[1], ""), ("d_weight", tile[2], "sums" if parts[2] else "direct"),
                ("d_hidden", tile[3], "pieces" if n > 1 else "sums" if parts[3] else "direct")}
        i += 1
    return out


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_the_shapes_take_every_variant(dt):
    want = {(p, t, "") for p in ("logits", "logit gradients") for t in TILES}
    want |= {("d_weight", t, f) for t in TILES for f in ("direct", "sums")} | {("d_hidden", t, f) for t in TILES for f in ("direct", "sums", "pieces")}
    got = set().union(*(variants(*s, dt) for s in SHAPES))
    assert got == want, (want - got, got - want)


def test_refusals_of_the_query():
    import nerf_kinematics_amd as nk
    from nerf_kinematics_amd import lib as nklib
    L, cuts = nk.load(), (ctypes.c_int32 * 4)()
    o = lambda **k: nklib.NkXentOpts(**{**dict(N=4, D=8, V=5, hidden_stride=8, weight_stride=8, ignore_index=-100, dtype=1, reduction=1), **k})
    assert L.nk_linear_xent_cuts(o(), 1024, 1024, 0, cuts) == 1
    assert L.nk_linear_xent_cuts(o(V=1000, piece=256), 1024, 1024, 3, cuts) == 4
    for opts, piece, to, rc in ((o(), 1, cuts, -1), (o(), -1, cuts, -1), (o(), 0, None, -1), (o(N=0), 0, cuts, -1), (o(D=0), 0, cuts, -1), (o(V=1 << 27), 0, cuts, -2)):
        assert L.nk_linear_xent_cuts(opts, 1024, 1024, piece, to) == rc


@gpu
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_variants(shape, dt):
    N, D, V, piece = shape
    k = SHAPES.index(shape)
    h, w, t, g = make(N, D, V, dt, 40 + k)
    check(h, w, t, ("mean", "none", "sum")[k % 3], g, piece=piece)
