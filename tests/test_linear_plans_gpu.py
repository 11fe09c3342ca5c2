"""K9: every tiling that the host can choose, on sizes for which it chooses it.

tile 32, 64 or 128 weight rows (gated: half of them gate rows) against 128 rows of x,
K over 1 to 8 CTAs of a cluster; one size per tiling with whole 8-byte accesses and one
with an odd number of columns, K ending inside a slice, and where a tiling is chosen for
few slices, CTAs that no slice falls to (9 slices over 4, 49 over 8)."""
import ctypes as C
import math

import pytest
import torch

import a11spec
import layer_reference as R
from a11spec import _lib
from test_layer_ops_gpu import BF, _linear_case, _linear_ref

pytestmark = pytest.mark.gpu

PLANS = [  # gated, tile, split, rows, slices of K, N
    (False, 32, 1, 33, 1, 16), (False, 32, 1, 33, 1, 21), (False, 32, 2, 35, 2, 16), (False, 32, 2, 33, 2, 21),
    (False, 32, 4, 33, 7, 16), (False, 32, 4, 37, 9, 21), (False, 32, 8, 33, 49, 16), (False, 32, 8, 129, 49, 21),
    (False, 64, 1, 33, 1, 4752), (False, 64, 1, 129, 1, 2411), (False, 64, 2, 33, 10, 2560), (False, 64, 2, 135, 10, 1185),
    (False, 64, 4, 35, 19, 1224), (False, 64, 4, 129, 19, 585), (False, 64, 8, 33, 97, 624), (False, 64, 8, 135, 100, 307),
    (False, 128, 1, 35, 35, 10064), (False, 128, 1, 139, 36, 4895), (False, 128, 2, 35, 13, 4840), (False, 128, 2, 131, 12, 2559),
    (False, 128, 4, 35, 28, 2480), (False, 128, 4, 139, 27, 1247), (False, 128, 8, 33, 150, 1232), (False, 128, 8, 145, 151, 635),
    (True, 32, 1, 33, 1, 16), (True, 32, 1, 33, 1, 21), (True, 32, 2, 33, 2, 16), (True, 32, 2, 33, 2, 21),
    (True, 32, 4, 33, 7, 16), (True, 32, 4, 35, 9, 21), (True, 64, 1, 33, 1, 2456), (True, 64, 1, 129, 1, 1189),
    (True, 64, 2, 35, 10, 1232), (True, 64, 2, 131, 10, 679), (True, 64, 4, 35, 19, 648), (True, 64, 4, 131, 19, 309),
    (True, 64, 8, 33, 94, 16), (True, 64, 8, 35, 97, 21), (True, 128, 1, 35, 35, 4832), (True, 128, 1, 133, 35, 2409),
    (True, 128, 2, 33, 12, 2576), (True, 128, 2, 129, 12, 1273), (True, 128, 4, 33, 27, 1272), (True, 128, 4, 141, 29, 613),
    (True, 128, 8, 33, 152, 600), (True, 128, 8, 133, 150, 295),
    (False, 0, 1, 32, 5, 100), (True, 0, 1, 1, 3, 21), (False, 256, 1, 2048, 8, 2048), (True, 256, 1, 1062, 1, 3190),
]


def _plan(e4m3, rows, K, N, gated):
    tile, split = C.c_int32(-1), C.c_int32(-1)
    _lib.check(_lib.lib.a11s_linear_plan(_lib.E4M3 if e4m3 else _lib.BF16, rows, K, N, int(gated), C.byref(tile), C.byref(split)))
    return tile.value, split.value


@pytest.mark.parametrize("gated,tile,split,rows,slices,N", PLANS)
@pytest.mark.parametrize("e4m3", [False, True])
def test_linear_plan(dev, gated, tile, split, rows, slices, N, e4m3):
    K = 128 * slices - 48 if e4m3 else 64 * slices - 24
    assert _plan(e4m3, rows, K, N, gated) == (tile, split)
    for activation, bias, residual in (("silu", False, True), ("gelu", True, False)) if gated else ((None, False, False), ("gelu", True, True)):
        x, w, kw = _linear_case(rows + 7 * K + 31 * N, rows, K, N, e4m3, gated, bias, residual)
        ref, tol = _linear_ref(x, w, kw, activation)
        buf = torch.full((rows + 2, N), math.nan, dtype=BF, device="cuda")  # a row before and one behind stay
        y = a11spec.linear(x, w, activation=activation, out=buf[1:-1], check_status=True, **kw)
        r = R.worst(y, ref, tol)
        assert r <= 1, (activation, r)
        assert bool(buf[0].isnan().all()) and bool(buf[-1].isnan().all())
        assert torch.equal(y, a11spec.linear(x, w, activation=activation, **kw))  # equal calls, equal bits


def test_every_tiling_is_among_them():
    """All that choose() can give: every tile width with every split, but for gated 32-row tiles over 8."""
    want = {(g, t, s) for g in (False, True) for t in (32, 64, 128) for s in (1, 2, 4, 8)} - {(True, 32, 8)}
    want |= {(g, t, 1) for g in (False, True) for t in (0, 256)}
    assert {p[:3] for p in PLANS} == want


@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 24, 25, 32])
@pytest.mark.parametrize("K,N", [(2112, 4741), (272, 5000), (288, 4735), (4112, 83), (1040, 2048)])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_streamed_weights(dev, rows, K, N, e4m3, gated):
    """Every number of row tiles, one and two column tiles a block (N from 32 * 148 on), 8 and
    16 warps (few blocks over a long K), rows in whole 32-byte pieces and not, and the largest
    exchange of sums."""
    activation, bias, residual = ("silu", True, True) if gated else ("gelu", True, True)
    assert _plan(e4m3, rows, K, N, gated) == (0, 1)
    x, w, kw = _linear_case(rows + 7 * K + 31 * N, rows, K, N, e4m3, gated, bias, residual)
    ref, tol = _linear_ref(x, w, kw, activation)
    buf = torch.full((rows + 2, N), math.nan, dtype=BF, device="cuda")
    y = a11spec.linear(x, w, activation=activation, out=buf[1:-1], check_status=True, **kw)
    r = R.worst(y, ref, tol)
    assert r <= 1, r
    assert bool(buf[0].isnan().all()) and bool(buf[-1].isnan().all())
    assert torch.equal(y, a11spec.linear(x, w, activation=activation, **kw))
