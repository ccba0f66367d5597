"""Tiles of the gated block's products whose last rows and columns end inside a warp, so that lanes of one warp go different ways in
front of what only a whole warp may do (reads of tensor memory, the barrier of a cluster): by one CTA a tile, by pairs, and split
along k between two, four and eight CTAs.  Bounds as in test_gpu_gated_ffn.py; every call of a case gives the same bits."""
import pytest
import torch

from test_gpu_gated_ffn import _check, _formula, _inputs, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["silu", "relu"])
@pytest.mark.parametrize("rows,n_in,n_mid,n_out", [(33, 4096, 1032, 24), (45, 2056, 4104, 40), (77, 520, 5640, 200), (97, 72, 2056, 8),
                                                   (129, 1096, 2056, 72), (333, 776, 2056, 776), (333, 2056, 5640, 2056),
                                                   (601, 4096, 4104, 1032)])
def test_split_tiles(rows, n_in, n_mid, n_out, act):
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, _ = _inputs(rows, n_in, n_mid, n_out, torch.bfloat16, 37)
    for residual in (None, r):
        with torch.no_grad():
            got = gated_feed_forward(x, wg, wu, wd, act, residual)
            _within(got, _formula(x, wg, wu, wd, act, residual, None)["y"], "y")
            for _ in range(20):
                assert torch.equal(gated_feed_forward(x, wg, wu, wd, act, residual), got)
        kept = gated_feed_forward(x, wg.clone().requires_grad_(), wu, wd, act, residual)
        assert torch.equal(kept.detach(), got)


@pytest.mark.parametrize("rows,n_in,n_mid,n_out", [(35, 72, 40, 24), (131, 136, 72, 200), (1300, 520, 1048, 1032), (4999, 264, 2056, 520),
                                                   (9001, 1032, 1544, 264)])
def test_whole_tiles_and_gradients(rows, n_in, n_mid, n_out):
    for with_residual in (False, True):
        _check(rows, n_in, n_mid, n_out, torch.bfloat16, "silu", with_residual, seed=41)


@pytest.mark.parametrize("rows,n_in,n_mid,n_out", [(12037, 64, 64, 36), (12037, 128, 192, 100), (6005, 384, 384, 260)])
def test_fp32_tiles(rows, n_in, n_mid, n_out):
    for with_residual in (False, True):
        _check(rows, n_in, n_mid, n_out, torch.float32, "silu", with_residual, seed=43)


@pytest.mark.parametrize("rows", [1, 16, 40, 300, 2100])
@pytest.mark.parametrize("n_in,n_mid,n_out", [(65536, 8, 8), (8, 65536, 8), (8, 8, 65536), (65536, 24, 40)])
def test_the_widest_and_the_narrowest(rows, n_in, n_mid, n_out):
    _check(rows, n_in, n_mid, n_out, torch.bfloat16, "silu", rows % 2 == 0, seed=47)
