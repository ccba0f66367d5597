"""Host side of the operators around the attention: bucket borders, refusals, what runs without a GPU."""
import ctypes
import math

import pytest
import torch


def test_borders_follow_the_logarithm_and_cover_every_distance():
    from torchgt_b200.position_bias import bucket_borders
    assert bucket_borders(32, 128, True) == (1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91)
    for buckets, distance, both_ways in ((32, 128, True), (32, 128, False), (64, 1000, True), (10, 50, True), (2, 2, False),
                                         (4, 2, True), (512, 2 ** 31 - 1, False), (3, 9, False), (16, 9, False)):
        count = buckets // 2 if both_ways else buckets
        exact = count // 2
        borders = bucket_borders(buckets, distance, both_ways)
        assert len(borders) == count - 1 and list(borders) == sorted(borders) and borders[0] == 1
        assert list(borders[:exact]) == list(range(1, exact + 1))
        for j, border in enumerate(borders[exact:], 1):
            line = exact * (distance / exact) ** (j / (count - exact))
            assert border == math.ceil(line) or abs(border - line) < 1 + 1e-9 * line


@pytest.mark.parametrize("buckets,distance,both_ways", [(1, 128, False), (2, 128, True), (33, 128, True), (0, 4, False), (513, 9999, False),
                                                        (32, 8, True), (32, 2 ** 31, True), (1024, 5000, True)])
def test_borders_that_cannot_be(buckets, distance, both_ways):
    from torchgt_b200 import RelativePositionBias
    from torchgt_b200.position_bias import bucket_borders
    with pytest.raises(ValueError):
        bucket_borders(buckets, distance, both_ways)
    with pytest.raises(ValueError):
        RelativePositionBias(8, buckets, distance, both_ways)


def test_host_tensors_are_refused_or_run_as_torch():
    from torchgt_b200 import RMSNorm
    from torchgt_b200.position_bias import edge_position_bias
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm_quantized
    x, w = torch.randn(5, 64), torch.randn(64)
    with pytest.raises(RuntimeError, match="CUDA"):
        rms_norm_quantized(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        edge_position_bias(torch.randn(32, 8), torch.zeros(2, 4, dtype=torch.long))
    with pytest.raises(TypeError):
        edge_position_bias(torch.randn(32, 8), [[0], [1]])
    y, total = add_rms_norm(x, x, w, 1e-6)
    assert torch.equal(total, x + x) and torch.equal(y, torch.nn.functional.rms_norm(x + x, (64,), w, 1e-6))
    module = RMSNorm(64)
    assert torch.equal(module(x), torch.nn.RMSNorm(64)(x)) and list(module.state_dict()) == ["weight"]


def test_argument_checks_run_before_any_cuda_call():
    from torchgt_b200 import _cabi
    from torchgt_b200.build import build
    build()
    lib = _cabi.load()
    n = ctypes.c_size_t()
    borders = (ctypes.c_int32 * 3)(1, 2, 4)
    backwards = (ctypes.c_int32 * 3)(1, 4, 2)
    zero = (ctypes.c_int32 * 1)(0)
    # norm: types, sizes, null pointers
    assert lib.tgt_rms_norm_fwd(None, None, None, 0.0, 1, 64, 9, None, None, None, None, None) == 1
    assert lib.tgt_rms_norm_fwd(None, None, None, 0.0, -1, 64, 0, None, None, None, None, None) == 1
    assert lib.tgt_rms_norm_fwd(None, None, None, 0.0, 1, 0, 0, None, None, None, None, None) == 1
    assert lib.tgt_rms_norm_fwd(None, None, None, 0.0, 1, 16385, 0, None, None, None, None, None) == 3
    assert lib.tgt_rms_norm_fwd(None, None, None, 0.0, 1, 64, 0, None, None, None, None, None) == 1
    assert lib.tgt_rms_norm_fwd(16, None, 16, 0.0, 1, 64, 0, 16, None, 16, None, None) == 1          # a sum without a residual
    assert lib.tgt_rms_norm_fwd(16, 16, 16, 0.0, 1, 64, 0, 16, 16, 16, None, None) == 1            # a rest of fp32
    assert lib.tgt_rms_norm_fwd(16, 16, 16, 0.0, 1, 64, 1, None, 16, 16, None, None) == 1          # of no sum
    assert lib.tgt_rms_norm_fwd(None, None, None, 0.0, 0, 64, 0, None, None, None, None, None) == 0  # no rows
    assert lib.tgt_rms_norm_e4m3(None, None, None, 0.0, 0, 64, 1, None, None, None, None) == 0
    assert lib.tgt_rms_norm_e4m3(16, None, 16, 0.0, 1, 64, 1, None, 16, None, None) == 1
    assert lib.tgt_rms_norm_bwd_scratch_bytes(10, 64, 0, None) == 1
    assert lib.tgt_rms_norm_bwd(None, None, None, None, None, None, 1, 64, 0, None, None, None, 0, None) == 1
    # bias: borders, sizes, null pointers
    assert lib.tgt_edge_position_bias(None, 0, 1, None, 0, 0, borders, 3, 1, None, 8, None, None, None) == 0
    assert lib.tgt_edge_position_bias(None, 1, 1, None, 0, 0, borders, 3, 1, None, 8, None, None, None) == 1
    assert lib.tgt_edge_position_bias(None, -1, 1, None, 0, 0, borders, 3, 1, None, 8, None, None, None) == 1
    assert lib.tgt_edge_position_bias(None, 0, 1, None, 0, 0, backwards, 3, 1, None, 8, None, None, None) == 1
    assert lib.tgt_edge_position_bias(None, 0, 1, None, 0, 0, zero, 1, 1, None, 8, None, None, None) == 1
    assert lib.tgt_edge_position_bias(None, 0, 1, None, 0, 0, None, 3, 1, None, 8, None, None, None) == 1
    assert lib.tgt_edge_position_bias(None, 0, 1, None, 0, 0, None, 512, 0, None, 8, None, None, None) == 1
    assert lib.tgt_edge_position_bias(None, 0, 1, None, 0, 0, borders, 3, 1, None, 257, None, None, None) == 3
    assert lib.tgt_edge_position_bias_grad_scratch_bytes(10, 513, 8, ctypes.byref(n)) == 3
    assert lib.tgt_edge_position_bias_grad(None, None, 1, 32, 8, None, None, 0, None) == 1


def test_gated_block_arguments():
    from torchgt_b200 import GatedFeedForward, _cabi, gated_feed_forward
    x, wg, wu, wd = torch.randn(5, 64), torch.randn(96, 64), torch.randn(96, 64), torch.randn(64, 96)
    want = (torch.nn.functional.silu(x @ wg.t()) * (x @ wu.t())) @ wd.t()
    torch.testing.assert_close(gated_feed_forward(x, wg, wu, wd), want)
    torch.testing.assert_close(gated_feed_forward(x, wg, wu, wd, residual=x), want + x)
    for bad in ((x, wg, wu[:50], wd), (x, wg, wu, wd.t()), (x[:, :32], wg, wu, wd), (x, wg[0], wu, wd)):
        with pytest.raises(ValueError):
            gated_feed_forward(*bad)
    with pytest.raises(ValueError):
        gated_feed_forward(x, wg, wu, wd, "tanh")
    with pytest.raises(ValueError):
        gated_feed_forward(x, wg, wu, wd, "silu", x[0])
    with pytest.raises(ValueError):
        GatedFeedForward(64, 96, "tanh")
    lib, n = _cabi.load(), ctypes.c_size_t()
    hidden = lambda rows, i, m, act, dtype: lib.tgt_gated_hidden(None, None, None, rows, i, m, act, dtype, None, None, None, None, None)  # noqa: E731
    assert hidden(0, 64, 64, 3, 1) == 0 and hidden(1, 64, 64, 3, 1) == 1 and hidden(-1, 64, 64, 3, 1) == 1
    assert hidden(1, 64, 64, 0, 1) == 1 and hidden(1, 64, 64, 3, 7) == 1 and hidden(1, 0, 64, 3, 1) == 1
    assert hidden(1, 60, 64, 3, 1) == 3 and hidden(1, 64, 65544, 3, 1) == 3 and hidden(2 ** 31, 64, 64, 3, 1) == 3
    assert lib.tgt_gated_hidden(16, 16, 16, 1, 64, 64, 3, 1, 24, None, None, None, None) == 1        # alignment
    assert lib.tgt_gated_hidden(16, 16, 16, 1, 64, 64, 3, 1, 16, 16, None, 16, None) == 1          # gate without up
    assert lib.tgt_gated_hidden(16, 16, 16, 1, 64, 64, 3, 1, 16, 16, 16, None, None) == 1          # without the bits below
    assert lib.tgt_gated_hidden(16, 16, 16, 1, 64, 64, 3, 0, 16, None, None, None, None) == 1        # fp32 needs both
    assert lib.tgt_gated_output(None, None, None, 1, 64, 64, 1, None, None) == 1
    assert lib.tgt_gated_hidden_grad(None, None, None, None, None, 1, 64, 64, 3, 1, None, None, None) == 1
    assert lib.tgt_gated_input_grad(None, None, None, None, 1, 64, 64, 1, None, None) == 1
    assert lib.tgt_gated_weight_grad_scratch_bytes(3, 1, 64, 64, 1, ctypes.byref(n)) == 1
    assert lib.tgt_gated_weight_grad_scratch_bytes(1, 1, 64, 60, 1, ctypes.byref(n)) == 3
    assert lib.tgt_gated_weight_grad_scratch_bytes(2, 0, 64, 64, 1, ctypes.byref(n)) == 0 and n.value == 0
    dw = (ctypes.c_void_p * 2)(16, 16)
    assert lib.tgt_gated_weight_grad(None, None, 2, 1, 64, 64, 1, dw, None, 0, None) == 1
    few = lambda rows, i, m, o, act: lib.tgt_gated_few_rows(None, None, None, None, None, rows, i, m, o, act, None, None, None)  # noqa: E731
    assert few(0, 64, 64, 64, 3) == 0 and few(1, 64, 64, 64, 3) == 1 and few(33, 64, 64, 64, 3) == 1 and few(-1, 64, 64, 64, 3) == 1
    assert few(1, 64, 60, 64, 3) == 3 and few(1, 64, 64, 65544, 3) == 3 and few(1, 64, 64, 64, 0) == 1
