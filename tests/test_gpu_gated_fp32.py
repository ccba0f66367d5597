"""The gated block's fp32 products with the gate in their finish, at sizes that reach them (80 tiles of 128 rows x 64 columns or more,
up to six chunks of 64 of the reduction): every activation against the formula in 64 bits, under the bounds of
test_gpu_gated_ffn.py, and rows whose sums leave the range of fp32 or are no numbers, which are summed again apart from the others."""
import ctypes

import pytest
import torch

from test_gpu_gated_ffn import E, _check, _inputs

pytestmark = pytest.mark.gpu

ACTS = {"relu": 1, "gelu": 2, "silu": 3}
FUSED = [(12000, 64, 128, 64), (6000, 192, 320, 192), (4000, 384, 384, 384)]     # one chunk and two, three and five, six


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("rows,n_in,n_mid,n_out", FUSED)
def test_values_and_gradients(rows, n_in, n_mid, n_out, act):
    _check(rows, n_in, n_mid, n_out, torch.float32, act, rows % 4000 == 0, seed=51)


def _hidden(x, wg, wu, act):
    from torchgt_b200 import _cabi
    h, gate, up = (torch.empty(x.shape[0], wg.shape[0], device="cuda") for _ in range(3))
    _cabi.check(_cabi.load().tgt_gated_hidden(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), x.shape[0], x.shape[1], wg.shape[0], ACTS[act], 0,
                                              h.data_ptr(), gate.data_ptr(), up.data_ptr(), None,
                                              ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    return h, gate, up


def _hidden_grad(dy, wd, gate, up, act):
    from torchgt_b200 import _cabi
    dgate, dup = torch.empty_like(gate), torch.empty_like(up)
    _cabi.check(_cabi.load().tgt_gated_hidden_grad(dy.data_ptr(), wd.data_ptr(), gate.data_ptr(), up.data_ptr(), None, dy.shape[0],
                                                   dy.shape[1], gate.shape[1], ACTS[act], 0, dgate.data_ptr(), dup.data_ptr(),
                                                   ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    return dgate, dup


def _as_summed(got, a, w):
    """``got`` is ``a @ w`` as fp32 has it: not a number and infinite where the sum is, what it is where that is in the range.
    Sums of 64 bits within 2^-10 of the range's end may go either way in fp32."""
    want, size = a.double() @ w.double(), a.double().abs() @ w.double().abs()
    finite = want.isfinite() & (size < 2.0 ** 128 * (1 - 2.0 ** -10))
    assert torch.equal(got.isnan() & ~finite, want.isnan())
    infinite = want.isinf()
    assert torch.equal(got[infinite].double(), want[infinite])
    off = (got.double() - want)[finite].abs()
    assert bool((off <= (a.shape[1] + 16) * E * size[finite]).all())


# a row's place in the operand and what it holds: (row, column or all, value)
SPOILT = [(0, 3, float("nan")), (31, None, float("inf")), (32, 0, float("-inf")), (127, 17, 3.39e38), (128, None, 2.0 ** 120),
          (1000, 40, float("inf")), (1001, 41, float("nan")), (3999, None, float("nan"))]


def _spoil(t, n):
    for row, column, value in SPOILT:
        if column is None:
            t[row] = t[row].sign() * value if value == 2.0 ** 120 else value
        else:
            t[row, column % n] = value
    return [i for i in range(t.shape[0]) if i not in [row for row, _, _ in SPOILT]]


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("rows,n_in,n_mid,n_out", FUSED)
def test_rows_that_are_no_numbers(rows, n_in, n_mid, n_out, act):
    """Both projections and both gradients, value by value, and the rows beside them bit by bit."""
    x, wg, wu, wd, _, dy = _inputs(rows, n_in, n_mid, n_out, torch.float32, 53)
    clean = _hidden(x, wg, wu, act)
    others = _spoil(x, n_in)
    h, gate, up = _hidden(x, wg, wu, act)
    for got, want in zip((h, gate, up), clean):
        assert torch.equal(got[others], want[others])
    _as_summed(gate, x, wg.t())
    _as_summed(up, x, wu.t())
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}[act]
    want = f(gate) * up                                     # from the sums as they were written
    assert torch.equal(h.isnan(), want.isnan())
    some = [row for row, _, _ in SPOILT]
    bad = ~want[some].isfinite()
    assert torch.equal(h[some][bad].nan_to_num(), want[some][bad].nan_to_num())

    _, gate, up = clean
    clean_grads = _hidden_grad(dy, wd, gate, up, act)
    others = _spoil(dy, n_out)
    grads = _hidden_grad(dy, wd, gate, up, act)
    for got, want in zip(grads, clean_grads):
        assert torch.equal(got[others], want[others])
    # with every projection 1 and relu, both gradients are the sums themselves
    one = torch.ones_like(gate)
    for got in _hidden_grad(dy, wd, one, one, "relu"):
        _as_summed(got, dy, wd)


@pytest.mark.parametrize("act", sorted(ACTS))
def test_a_spoilt_row_through_the_block(act):
    """Forward and backward of a call with such rows in its input: other rows of y and dx as without them."""
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, dy = _inputs(12000, 64, 128, 64, torch.float32, 55)

    def step(x, dy):
        x = x.clone().requires_grad_()
        y = gated_feed_forward(x, wg, wu, wd, act, r)
        return y.detach(), torch.autograd.grad(y, [x], dy)[0]
    y, dx = step(x, dy)
    bad = x.clone()
    others = _spoil(bad, 64)
    spoilt_y, spoilt_dx = step(bad, dy)
    assert torch.equal(spoilt_y[others], y[others]) and torch.equal(spoilt_dx[others], dx[others])
    assert bool(spoilt_y[[0, 1001, 3999]].isnan().all()) and not bool(spoilt_y[31].isfinite().any())
    bad = dy.clone()
    others = _spoil(bad, 64)
    same_y, spoilt_dx = step(x, bad)
    assert torch.equal(same_y, y) and torch.equal(spoilt_dx[others], dx[others]) and bool(spoilt_dx[[0, 3999]].isnan().all())
