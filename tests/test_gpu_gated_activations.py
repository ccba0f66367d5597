"""The gated block's activations over their range, from sums that are exact: a row of x is (gate, 1, 0, ...) and the weights pick the two,
so every sum is the gate itself, or 1, whatever the order of the products.

fp32, `logistic`: 2^t and the reciprocal are 2^-22 off each at most, t ln 2 is 2^-22 with the constant's rounding over the range, the rest
are three roundings of 2^-24: below 2^-20 of it.  Below -87 it is 0, which is 2^-125 off.  silu is that times the gate; its slope
s (1 + x (1 - s)) has what s is off in three places, x s^2 being the one that its other term may cancel.
bf16, `sigmoid` and the few rows' quotient: the power's rounding is in it too, |x| 2^-23, next to 2^-20, before h (and dgate) are rounded to
2^-8.  Below -87 reciprocals and powers leave fp32's normal numbers: 2^-125 again.
gelu is x (1 + erf) / 2: the sum's rounding, 2^-24, and erf's, 2^-23, count whole on the negative side; its slope adds
x times a density with 2^-21 and, in bf16, the square's rounding x^2 2^-23."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = {"relu": 1, "gelu": 2, "silu": 3}
WIDTH = 64


def _defined(act, g, wide):
    """act(g) and its slope, and what of them may be lost (the two bounds) in the fp32 kernels or before bf16's rounding, in 64 bits."""
    if act == "relu":
        return g.clamp(min=0), (g > 0).double(), torch.zeros_like(g), torch.zeros_like(g)
    if act == "silu":
        s = torch.sigmoid(g)
        value, slope = g * s, s * (1 + g * (1 - s))
        off = 2.0 ** -20 + (0 if wide else g.abs() * 2.0 ** -23)
        return value, slope, off * value.abs() + g.abs() * 2.0 ** -125, \
            off * (slope.abs() + s * s * g.abs()) + 4 * 2.0 ** -24 * s * (1 + g.abs() * (1 - s)) + (1 + g.abs()) * 2.0 ** -125
    cdf = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)
    density = g * torch.exp(-g * g / 2) * (2 * torch.pi) ** -0.5
    return g * cdf, cdf + density, g.abs() * 2.0 ** -22, 2.0 ** -22 + density.abs() * (2.0 ** -20 + g * g * 2.0 ** -23)


def _gates(rows, dtype):
    """From -110 to 110 and closer together around 0, every one of them as `dtype` has it."""
    far = torch.linspace(-110, 110, rows - rows // 2, dtype=torch.float64)
    near = torch.linspace(-6, 6, rows // 2, dtype=torch.float64)
    return torch.cat([far, near]).to(dtype).cuda()


def _operands(gates):
    x = torch.zeros(gates.shape[0], WIDTH, dtype=gates.dtype, device="cuda")
    x[:, 0], x[:, 1] = gates, 1
    wg, wu, wd = (torch.zeros(WIDTH, WIDTH, dtype=gates.dtype, device="cuda") for _ in range(3))
    wg[:, 0], wu[:, 1] = 1, 1
    wd[0] = 1 / WIDTH                                          # dh is dy[:, 0] / 64
    return x, wg, wu, wd


def _check(name, got, want, lost, rounding):
    bound = lost + rounding * (want.abs() + lost)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (name, float((off / (bound + 1e-300)).max()))


# rows: in fp32 a kernel of its own between the products, and in their finish; in bf16 one tile, a few, and rounds of them
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("dtype,rows", [(torch.float32, 3000), (torch.float32, 40001), (torch.bfloat16, 16), (torch.bfloat16, 500),
                                        (torch.bfloat16, 40001)])
def test_over_the_range(dtype, rows, act):
    from torchgt_b200 import _cabi
    lib, stream = _cabi.load(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    gates = _gates(rows, dtype)
    x, wg, wu, wd = _operands(gates)
    wide = dtype == torch.float32
    value, slope, value_lost, slope_lost = _defined(act, gates.double(), wide)
    rounding, code = (2.0 ** -24, 0) if wide else (2.0 ** -8, 1)
    h, gate, up, low, dgate, dup = (torch.empty(rows, WIDTH, dtype=dtype, device="cuda") for _ in range(6))
    _cabi.check(lib.tgt_gated_hidden(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), rows, WIDTH, WIDTH, ACTS[act], code, h.data_ptr(),
                                     gate.data_ptr(), up.data_ptr(), None if wide else low.data_ptr(), stream))
    assert bool((gate == gates[:, None]).all()) and bool((up == 1).all())
    for column in (0, 31, 32, WIDTH - 1):
        _check("h", h[:, column], value, value_lost, rounding)
    dy = torch.zeros(rows, WIDTH, dtype=dtype, device="cuda")
    dy[:, 0] = WIDTH
    _cabi.check(lib.tgt_gated_hidden_grad(dy.data_ptr(), wd.data_ptr(), gate.data_ptr(), up.data_ptr(), None if wide else low.data_ptr(), rows,
                                          WIDTH, WIDTH, ACTS[act], code, dgate.data_ptr(), dup.data_ptr(), stream))
    for column in (0, WIDTH - 1):
        _check("dup", dup[:, column], value, value_lost, rounding)
        _check("dgate", dgate[:, column], slope, slope_lost, rounding)


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("rows", [1, 16, 27, 32])
def test_few_rows_over_the_range(rows, act):
    """As serving calls it; wd's first row takes one column of h, so y is h as it was rounded."""
    from torchgt_b200 import gated_feed_forward
    for start in range(0, 1000, 1000 if rows == 1 else 250):
        gates = _gates(1000, torch.bfloat16)[start:start + rows]
        x, wg, wu, wd = _operands(gates)
        wd[0] = 0
        wd[0, 5] = 1
        value, _, lost, _ = _defined(act, gates.double(), False)
        with torch.no_grad():
            _check("y", gated_feed_forward(x, wg, wu, wd, act)[:, 0], value, lost, 2.0 ** -8)
