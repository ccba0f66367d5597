"""Gradients of the residual norm that are themselves differentiated, or many at once, are recorded as operations: of a bf16 sum from the
same value as the kernel's, the stored sum with the 8 bits that its rounding took.

Bounds as in test_gpu_rms_norm.py: the result's own rounding 2^-8, v to 2^-15 in both places, sums 64 (weight 128) times 2^-24;
operations round every intermediate step, a dozen of them."""
import pytest
import torch

from test_gpu_rms_norm import E, EPS, ROUNDING, _formula, _inputs, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,hidden", [(40, 64), (301, 100), (17, 2048)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_recorded_gradients_have_the_kernels_bounds(rows, hidden, dtype):
    from torchgt_b200.rms_norm import add_rms_norm
    x, r, w, dy, ds = _inputs(rows, hidden, dtype, 61)
    ref = _formula(x, r, w, dy, ds)
    u, seen = ROUNDING[dtype], 2 * 2.0 ** -15 if dtype == torch.bfloat16 else 0
    bounds = (u * ref["dx"].abs() + (128 * E + seen) * ref["dx_size"], u * ref["dw"].abs() + (256 * E + seen) * ref["dw_size"])
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    for recorded in (lambda out: torch.autograd.grad(out, leaves, [dy, ds], create_graph=True),
                     lambda out: [g[1] for g in torch.autograd.grad(out, leaves, [torch.stack([ds, dy]), torch.stack([dy, ds])],
                                                                    is_grads_batched=True)]):
        dx, dr, dw = recorded(list(add_rms_norm(*leaves, EPS)))
        _within(dx.detach(), ref["dx"], bounds[0])
        _within(dw.detach(), ref["dw"], bounds[1])
        assert dx.dtype == dtype and torch.equal(dx, dr)


def test_second_order_of_a_bf16_sum():
    """The gradient of a gradient next to the formula's in 64 bits; the first is rounded to bf16 before the second is taken from it."""
    from torchgt_b200.rms_norm import add_rms_norm
    x, r, w, dy, _ = _inputs(12, 64, torch.bfloat16, 62)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    first, = torch.autograd.grad(add_rms_norm(*leaves, EPS)[0], leaves[:1], dy, create_graph=True)
    got = torch.autograd.grad((first.float() * dy.float()).sum(), leaves)
    d = [t.detach().double().requires_grad_() for t in leaves]
    v = d[0] + d[1]
    y = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * d[2]
    first, = torch.autograd.grad(y, d[:1], dy.double(), create_graph=True)
    for a, b in zip(got, torch.autograd.grad((first * dy.double()).sum(), d)):
        # three roundings to bf16 on the way, the result's among them, and the sums' cancellation
        assert float((a.double() - b).abs().max()) <= 8 * 2.0 ** -8 * float(b.abs().max())


def test_sums_at_the_ends_of_the_range():
    """Sums that bf16 rounds to infinity, zeros and numbers that are none: recorded gradients are numbers where the kernel's are."""
    from torchgt_b200.rms_norm import add_rms_norm
    x, r, w, dy, ds = _inputs(6, 64, torch.bfloat16, 63)
    x[0, 3], r[0, 3] = 3.3895e38, 1e36                       # x + r is in fp32's range, its rounding is not
    x[1], r[1] = 0, 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    want = torch.autograd.grad(list(add_rms_norm(*leaves, EPS)), leaves, [dy, ds])
    got = torch.autograd.grad(list(add_rms_norm(*leaves, EPS)), leaves, [dy, ds], create_graph=True)
    assert torch.equal(got[0].isfinite(), want[0].isfinite())
    assert bool(want[0][[1, 4, 5]].isfinite().all()) and bool(want[0][[2, 3]].isnan().any(-1).all())
