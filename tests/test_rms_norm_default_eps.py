"""The norms' eps where the caller gives none: torch's, which is the machine epsilon of the type it computes in, fp32's for fp32
and bf16 rows.  Rows' root mean squares go down to 2^-12, where fp32's epsilon is twice the mean square and bf16's
would be 2^17 times it.

Tolerances are those of test_gpu_rms_norm.py: a result's own rounding u (2^-24, bf16 2^-8), sums and their root below 64 * 2^-24; the
weight's gradient 128; a bf16 sum has v to 2^-15 twice.  torch's own rows may be rounded before the weight's product too: two
roundings, and ours the third of a comparison."""
import pytest
import torch

ROUNDING = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24
SIZES = (2.0 ** -12, 2.0 ** -6, 0.05, 0.3, 1.0)                   # of a row's values


def _rows(dtype, hidden, seed, device):
    gen = torch.Generator().manual_seed(seed)
    draw = lambda: torch.randn(7 * len(SIZES), hidden, generator=gen) * torch.tensor(SIZES).repeat(7)[:, None]   # noqa: E731
    weight = torch.randn(hidden, generator=gen) * 0.3 + 1
    return [t.to(dtype).to(device) for t in (draw(), draw() / 4, weight, draw() * 8, draw())]


def _formula(v, w, dy):
    v, w, dy = v.double(), w.double(), dy.double()
    rstd = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + torch.finfo(torch.float32).eps)
    u, g = v * rstd, dy * w
    return {"y": u * w, "dx": rstd * (g - u * (g * u).mean(-1, keepdim=True)), "dw": (dy * u).sum(0),
            "dx_size": rstd * (g.abs() + u.abs() * (g * u).abs().mean(-1, keepdim=True)), "dw_size": (dy * u).abs().sum(0)}


def _within(got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound + 1e-300).all()), float((off / (bound + 1e-300)).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_eps_is_the_one_torch_takes(dtype):
    """From torch's own results: the formula with the eps that the kernels get is what torch makes of rows without one."""
    from torchgt_b200.rms_norm import _eps
    x, _, w, _, _ = _rows(dtype, 64, 1, "cpu")
    eps = _eps(x, None)
    want = x.double() / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + eps) * w.double()
    _within(torch.nn.functional.rms_norm(x, (64,), w), want, (2 * ROUNDING[dtype] + 64 * E) * want.abs())
    assert _eps(x, 1e-3) == 1e-3 and _eps(x, 0.0) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [64, 100, 2048])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_and_gradients_without_an_eps(dtype, hidden):
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm
    x, r, w, dy, ds = _rows(dtype, hidden, 2, "cuda")
    u = ROUNDING[dtype]
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    y = rms_norm(*leaves)
    ref = _formula(x, w, dy)
    _within(y, ref["y"], (u + 64 * E) * ref["y"].abs())
    dx, dw = torch.autograd.grad(y, leaves, dy)
    _within(dx, ref["dx"], u * ref["dx"].abs() + 64 * E * ref["dx_size"])
    _within(dw, ref["dw"], u * ref["dw"].abs() + 128 * E * ref["dw_size"])
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, total = add_rms_norm(*leaves)
    ref, seen = _formula(x.double() + r.double(), w, dy), 2 * 2.0 ** -15 if dtype == torch.bfloat16 else 0
    _within(y, ref["y"], (u + 64 * E) * ref["y"].abs())
    dx, dr, dw = torch.autograd.grad([y, total], leaves, [dy, ds])
    want, size = ref["dx"] + ds.double(), ref["dx_size"] + ds.double().abs()
    _within(dx, want, u * want.abs() + (64 * E + seen) * size)
    _within(dw, ref["dw"], u * ref["dw"].abs() + (128 * E + seen) * ref["dw_size"])
    assert torch.equal(dx, dr)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_eight_bit_rows_without_an_eps(dtype):
    from torchgt_b200.rms_norm import rms_norm_quantized
    x, r, w, dy, _ = _rows(dtype, 256, 3, "cuda")
    for residual, v in ((None, x.double()), (r, x.double() + r.double())):
        values, scales, _ = rms_norm_quantized(x, w, residual=residual)
        y = _formula(v, w, dy)["y"]
        scale = (y.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
        _within(scales, scale, 66 * E * scale)
        half = torch.maximum(y.abs() * 2.0 ** -4, scale[:, None] * 2.0 ** -10)
        _within(values.double() * scales.double()[:, None], y, half + 130 * E * y.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_module_without_an_eps_is_torchs(dtype):
    """Next to nn.RMSNorm, and to itself on the host and under autocast."""
    from torchgt_b200 import RMSNorm
    x, r, w, _, _ = _rows(dtype, 64, 4, "cuda")
    ours, theirs = RMSNorm(64).to(dtype).cuda(), torch.nn.RMSNorm(64).to(dtype).cuda()
    for module in (ours, theirs):
        module.weight.data.copy_(w)
    u = ROUNDING[dtype]
    with torch.no_grad():
        y, want = ours(x).double(), theirs(x).double()
        _within(y, want, (3 * u + 128 * E) * want.abs())
        _within(ours.cpu()(x.cpu()).cuda(), y, (3 * u + 128 * E) * y.abs())
        ours.cuda()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            _within(ours(x), y, (3 * u + 128 * E) * y.abs())
        y, total = ours.add(x, r)
        want = _formula(x.double() + r.double(), w, r)["y"]
        _within(y, want, (u + 64 * E) * want.abs())
