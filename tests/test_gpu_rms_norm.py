"""The root-mean-square norm's kernels (alone, with the residual addition, in 8 bits, backward) against the formula in 64 bits.

Tolerances, u the rounding of the tensors' type (fp32 2^-24, bf16 2^-8) and e = 2^-24 that of the sums: a result's own
rounding is u.  A sum of squares, or of products, over a row is at most 16 terms in a thread, 5 steps in a warp and 32 over warps, its
reciprocal root 2 units and the products around it 3: below 64 e of the sum of the magnitudes.  The backward of a bf16 sum has v to
2^-15 (8 bits next to the rounded sum, cut to a byte's range), in every place it has v.  A weight's gradient adds that over the rows: below 128 e of the sum of magnitudes for
up to 5,000 rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
ROUNDING = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
EPS = 1e-6


def _inputs(rows, hidden, dtype, seed, shape=None):
    gen = torch.Generator().manual_seed(seed)
    draw = lambda *s: torch.randn(*s, generator=gen)   # noqa: E731
    x, r, dy, ds = ((draw(rows, hidden) * 2 + 0.3).to(dtype).cuda() for _ in range(4))
    return x, r, (draw(hidden) * 0.3 + 1).to(dtype).cuda(), dy, ds


def _formula(x, r, w, dy=None, ds=None):
    x, w = x.double().cpu(), w.double().cpu()
    v = x if r is None else x + r.double().cpu()
    rstd = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    u = v * rstd
    out = {"v": v, "y": u * w}
    if dy is not None:
        dy = dy.double().cpu()
        g = dy * w
        m, ma = (g * u).mean(-1, keepdim=True), (g * u).abs().mean(-1, keepdim=True)
        out["dx"] = rstd * (g - u * m) + (0 if ds is None else ds.double().cpu())
        out["dx_size"] = rstd * (g.abs() + u.abs() * ma) + (0 if ds is None else ds.double().cpu().abs())
        out["dw"], out["dw_size"] = (dy * u).flatten(0, -2).sum(0), (dy * u).abs().flatten(0, -2).sum(0)
    return out


def _within(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound + 1e-300).all()), float((off / (bound + 1e-300)).max())


SIZES = [(1, 1), (3, 7), (5, 8), (257, 64), (33, 100), (4099, 64), (64, 479), (7, 512), (300, 768), (17, 1000), (129, 1032),
         (40, 2048), (9, 4097), (3, 8192), (2, 8200), (2, 16384), (2, 16383)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,hidden", SIZES)
def test_forward_and_gradients(rows, hidden, dtype):
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm
    x, r, w, dy, ds = _inputs(rows, hidden, dtype, rows * 31 + hidden)
    u = ROUNDING[dtype]
    for residual in (None, r):
        leaves = [t.clone().requires_grad_() for t in ((x, w) if residual is None else (x, residual, w))]
        if residual is None:
            y = rms_norm(leaves[0], leaves[1], EPS)
            grads = torch.autograd.grad(y, leaves, dy)
            ref = _formula(x, None, w, dy)
        else:
            y, total = add_rms_norm(*leaves, EPS)
            grads = torch.autograd.grad([y, total], leaves, [dy, ds])
            ref = _formula(x, residual, w, dy, ds)
            _within(total, ref["v"], u * ref["v"].abs())
            assert torch.equal(grads[0], grads[1])
        assert y.dtype == dtype and y.shape == x.shape
        _within(y, ref["y"], (u + 64 * E) * ref["y"].abs())
        seen = 2 * 2.0 ** -15 if residual is not None and dtype == torch.bfloat16 else 0      # v's rounding, twice in a product
        _within(grads[0], ref["dx"], u * ref["dx"].abs() + (64 * E + seen) * ref["dx_size"])
        _within(grads[-1], ref["dw"], u * ref["dw"].abs() + (128 * E + seen) * ref["dw_size"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,hidden", SIZES)
def test_eight_bit_rows_and_their_scales(rows, hidden, dtype):
    from torchgt_b200.rms_norm import rms_norm_quantized
    x, r, w, _, _ = _inputs(rows, hidden, dtype, rows * 17 + hidden)
    x[rows // 2] = 0                                     # a row of zeros next to others
    r[rows // 2] = 0
    for residual in (None, r):
        values, scales, total = rms_norm_quantized(x, w, EPS, residual)
        assert values.dtype == torch.float8_e4m3fn and values.shape == x.shape and scales.shape == (rows,)
        ref = _formula(x, residual, w)
        scale = (ref["y"].abs().amax(-1) / 448).clamp(min=2.0 ** -126)
        _within(scales, scale, 66 * E * scale)
        # half a step of e4m3 is 2^-4 of the value, or 2^-10 below its normal numbers, of the scale
        half = torch.maximum(ref["y"].abs() * 2.0 ** -4, scale[:, None] * 2.0 ** -10)
        _within(values.cpu().double() * scales.cpu().double()[:, None], ref["y"], half + 130 * E * ref["y"].abs())
        if residual is None:
            assert total is None
        else:
            _within(total, ref["v"], ROUNDING[dtype] * ref["v"].abs())


def test_a_rows_nan_and_infinity_stay_in_the_row():
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm_quantized
    x, r, w, _, _ = _inputs(40, 200, torch.float32, 1)
    clean = add_rms_norm(x, r, w, EPS)[0]
    values, scales, _ = rms_norm_quantized(x, w, EPS, r)
    x[3, 5], x[17, 0], x[18, 199] = float("nan"), float("inf"), float("-inf")
    y = add_rms_norm(x, r, w, EPS)[0]
    bad_values, bad_scales, _ = rms_norm_quantized(x, w, EPS, r)
    others = [i for i in range(40) if i not in (3, 17, 18)]
    assert torch.equal(y[others], clean[others]) and torch.equal(bad_scales[others], scales[others])
    assert torch.equal(bad_values.view(torch.uint8)[others], values.view(torch.uint8)[others])
    assert bool(y[3].isnan().all()) and bool(y[17, 0].isnan()) and bool(y[18, 199].isnan())
    assert bool(bad_scales[[3, 17, 18]].isnan().all())


def test_values_far_from_one():
    """Rows around 2^-60 and 2^50: eps rules the first, squares are far from the range's ends in both."""
    from torchgt_b200.rms_norm import rms_norm, rms_norm_quantized
    x, _, w, _, _ = _inputs(6, 128, torch.float32, 2)
    x[:3] *= 2.0 ** -60
    x[3:] *= 2.0 ** 50
    ref = _formula(x, None, w)
    _within(rms_norm(x, w, EPS), ref["y"], 65 * E * ref["y"].abs())
    values, scales, _ = rms_norm_quantized(x, w, EPS)
    scale = ref["y"].abs().amax(-1) / 448
    _within(scales, scale, 66 * E * scale)
    x.mul_(0).add_(2.0 ** -140)                          # scales at their lower end: no infinite reciprocal
    values, scales, _ = rms_norm_quantized(x, w, 1.0)
    assert bool((scales == 2.0 ** -126).all()) and bool(values.float().isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_strides_and_places_off_a_16_byte_boundary(dtype):
    from torchgt_b200.rms_norm import add_rms_norm
    x, r, w, dy, ds = _inputs(50, 96, dtype, 3)
    want = add_rms_norm(x, r, w, EPS)
    wide = torch.zeros(50, 200, dtype=dtype, device="cuda")
    wide[:, 3:99] = x
    flat = torch.zeros(50 * 96 + 1, dtype=dtype, device="cuda")
    flat[1:] = r.flatten()
    off = torch.zeros(97, dtype=dtype, device="cuda")
    off[1:] = w
    leaves = [wide[:, 3:99].requires_grad_(), flat[1:].view(50, 96).requires_grad_(), off[1:].requires_grad_()]
    got = add_rms_norm(*leaves, EPS)
    ref = _formula(x, r, w, dy, ds)
    u = ROUNDING[dtype]
    _within(got[0], ref["y"], (u + 64 * E) * ref["y"].abs())
    assert torch.equal(got[1], want[1])
    grads = torch.autograd.grad(got, leaves, [dy.t().contiguous().t(), ds])
    seen = 2 * 2.0 ** -15 if dtype == torch.bfloat16 else 0
    _within(grads[0], ref["dx"], u * ref["dx"].abs() + (64 * E + seen) * ref["dx_size"])
    batch = x.view(5, 10, 96).transpose(0, 1)
    y, total = add_rms_norm(batch, r.view(5, 10, 96).transpose(0, 1), w, EPS)
    assert torch.equal(y.transpose(0, 1).reshape(50, 96), want[0]) and total.shape == batch.shape


def test_no_rows_and_one_dimension():
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm, rms_norm_quantized
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    y = rms_norm(x, w, EPS)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))
    with torch.no_grad():
        values, scales, _ = rms_norm_quantized(x, w, EPS)
        assert values.shape == (0, 64) and scales.shape == (0,)
        one = torch.randn(64, device="cuda")
        y, total = add_rms_norm(one, one, w, EPS)
        assert y.shape == (64,) and torch.equal(total, one + one)
        values, scales, _ = rms_norm_quantized(one, w, EPS)
        assert scales.shape == ()


def test_only_one_of_the_outputs_is_used():
    from torchgt_b200.rms_norm import add_rms_norm
    x, r, w, dy, ds = _inputs(20, 64, torch.float32, 4)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    y, total = add_rms_norm(*leaves, EPS)
    dx, dr = torch.autograd.grad(total, leaves[:2], ds, retain_graph=True)
    assert torch.equal(dx, ds) and torch.equal(dr, ds)
    dx, dr, dw = torch.autograd.grad(y, leaves, dy)
    ref = _formula(x.detach(), r.detach(), w.detach(), dy)
    _within(dx, ref["dx"], 65 * E * ref["dx_size"])
    with torch.no_grad():
        y, total = add_rms_norm(*leaves, EPS, want_sum=False)
        assert total is None
    y, _ = add_rms_norm(x, x, w, EPS)                      # the same tensor on both sides: both gradients
    dx, = torch.autograd.grad(y, [x], dy)
    _within(dx, 2 * _formula(x.detach(), x.detach(), w.detach(), dy)["dx"],
            130 * E * _formula(x.detach(), x.detach(), w.detach(), dy)["dx_size"])


def test_differences_second_order_and_batched_gradients():
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm
    x, r, w, dy, ds = _inputs(4, 16, torch.float32, 5)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    y, total = add_rms_norm(*leaves, EPS)
    grads = torch.autograd.grad([y, total], leaves, [dy, ds])
    f = lambda x, r, w: float((_formula(x, r, w)["y"] * dy.double().cpu()).sum() +   # noqa: E731
                              ((x + r).double().cpu() * ds.double().cpu()).sum())
    d = [t.detach().double() for t in leaves]
    for k in range(3):
        step = torch.randn_like(d[k]) * 1e-4
        up, down = [list(d), list(d)]
        up[k], down[k] = d[k] + step, d[k] - step
        want = (f(*up) - f(*down)) / 2
        got = float((grads[k].double() * step).sum())
        assert abs(got - want) <= 1e-6 * float((grads[k].double().abs() * step.abs()).sum()), (k, got, want)
    y = rms_norm(x, w, EPS)
    g, = torch.autograd.grad(y, [x], dy, create_graph=True)
    second, = torch.autograd.grad(g.square().sum(), [w])
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    yd = torch.nn.functional.rms_norm(xd, (16,), wd, EPS)
    gd, = torch.autograd.grad(yd, [xd], dy.double(), create_graph=True)
    wanted, = torch.autograd.grad(gd.square().sum(), [wd])
    # recorded operations in fp32: a few hundred roundings over 64 terms
    _within(second, wanted.cpu(), 1e-5 * wanted.abs().max().cpu())
    y, total = add_rms_norm(*leaves, EPS)
    many = torch.autograd.grad(y, leaves, torch.stack([dy, ds]), is_grads_batched=True)
    assert many[0].shape == (2, 4, 16) and many[2].shape == (2, 16)
    _within(many[0][0], _formula(x.detach(), r.detach(), w.detach(), dy)["dx"],
            128 * E * _formula(x.detach(), r.detach(), w.detach(), dy)["dx_size"])


def test_same_bits_on_other_streams_and_from_a_graph():
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm_quantized
    x, r, w, dy, ds = _inputs(3000, 192, torch.bfloat16, 6)
    def step():
        leaves = [t.detach().requires_grad_() for t in (x, r, w)]
        y, total = add_rms_norm(*leaves, EPS)
        with torch.no_grad():
            q = rms_norm_quantized(x, w, EPS, r)
        return [y.detach(), total.detach(), *torch.autograd.grad([y, total], leaves, [dy, ds]), q[0].view(torch.uint8), q[1]]
    want = step()
    for a, b in zip(step(), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    x.mul_(0.5)
    graph.replay()
    halved = [t.clone() for t in captured]
    x.mul_(2)
    graph.replay()
    for a, b, c, d in zip(others, want, captured, halved):
        assert torch.equal(a, b) and torch.equal(c, b)
    assert not torch.equal(halved[0], want[0])


def test_module_is_a_drop_in():
    from torchgt_b200 import RMSNorm
    ours, theirs = RMSNorm(64).cuda(), torch.nn.RMSNorm(64).cuda()
    theirs.weight.data.normal_()
    ours.load_state_dict(theirs.state_dict())
    x = torch.randn(3, 50, 64, device="cuda")
    ref = theirs.double()(x.double()).cpu()
    _within(ours(x), ref, 65 * E * ref.abs())
    y, total = ours.add(x, x)
    assert torch.equal(total, x + x)
    seen = []
    handle = ours.register_forward_hook(lambda m, a, out: seen.append(out))
    hooked, _ = ours.add(x, x)
    handle.remove()
    assert len(seen) == 1 and torch.equal(seen[0], hooked)
    _within(hooked, y.double().cpu(), 130 * E * y.double().cpu().abs())
    half = torch.randn(5, 64, device="cuda", dtype=torch.float16)
    assert torch.equal(RMSNorm(64).cuda().half()(half), torch.nn.RMSNorm(64).cuda().half()(half))
    odd = RMSNorm((2, 32)).cuda()
    assert torch.equal(odd(x.view(150, 2, 32)), torch.nn.functional.rms_norm(x.view(150, 2, 32), (2, 32), odd.weight))
