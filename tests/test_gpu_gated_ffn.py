"""The gated feed-forward block's kernels against the formula in 64 bits.

Bounds, u the rounding of the tensors' type (bf16 2^-8, fp32 2^-24) and e = 2^-24 of the sums.  With |.| the sums of magnitudes of a
product's terms: a product of length k is off by at most s(k) = (k + 16) e of its magnitudes (every step of a running sum, the
tensor cores' rounding towards zero at every sixteen terms among them), fast exponentials and quotients add 2^-19.  Written out:
  g, u:  s(in) |.|            h:  u |h| + what g and u are off, times the slope (at most 1.13 for silu, gelu, relu) and |u|, |act(g)|
  y:     u |y| + s(mid) |.| + what h is off, through |Wd|
Backward, g and u as they were kept (in bf16 cut off after 16 bits): dg, du are rounded once, dh is s(out), and the slope moves by its
own derivative (at most 1.2) times what g is off.  All of it is carried through below with magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E, FAST = 2.0 ** -24, 2.0 ** -19
ROUNDING = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _activation(name, g):
    if name == "relu":
        return g.clamp(min=0), (g > 0).double()
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
    return g * cdf, cdf + g * torch.exp(-g * g / 2) * (2 * torch.pi) ** -0.5


def _formula(x, wg, wu, wd, act, residual, dy):
    """{name: (value, bound)} with bounds carried through by magnitudes."""
    u_ = ROUNDING[x.dtype]
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))
    n_in, n_mid, n_out, rows = wg.shape[1], wg.shape[0], wd.shape[0], x.shape[0]
    s = lambda k: (k + 16) * E   # noqa: E731
    g, u = x @ wg.T, x @ wu.T
    gm, um = x.abs() @ wg.abs().T, x.abs() @ wu.abs().T
    dg_, du_ = s(n_in) * gm, s(n_in) * um                      # what g and u are off
    a, slope = _activation(act, g)
    a_off = 1.13 * dg_ + FAST * a.abs()
    h = a * u
    h_off = u_ * h.abs() + (a_off * u.abs() + a.abs() * du_) * 1.01 + 8 * E * h.abs()
    y = h @ wd.T + (0 if residual is None else residual.detach().double())
    y_mag = h.abs() @ wd.abs().T + (0 if residual is None else residual.detach().double().abs())
    out = {"y": (y, u_ * y.abs() + s(n_mid) * y_mag + 1.01 * h_off @ wd.abs().T)}
    if dy is None:
        return out
    dy = dy.double()
    cut = 0 if u_ == 2.0 ** -24 else 2.0 ** -15
    gk, uk = dg_ + cut * g.abs(), du_ + cut * u.abs()          # g and u as kept
    dh, dh_off = dy @ wd, s(n_out) * (dy.abs() @ wd.abs())
    slope_off = 1.2 * gk + FAST if act != "relu" else (gk >= g.abs()).double()      # relu: one side of zero for the other
    ak_off = 1.13 * gk + FAST * a.abs()
    dg, du = dh * u * slope, dh * a
    dg_off = u_ * dg.abs() + 1.02 * (dh_off * (u * slope).abs() + dh.abs() * uk * slope.abs() + (dh * u).abs() * slope_off) + 8 * E * dg.abs()
    du_off = u_ * du.abs() + 1.02 * (dh_off * a.abs() + dh.abs() * ak_off) + 8 * E * du.abs()
    dx = dg @ wg + du @ wu
    out["dx"] = (dx, u_ * dx.abs() + s(2 * n_mid) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()) + 1.01 * (dg_off @ wg.abs() + du_off @ wu.abs()))
    for name, d, off, of, of_off in (("dgate", dg, dg_off, x, 0), ("dup", du, du_off, x, 0), ("ddown", dy, 0, h, h_off)):
        value = d.T @ of
        carried = (off.T @ of.abs() if torch.is_tensor(off) else 0) + (d.abs().T @ of_off if torch.is_tensor(of_off) else 0)
        out[name] = (value, u_ * value.abs() + s(rows) * (d.abs().T @ of.abs()) + 1.01 * carried)
    return out


def _within(got, ref, name):
    value, bound = ref
    off = (got.double() - value.view(got.shape)).abs()
    assert bool((off <= bound.view(got.shape) + 1e-300).all()), (name, float((off / (bound.view(got.shape) + 1e-300)).max()))


def _inputs(rows, n_in, n_mid, n_out, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, device="cuda") * scale).to(dtype)   # noqa: E731
    return (draw(rows, n_in), draw(n_mid, n_in, scale=n_in ** -0.5), draw(n_mid, n_in, scale=n_in ** -0.5),
            draw(n_out, n_mid, scale=n_mid ** -0.5), draw(rows, n_out), draw(rows, n_out))


def _check(rows, n_in, n_mid, n_out, dtype, act, with_residual, seed=0):
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, dy = _inputs(rows, n_in, n_mid, n_out, dtype, seed + rows + n_mid)
    residual = r if with_residual else None
    with torch.no_grad():
        plain = gated_feed_forward(x, wg, wu, wd, act, residual)
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)] + ([r.requires_grad_()] if with_residual else [])
    y = gated_feed_forward(x, wg, wu, wd, act, residual)
    assert y.dtype == dtype and y.shape == (rows, n_out)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = _formula(x, wg, wu, wd, act, residual, dy)
    _within(y.detach(), ref["y"], "y")
    _within(plain, ref["y"], "y without gradients")
    for name, got in zip(("dx", "dgate", "dup", "ddown"), grads):
        _within(got, ref[name], name)
    if with_residual:
        assert torch.equal(grads[4], dy)


BF16 = [(1, 8, 8, 8), (1, 64, 128, 64), (2, 2048, 5632, 2048), (5, 72, 200, 40), (17, 768, 2048, 768), (33, 264, 136, 520),
        (64, 512, 512, 512), (127, 64, 64, 64), (128, 128, 256, 128), (129, 1000, 1544, 328), (333, 768, 2048, 768), (1000, 64, 128, 64),
        (2049, 520, 1032, 264), (4097, 64, 192, 64), (20000, 128, 64, 72),
        (16384, 1024, 2816, 1024)]      # 88 tiles of the weights' gradients: some whole, some shared


@pytest.mark.parametrize("rows,n_in,n_mid,n_out", BF16)
def test_bf16(rows, n_in, n_mid, n_out):
    _check(rows, n_in, n_mid, n_out, torch.bfloat16, "silu", rows % 2 == 1)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 24, 31, 32])
def test_a_few_rows_without_gradients(rows, act):
    """As serving calls it: widths around the kernels' steps of 8, 16, 32 and whole turns of k."""
    from torchgt_b200 import gated_feed_forward
    for n_in, n_mid, n_out in ((8, 8, 8), (40, 24, 56), (256, 136, 264), (2048, 512, 40), (2056, 4104, 72)):
        x, wg, wu, wd, r, _ = _inputs(rows, n_in, n_mid, n_out, torch.bfloat16, 23)
        for residual in (None, r):
            got = gated_feed_forward(x, wg, wu, wd, act, residual)
            _within(got, _formula(x, wg, wu, wd, act, residual, None)["y"], (n_in, n_mid, n_out))
        again = gated_feed_forward(x, wg, wu, wd, act, r)
        assert torch.equal(again, got)
        # a row's result does not depend on how many there are beside it
        assert torch.equal(gated_feed_forward(x[:1], wg, wu, wd, act, r[:1]), got[:1]) or rows > 8


@pytest.mark.parametrize("rows", [1, 8, 13, 16, 27, 32])
@pytest.mark.parametrize("n_in,n_mid,n_out", [(264, 11016, 1016), (136, 1800, 2376), (1032, 72, 4096), (64, 4744, 4744), (24, 200, 16392)])
def test_a_few_rows_of_wide_outputs(rows, n_in, n_mid, n_out):
    """One set of columns of y a CTA, two, and more CTAs than SMs; more of k than the steps that are under way."""
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, _ = _inputs(rows, n_in, n_mid, n_out, torch.bfloat16, 31)
    got = gated_feed_forward(x, wg, wu, wd, "silu", r)
    _within(got, _formula(x, wg, wu, wd, "silu", r, None)["y"], "y")
    x[rows - 1] = float("inf")
    spoilt = gated_feed_forward(x, wg, wu, wd, "silu", r)
    assert torch.equal(spoilt[:rows - 1], got[:rows - 1]) and not bool(spoilt[rows - 1].isfinite().any())
    h = torch.cuda.CUDAGraph()
    with torch.cuda.graph(h):
        y = gated_feed_forward(x, wg, wu, wd, "silu", r)
    x[rows - 1] = 0.5
    want = gated_feed_forward(x, wg, wu, wd, "silu", r)
    for _ in range(3):
        h.replay()
    assert torch.equal(y, want)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("rows,n_in,n_mid,n_out", [(33, 2048, 512, 64), (40, 4096, 72, 768), (100, 520, 5632, 200), (129, 1096, 2056, 72),
                                                   (333, 768, 2048, 768), (500, 4104, 264, 136), (700, 64, 4096, 8)])
def test_tiles_split_along_k(rows, n_in, n_mid, n_out, act):
    """Products with fewer tiles than the chip has SMs, some of them several CTAs to a tile; with and without what gradients keep."""
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, _ = _inputs(rows, n_in, n_mid, n_out, torch.bfloat16, 29)
    for residual in (None, r):
        want = _formula(x, wg, wu, wd, act, residual, None)["y"]
        with torch.no_grad():
            got = gated_feed_forward(x, wg, wu, wd, act, residual)
        _within(got, want, "y")
        kept = gated_feed_forward(x.clone().requires_grad_(), wg, wu, wd, act, residual)
        assert torch.equal(got, kept.detach())
    x[3] = float("nan")
    with torch.no_grad():
        spoilt = gated_feed_forward(x, wg, wu, wd, act, r)
    others = [i for i in range(rows) if i != 3]
    assert torch.equal(spoilt[others], got[others]) and bool(spoilt[3].isnan().all())


@pytest.mark.parametrize("rows,n_in,n_mid,n_out", [(1, 64, 64, 64), (3, 64, 128, 4), (200, 128, 64, 100), (4097, 64, 128, 64), (9000, 64, 64, 64),
                                                   (700, 1024, 1024, 1024)])
def test_fp32(rows, n_in, n_mid, n_out):
    _check(rows, n_in, n_mid, n_out, torch.float32, "silu", rows % 2 == 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["gelu", "relu"])
def test_other_activations(act, dtype):
    for rows in (3, 40, 600):
        _check(rows, 192, 320, 192, dtype, act, True, seed=7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows_other_shapes_and_views(dtype):
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, dy = _inputs(60, 64, 128, 64, dtype, 3)
    want = gated_feed_forward(x, wg, wu, wd, "silu", r)
    none = x[:0].requires_grad_()
    weights = [t.clone().requires_grad_() for t in (wg, wu, wd)]
    y = gated_feed_forward(none, *weights)
    grads = torch.autograd.grad(y, [none, *weights], torch.zeros_like(y))
    assert y.shape == (0, 64) and all(not bool(g.any()) for g in grads)
    x = x.detach()
    assert torch.equal(gated_feed_forward(x.view(3, 20, 64), wg, wu, wd, "silu", r.view(3, 20, 64)).view(60, 64), want)
    flat = torch.zeros(60 * 64 + 1, dtype=dtype, device="cuda")
    flat[1:] = x.flatten()
    wide = torch.zeros(128, 100, dtype=dtype, device="cuda")
    wide[:, 20:84] = wg
    turned = wd.t().contiguous().t()
    assert torch.equal(gated_feed_forward(flat[1:].view(60, 64), wide[:, 20:84], wu, turned, "silu", r), want)
    one = gated_feed_forward(x[7], wg, wu, wd, "silu", r[7])
    assert one.shape == (64,)
    ref = _formula(x[7:8], wg, wu, wd, "silu", r[7:8], None)["y"]
    _within(one.view(1, 64), ref, "one row")


def test_rows_behind_the_last_and_next_to_a_nan():
    """A row with a NaN or an infinity changes no other; memory behind the results stays as it was."""
    import ctypes
    from torchgt_b200 import _cabi, gated_feed_forward
    for rows in (5, 300):
        x, wg, wu, wd, r, dy = _inputs(rows, 128, 192, 128, torch.bfloat16, 9)
        clean = gated_feed_forward(x, wg, wu, wd)
        x[1, 3], x[4, 100] = float("nan"), float("inf")
        got = gated_feed_forward(x, wg, wu, wd)
        others = [i for i in range(rows) if i not in (1, 4)]
        assert torch.equal(got[others], clean[others]) and bool(got[1].isnan().all()) and not bool(got[4].isfinite().all())
        h = torch.full((rows + 9, 192), 7.0, dtype=torch.bfloat16, device="cuda")
        y = torch.full((rows + 9, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        lib, stream = _cabi.load(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        _cabi.check(lib.tgt_gated_hidden(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), rows, 128, 192, 3, 1, h.data_ptr(), None, None,
                                         None, stream))
        _cabi.check(lib.tgt_gated_output(h.data_ptr(), wd.data_ptr(), None, rows, 192, 128, 1, y.data_ptr(), stream))
        assert bool((h[rows:] == 7).all()) and bool((y[rows:] == 7).all()) and torch.equal(y[:rows].nan_to_num(), got.nan_to_num())
    _cabi.check(lib.tgt_products_status())


def test_gradients_of_some_inputs_only():
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, dy = _inputs(200, 64, 128, 64, torch.bfloat16, 11)
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd, r)]
    every = torch.autograd.grad(gated_feed_forward(*leaves[:4], "silu", leaves[4]), leaves, dy)
    for k in range(5):
        some = [t.detach().requires_grad_(i == k) for i, t in enumerate(leaves)]
        got, = torch.autograd.grad(gated_feed_forward(*some[:4], "silu", some[4]), [some[k]], dy)
        assert torch.equal(got, every[k])
    # one tensor as the input and the residual
    x = leaves[0].detach().requires_grad_()
    both, = torch.autograd.grad(gated_feed_forward(x, wg, wu, wd, "silu", x), [x], dy)
    assert torch.equal(both, every[0] + dy)


def test_differences_second_order_and_batched_gradients():
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, dy = _inputs(6, 64, 64, 64, torch.float32, 13)
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    for act in ("silu", "gelu"):
        grads = torch.autograd.grad(gated_feed_forward(*leaves, act), leaves, dy)
        f = lambda *t: float((_formula(*t, act, None, None)["y"][0] * dy.double()).sum())   # noqa: E731
        d = [t.detach().double() for t in leaves]
        ROUNDING[torch.float64] = 0.0
        for k in range(4):
            step = torch.randn_like(d[k]) * 1e-5
            up, down = list(d), list(d)
            up[k], down[k] = d[k] + step, d[k] - step
            want, got = (f(*up) - f(*down)) / 2, float((grads[k].double() * step).sum())
            assert abs(got - want) <= 1e-6 * float((grads[k].double().abs() * step.abs()).sum()), (act, k)
        g, = torch.autograd.grad(gated_feed_forward(*leaves, act), [x], dy, create_graph=True)
        second = torch.autograd.grad(g.square().sum(), leaves[1:])
        d = [t.detach().double().requires_grad_() for t in leaves]
        a = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act]
        gd, = torch.autograd.grad((a(d[0] @ d[1].T) * (d[0] @ d[2].T)) @ d[3].T, [d[0]], dy.double(), create_graph=True)
        for got, want in zip(second, torch.autograd.grad(gd.square().sum(), d[1:])):
            # fp32 operations with sums of 64 terms, a dozen of them in a row
            assert float((got.double() - want).abs().max()) <= 1e-4 * float(want.abs().max())
        many = torch.autograd.grad(gated_feed_forward(*leaves, act), leaves, torch.stack([dy, 2 * dy]), is_grads_batched=True)
        for one, batch in zip(grads, many):
            assert batch.shape == (2,) + one.shape
            assert float((batch[0] - one).abs().max()) <= 1e-4 * float(one.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_bits_on_other_streams_and_from_two_graphs(dtype):
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, dy = _inputs(1500, 192, 256, 192, dtype, 17)
    few = x[:3].clone()

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd, r)]
        y = gated_feed_forward(*leaves[:4], "silu", leaves[4])
        with torch.no_grad():
            short = gated_feed_forward(few, wg, wu, wd)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy), short]
    want = step()
    for a, b in zip(step(), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, held = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(step())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for a, b, c, d in zip(want, other, *held):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)


def test_what_the_kernels_do_not_cover_is_the_same_block_of_torch():
    from torchgt_b200 import GatedFeedForward, gated_feed_forward
    for dtype, widths in ((torch.float16, (64, 128, 64)), (torch.bfloat16, (60, 100, 60)), (torch.float32, (60, 100, 60))):
        x, wg, wu, wd, r, _ = _inputs(10, *widths, dtype, 1)
        want = (torch.nn.functional.silu(x @ wg.t()) * (x @ wu.t())) @ wd.t() + r
        torch.testing.assert_close(gated_feed_forward(x, wg, wu, wd, "silu", r), want, rtol=2e-2, atol=2e-2)
    module = GatedFeedForward(64, 128, "gelu").cuda()
    x = torch.randn(2, 100, 64, device="cuda")
    assert sorted(module.state_dict()) == ["down", "gate", "up"]
    ref = _formula(x.view(200, 64), module.gate, module.up, module.down, "gelu", x.view(200, 64), None)["y"]
    _within(module(x, x).detach().view(200, 64), ref, "module")
