"""Tensors of more than 2^31 values: offsets that 32 bits do not hold.  Rows near both ends are compared, bit by bit, with the same rows in
a short call or with the formula; sums over all rows with 64 bits, a piece of the rows at a time."""
import pytest
import torch

from test_gpu_gated_ffn import _formula as gated_formula
from test_gpu_gated_ffn import _inputs as gated_inputs
from test_gpu_gated_ffn import _within as gated_within

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def _summed(rows, f, step=1 << 17):
    """Sum of f(rows of a piece) over the pieces, in 64 bits."""
    total = None
    for at in range(0, rows, step):
        part = f(slice(at, min(rows, at + step)))
        total = part if total is None else total + part
    return total


@pytest.mark.parametrize("dtype,rows,hidden", [(torch.bfloat16, 1060001, 2056), (torch.float32, 540001, 4100)])
def test_norm(dtype, rows, hidden):
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm_quantized
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, r, dy = (torch.empty(rows, hidden, dtype=dtype, device="cuda").normal_(generator=gen) for _ in range(3))
    w = torch.rand(hidden, generator=gen, device="cuda").to(dtype) + 0.5
    assert x.numel() > 2 ** 31
    leaves = [t.requires_grad_() for t in (x, r, w)]
    y, total = add_rms_norm(*leaves, 1e-6)
    dx, _, dw = torch.autograd.grad([y, total], leaves, [dy, dy])
    with torch.no_grad():
        values, scales, _ = rms_norm_quantized(x, w, 1e-6, r)
        rstd = torch.cat([1 / torch.sqrt(((x[s].double() + r[s].double()) ** 2).mean(-1) + 1e-6) for s in
                          (slice(at, at + (1 << 17)) for at in range(0, rows, 1 << 17))])
        term = lambda s: dy[s].double() * (x[s].double() + r[s].double()) * rstd[s, None]   # noqa: E731
        want, size = _summed(rows, lambda s: term(s).sum(0)), _summed(rows, lambda s: term(s).abs().sum(0))
        u, seen = (2.0 ** -8, 2.0 ** -15) if dtype == torch.bfloat16 else (2.0 ** -24, 0)
        # a thread adds up the rows of every 148th to 600th CTA, 7,200 at most, one after the other, then CTAs' sums a few at a time
        assert bool(((dw.double() - want).abs() <= u * want.abs() + (8192 * E + seen) * size).all())
    for s in (slice(0, 40), slice(rows - 40, rows), slice(2 ** 31 // hidden - 20, 2 ** 31 // hidden + 20)):
        short = [t.detach()[s].clone().requires_grad_() for t in (x, r)] + [w.detach().clone().requires_grad_()]
        ys, ts = add_rms_norm(*short, 1e-6)
        dxs, _, _ = torch.autograd.grad([ys, ts], short, [dy[s], dy[s]])
        with torch.no_grad():
            vs, ss, _ = rms_norm_quantized(short[0], short[2], 1e-6, short[1])
        for a, b in ((y[s], ys), (total[s], ts), (dx[s], dxs), (values[s].view(torch.uint8), vs.view(torch.uint8)), (scales[s], ss)):
            assert torch.equal(a, b)


def test_bias():
    from torchgt_b200 import edge_position_bias
    edges, heads, nodes = 68000003, 32, 100000
    gen = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randint(0, nodes, (2, edges), generator=gen, device="cuda", dtype=torch.int32)
    positions = torch.randint(0, 300, (nodes,), generator=gen, device="cuda")
    table = torch.randn(32, heads, generator=gen, device="cuda").requires_grad_()
    assert edges * heads > 2 ** 31
    bias = edge_position_bias(table, ids, positions)
    for s in (slice(0, 1000), slice(edges - 1000, edges), slice(2 ** 31 // heads - 500, 2 ** 31 // heads + 500)):
        assert torch.equal(bias[s], edge_position_bias(table, ids[:, s], positions))
    dbias = torch.empty_like(bias).normal_(generator=gen)
    del bias
    got, = torch.autograd.grad(edge_position_bias(table, ids, positions), [table], dbias)
    tables = torch.eye(32, device="cuda")[:, :].contiguous()     # a bucket's number from the kernel's own rows, checked above
    number = lambda s: edge_position_bias(tables, ids[:, s], positions).argmax(1)   # noqa: E731
    add = lambda s, d: torch.zeros(32, heads, dtype=torch.float64, device="cuda").index_add_(0, number(s), d.double())   # noqa: E731
    want, size = _summed(edges, lambda s: add(s, dbias[s]), 1 << 21), _summed(edges, lambda s: add(s, dbias[s].abs()), 1 << 21)
    # a lane's sums are of one edge in every 888 CTAs x 8 warps: 68 M / 7,104 edges, a bucket has up to a fifth of them; then 300 parts
    assert bool(((got.double() - want).abs() <= 4096 * E * size).all())


@pytest.mark.parametrize("dtype,rows,n_in,n_mid,n_out", [(torch.bfloat16, 2100001, 64, 1032, 64), (torch.float32, 2200001, 64, 1024, 64)])
def test_gated_block(dtype, rows, n_in, n_mid, n_out):
    from torchgt_b200 import gated_feed_forward
    x, wg, wu, wd, r, dy = gated_inputs(rows, n_in, n_mid, n_out, dtype, 3)
    assert rows * n_mid > 2 ** 31
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves, "silu", r)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        for s in (slice(0, 300), slice(rows - 300, rows), slice(2 ** 31 // n_mid - 150, 2 ** 31 // n_mid + 150)):
            ref = gated_formula(x[s], wg, wu, wd, "silu", r[s], dy[s])
            gated_within(y[s], ref["y"], "y")
            gated_within(grads[0][s], ref["dx"], "dx")
        for k, name in enumerate(("dgate", "dup", "ddown"), 1):
            parts = lambda s: torch.stack(gated_formula(x[s], wg, wu, wd, "silu", r[s], dy[s])[name])   # noqa: B023,E731
            value, bound = _summed(rows, parts)
            # the pieces' bounds have a product of their own length in them, (131,072 + 16) e; the whole's is this much longer
            gated_within(grads[k], (value, bound * (rows / (1 << 17) + 1)), name)
