"""The widths that each C entry of the gated block takes in fp32: multiples of 4 up to 1,024, the input of weight gradients of 64."""
import ctypes

import pytest
import torch

from helpers import rel_err

ACTS = {"relu": 1, "gelu": 2, "silu": 3}


def test_refusals():
    from torchgt_b200 import _cabi
    from torchgt_b200.build import build
    build()
    lib, n = _cabi.load(), ctypes.c_size_t()
    for width in (6, 62, 1028):
        assert lib.tgt_gated_hidden(16, 16, 16, 1, width, 64, 3, 0, 16, 16, 16, None, None) == 3
        assert lib.tgt_gated_hidden(16, 16, 16, 1, 64, width, 3, 0, 16, 16, 16, None, None) == 3
        assert lib.tgt_gated_output(16, 16, None, 1, width, 64, 0, 16, None) == 3
        assert lib.tgt_gated_output(16, 16, None, 1, 64, width, 0, 16, None) == 3
        assert lib.tgt_gated_hidden_grad(16, 16, 16, 16, None, 1, width, 64, 3, 0, 16, 16, None) == 3
        assert lib.tgt_gated_hidden_grad(16, 16, 16, 16, None, 1, 64, width, 3, 0, 16, 16, None) == 3
        assert lib.tgt_gated_input_grad(16, 16, 16, 16, 1, width, 64, 0, 16, None) == 3
        assert lib.tgt_gated_input_grad(16, 16, 16, 16, 1, 64, width, 0, 16, None) == 3
    size = lambda out, into: lib.tgt_gated_weight_grad_scratch_bytes(2, 100, out, into, 0, ctypes.byref(n))   # noqa: E731
    assert size(100, 60) == 3 and size(100, 68) == 3 and size(102, 64) == 3 and size(1028, 64) == 3 and size(64, 1088) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("rows", [40, 12001])                # the gate in kernels of its own, and in the products' finish
@pytest.mark.parametrize("n_in,n_mid,n_out", [(36, 100, 44), (132, 68, 20), (4, 4, 4)])
def test_multiples_of_four(n_in, n_mid, n_out, rows, act):
    """Against 64 bits: sums of at most 200 terms, each off by 2^-24 of the magnitudes a dozen times, through three products."""
    from torchgt_b200 import _cabi
    lib, stream = _cabi.load(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    gen = torch.Generator(device="cuda").manual_seed(rows + n_in)
    draw = lambda *s, scale=1.0: torch.randn(*s, generator=gen, device="cuda") * scale   # noqa: E731
    x, dy, add = draw(rows, n_in), draw(rows, n_out), draw(rows, n_out)
    wg, wu, wd = draw(n_mid, n_in, scale=n_in ** -0.5), draw(n_mid, n_in, scale=n_in ** -0.5), draw(n_out, n_mid, scale=n_mid ** -0.5)
    h, gate, up, dgate, dup = (torch.full((rows + 1, n_mid), 7.0, device="cuda") for _ in range(5))
    y, dx = torch.full((rows + 1, n_out), 7.0, device="cuda"), torch.full((rows + 1, n_in), 7.0, device="cuda")
    p = lambda *t: [None if v is None else v.data_ptr() for v in t]   # noqa: E731
    _cabi.check(lib.tgt_gated_hidden(*p(x, wg, wu), rows, n_in, n_mid, ACTS[act], 0, *p(h, gate, up, None), stream))
    _cabi.check(lib.tgt_gated_output(*p(h, wd, add), rows, n_mid, n_out, 0, *p(y), stream))
    _cabi.check(lib.tgt_gated_hidden_grad(*p(dy, wd, gate, up, None), rows, n_out, n_mid, ACTS[act], 0, *p(dgate, dup), stream))
    _cabi.check(lib.tgt_gated_input_grad(*p(dgate, dup, wg, wu), rows, n_mid, n_in, 0, *p(dx), stream))
    d = [t.double().requires_grad_() for t in (x, wg, wu, wd)]
    g, u = d[0] @ d[1].t(), d[0] @ d[2].t()
    g.retain_grad(), u.retain_grad()
    hd = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}[act](g) * u
    yd = hd @ d[3].t() + add.double()
    yd.backward(dy.double())
    for got, want in ((gate, g), (up, u), (h, hd), (y, yd), (dgate, g.grad), (dup, u.grad), (dx, d[0].grad)):
        assert rel_err(got[:rows], want) <= 1e-5 and bool((got[rows:] == 7).all())
