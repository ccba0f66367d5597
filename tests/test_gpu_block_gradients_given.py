"""The gradients that the operators of a block are given, in forms that autograd has for them: lazily negated ones, as the imaginary
part of a conjugate is, and ones with tangents."""
import pytest
import torch

from helpers import TOL_F32, rel_err

pytestmark = pytest.mark.gpu


def _operators(dtype):
    """(what it is called, its output's function of its leaves, the leaves)"""
    from torchgt_b200 import SparseGraph, edge_position_bias, gated_feed_forward, sparse_graph_attention
    from torchgt_b200.layer_norm import layer_norm
    from torchgt_b200.linear import linear
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm
    gen = torch.Generator().manual_seed(71)
    draw = lambda *s, scale=1.0: (torch.randn(*s, generator=gen) * scale).to(dtype).cuda().requires_grad_()   # noqa: E731
    x, r, w = draw(300, 64), draw(300, 64), draw(64)
    wg, wu, wd = draw(128, 64, scale=0.125), draw(128, 64, scale=0.125), draw(64, 128, scale=0.09)
    edges = torch.randint(0, 300, (2, 2000), generator=gen).cuda()
    table = torch.randn(32, 8, generator=gen).cuda().requires_grad_()
    q, k, v = draw(300, 8, 8), draw(300, 8, 8), draw(300, 8, 8)
    scores = torch.randn(2000, 8, generator=gen).cuda().requires_grad_()
    graph = SparseGraph(edges, 300)
    more = []
    if dtype == torch.float32:
        more = [("layer norm", lambda x, w, b: layer_norm(x, w, b), [x, w, draw(64)]),
                ("linear", lambda x, w, b: linear(x, w, b), [x, draw(128, 64), draw(128)])]
    return more + [
            ("attention", lambda q, k, v: sparse_graph_attention(q, k, v, graph), [q, k, v]),
            ("attention with a bias", lambda q, k, v, b: sparse_graph_attention(q, k, v, graph, b), [q, k, v, scores]),
            ("norm", lambda x, w: rms_norm(x, w, 1e-6), [x, w]),
            ("norm of a sum", lambda x, r, w: add_rms_norm(x, r, w, 1e-6)[0], [x, r, w]),
            ("sum", lambda x, r, w: sum(add_rms_norm(x, r, w, 1e-6)), [x, r, w]),
            ("gated", lambda *t: gated_feed_forward(*t), [x, wg, wu, wd]),
            ("gated with a residual", lambda x, wg, wu, wd, r: gated_feed_forward(x, wg, wu, wd, "gelu", r), [x, wg, wu, wd, r]),
            ("bias", lambda t: edge_position_bias(t, edges), [table])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lazily_negated(dtype):
    for name, f, leaves in _operators(dtype):
        y = f(*leaves)
        dy = torch.randn(y.shape, device="cuda").to(y.dtype)
        want = torch.autograd.grad(f(*leaves), leaves, -dy)
        lazy = torch._neg_view(dy)
        assert lazy.is_neg() and lazy.is_contiguous()
        for a, b in zip(torch.autograd.grad(f(*leaves), leaves, lazy), want):
            assert torch.equal(a, b), name
        if y.dtype == torch.float32:                        # as a user comes by them
            z = torch.complex(torch.zeros_like(dy), dy).conj()
            assert z.imag.is_neg()
            for a, b in zip(torch.autograd.grad(f(*leaves), leaves, z.imag), want):
                assert torch.equal(a, b), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lazily_negated_inputs_of_the_attention(dtype):
    """Which it has kernels for only; the others are torch's operations for such inputs."""
    for name, f, leaves in _operators(dtype):
        if name.startswith("attention"):
            values = [t.detach() for t in leaves]
            assert torch.equal(f(*[torch._neg_view(t) for t in values]), f(*[-t for t in values])), name


def test_with_tangents():
    """Forward-mode derivatives of a backward pass: it is linear in what it is given, so its tangent is the backward of the tangent."""
    import torch.autograd.forward_ad as forward_ad
    for name, f, leaves in _operators(torch.float32):
        if not name.startswith(("norm", "sum", "gated", "bias")):
            continue
        y = f(*leaves)
        dy, tangent = torch.randn_like(y), torch.randn_like(y)
        want = [torch.autograd.grad(f(*leaves), leaves, t) for t in (dy, tangent)]
        with forward_ad.dual_level():
            for got, primal, slope in zip(torch.autograd.grad(f(*leaves), leaves, forward_ad.make_dual(dy, tangent)), *want):
                parts = forward_ad.unpack_dual(got)
                assert parts.tangent is not None, name
                assert rel_err(parts.primal, primal) <= TOL_F32 and rel_err(parts.tangent, slope) <= TOL_F32, name
