"""The operators of a pre-norm block together, as a model calls them: norm, projections, sparse attention with the relative
position bias, residual and norm, gated feed-forward half; training against the same block in 64 bits, and serving rows.

Five operators stand between an input and an output, each held to the parity contract by its own tests (1e-5 of the largest
value in fp32, 1e-2 in bf16): five times that here, and ten for gradients, which pass all of them twice.

Gradients through the scores are differences: an edge's is w (dO.V / Z - dZ), the two terms being equal where all of a row's edges
have the same value.  Then the result vanishes and its roundings do not: with one row for q, k and the table, and always for k's bias,
which adds the same to all scores of a row and is taken out by the quotient (1e-6 of it is left, by the 1e-6 in the denominator).  What
rounds are the terms, so these are held to the largest sum of the terms' magnitudes, w (|dO.V| / Z + |dZ|) |k| / sqrt(D) and so on."""
import pytest
import torch

from helpers import TOL_BF16, TOL_F32, rel_err

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, FFN, EPS = 64, 8, 128, 1e-6


def _block(dtype, seed=0):
    from torchgt_b200 import GatedFeedForward, Linear, RelativePositionBias, RMSNorm
    torch.manual_seed(seed)
    block = torch.nn.ModuleDict({"norm": RMSNorm(HIDDEN, eps=EPS), "q": Linear(HIDDEN, HIDDEN), "k": Linear(HIDDEN, HIDDEN),
                                 "v": Linear(HIDDEN, HIDDEN), "out": Linear(HIDDEN, HIDDEN), "ffn_norm": RMSNorm(HIDDEN, eps=EPS),
                                 "ffn": GatedFeedForward(HIDDEN, FFN), "bias": RelativePositionBias(HEADS)}).cuda()
    for name in ("norm", "q", "k", "v", "out", "ffn_norm", "ffn"):
        block[name].to(dtype)
    return block


def _forward(block, x, edges, graph, positions):
    from torchgt_b200 import sparse_graph_attention
    y = block["norm"](x)
    q, k, v = (block[n](y).view(-1, HEADS, HIDDEN // HEADS) for n in "qkv")
    attended = sparse_graph_attention(q, k, v, graph, block["bias"](edges, positions)).reshape(x.shape)
    y, x = block["ffn_norm"].add(block["out"](attended), x)
    return block["ffn"](y, x)


def _in_64_bits(parameters, x, edges, positions):
    from torchgt_b200.position_bias import bucket_borders
    p = parameters
    norm = lambda t, w: t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * w   # noqa: E731
    y = norm(x, p["norm.weight"])
    q, k, v = (torch.nn.functional.linear(y, p[f"{n}.weight"], p[f"{n}.bias"]).view(-1, HEADS, HIDDEN // HEADS) for n in "qkv")
    s, d = edges
    offset = positions[s] - positions[d]
    bucket = sum((offset.abs() >= b).long() for b in bucket_borders(32, 128, True)) + (offset > 0).long() * 16
    score = (k[s] * q[d]).sum(-1) / (HIDDEN // HEADS) ** 0.5
    w = torch.exp(score.clamp(-5, 5) + p["bias.weight"][bucket])
    u = torch.zeros_like(q).index_add_(0, d, w.unsqueeze(-1) * v[s])
    z = torch.zeros(q.shape[:2], dtype=q.dtype, device=q.device).index_add_(0, d, w)
    x = x + torch.nn.functional.linear((u / (z + 1e-6).unsqueeze(-1)).view(x.shape), p["out.weight"], p["out.bias"])
    second = norm(x, p["ffn_norm.weight"])
    out = x + (torch.nn.functional.silu(second @ p["ffn.gate"].t()) * (second @ p["ffn.up"].t())) @ p["ffn.down"].t()
    u.retain_grad()
    z.retain_grad()

    def sizes():
        """After a backward pass: the largest sum of magnitudes in the gradients through the scores."""
        m = w.detach() * ((u.grad[d] * v.detach()[s]).sum(-1).abs() + z.grad[d].abs())
        rows = lambda at, by: torch.zeros_like(q).index_add_(0, at, m.unsqueeze(-1) * by.detach().abs()) / (HIDDEN // HEADS) ** 0.5   # noqa: E731
        found = {"bias.weight": torch.zeros_like(p["bias.weight"]).index_add_(0, bucket, m).max()}
        for name, of in (("q", rows(d, k[s])), ("k", rows(s, q[d]))):
            of = of.detach().reshape(x.shape)
            found[f"{name}.bias"], found[f"{name}.weight"] = of.sum(0).max(), (of.t() @ y.detach().abs()).max()
        return {name: float(size) for name, size in found.items()}
    return out, sizes


@pytest.mark.parametrize("rows", [1, 37, 600, 12000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_block_trains(rows, dtype):
    from torchgt_b200 import SparseGraph
    gen = torch.Generator().manual_seed(rows)
    block = _block(dtype)
    edges = torch.cat([torch.randint(0, rows, (2, 5 * rows), generator=gen), torch.arange(rows).repeat(2, 1)], 1).cuda()
    edges = edges[:, edges[1] % 7 != 3].contiguous()                           # rows without edges
    positions = torch.randint(0, 400, (rows,), generator=gen).cuda()
    graph = SparseGraph(edges, rows)
    x, dy = (torch.randn(rows, HIDDEN, generator=gen).to(dtype).cuda() for _ in range(2))
    x.requires_grad_()
    y = _forward(block, x, edges, graph, positions)
    names, leaves = zip(*block.named_parameters())
    grads = torch.autograd.grad(y, (x, *leaves), dy)
    wide = {n: t.detach().double().requires_grad_() for n, t in zip(names, leaves)}
    xd = x.detach().double().requires_grad_()
    yd, sizes = _in_64_bits(wide, xd, edges, positions)
    yd.backward(dy.double())
    sizes = sizes()
    tol = TOL_F32 if dtype == torch.float32 else TOL_BF16
    assert rel_err(y, yd) <= 5 * tol
    for name, got, want in zip(("x",) + names, grads, (xd.grad, *(wide[n].grad for n in names))):
        off = float((got.double() - want).abs().max())
        assert off <= 10 * tol * sizes.get(name, float(want.abs().max())), (name, off)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_serving_rows_equal_the_same_rows_among_others(dtype):
    """The norm and the feed-forward half of one row, of a few and of many: within one rounding of the type of one another; and the
    8-bit rows of the norm in front stand for the same values."""
    from torchgt_b200.rms_norm import rms_norm_quantized
    block = _block(dtype, seed=1)
    x = torch.randn(500, HIDDEN, device="cuda").to(dtype)
    tol = TOL_F32 if dtype == torch.float32 else TOL_BF16
    with torch.no_grad():
        every, total = block["ffn_norm"].add(x, x)
        out = block["ffn"](every, total)
        for n in (1, 3, 16, 17, 40):
            y, s = block["ffn_norm"].add(x[:n], x[:n])
            assert torch.equal(y, every[:n]) and torch.equal(s, total[:n])
            assert rel_err(block["ffn"](y, s), out[:n]) <= tol
        values, scales, s = rms_norm_quantized(x, block["ffn_norm"].weight, EPS, x)
        assert torch.equal(s, total)
        got = values.float() * scales[:, None]
        # half a step of e4m3 is 2^-4 of a value, or 2^-10 of the scale; the value's own rounding is 2^-8 at most
        bound = every.float().abs() * (2.0 ** -4 + 2.0 ** -8) + scales[:, None] * 2.0 ** -10
        assert bool(((got - every.float()).abs() <= bound).all())


def test_a_captured_step_next_to_an_eager_one():
    """A training step of the block in a graph, replayed between eager steps of the same leaves."""
    from torchgt_b200 import SparseGraph
    block = _block(torch.float32, seed=2)
    gen = torch.Generator().manual_seed(5)
    edges, positions = torch.randint(0, 2000, (2, 12000), generator=gen).cuda(), torch.randint(0, 300, (2000,), generator=gen).cuda()
    graph = SparseGraph(edges, 2000, defer_check=False)
    graph.by_src
    x, dy = torch.randn(2000, HIDDEN, generator=gen).cuda(), torch.randn(2000, HIDDEN, generator=gen).cuda()
    leaves = list(block.parameters())
    step = lambda: torch.autograd.grad(_forward(block, x, edges, graph, positions), leaves, dy)   # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        held = step()
    eager = step()
    captured.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, eager, held):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_traced_transformed_and_compiled_calls_are_operations():
    """Under vmap, forward-mode derivatives, torch.func.grad and the tracer the operators are torch's operations, with the same
    values within the types' tolerance."""
    from torchgt_b200 import edge_position_bias, gated_feed_forward
    from torchgt_b200.rms_norm import add_rms_norm
    gen = torch.Generator().manual_seed(9)
    x, r, dx = (torch.randn(4, 30, HIDDEN, generator=gen).cuda() for _ in range(3))
    w = torch.randn(HIDDEN, generator=gen).cuda()
    wg, wu, wd = (torch.randn(HIDDEN, HIDDEN, generator=gen).cuda() / 8 for _ in range(3))
    edges = torch.randint(0, 30, (2, 100), generator=gen).cuda()
    tables = torch.randn(4, 32, HEADS, generator=gen).cuda()
    norm = lambda a, b: add_rms_norm(a, b, w, EPS)[0]                            # noqa: E731
    ffn = lambda a, b: gated_feed_forward(a, wg, wu, wd, "silu", b)              # noqa: E731
    for f in (norm, ffn):
        want = f(x, r)
        assert rel_err(torch.func.vmap(f)(x, r), want) <= TOL_F32
        assert rel_err(torch.jit.trace(f, (x, r))(x, r), want) <= TOL_F32
        value, tangent = torch.func.jvp(f, (x, r), (dx, torch.zeros_like(dx)))
        step = 2.0 ** -7                        # the difference of two fp32 results, each 1e-6 off, over this; third derivatives below 64
        slope = (f(x + step * dx, r).double() - f(x - step * dx, r).double()) / (2 * step)
        assert rel_err(value, want) <= TOL_F32 and rel_err(tangent, slope) <= 1e-6 / step + 64 * step * step
        leaf = x.clone().requires_grad_()
        g, = torch.autograd.grad(f(leaf, r).square().sum(), [leaf])
        assert rel_err(torch.func.grad(lambda a: f(a, r).square().sum())(x), g) <= 5 * TOL_F32
    want = torch.stack([edge_position_bias(t, edges) for t in tables])
    assert torch.equal(torch.func.vmap(lambda t: edge_position_bias(t, edges))(tables), want)
    assert torch.equal(torch.jit.trace(lambda t: edge_position_bias(t, edges), (tables[0],), check_trace=False)(tables[0]), want[0])
    value, tangent = torch.func.jvp(lambda t: edge_position_bias(t, edges), (tables[0],), (tables[1],))
    assert torch.equal(value, want[0]) and torch.equal(tangent, want[1])


def test_two_threads_on_streams_of_their_own():
    """Calls of every operator from two threads at once, each on its stream and with its sizes, give what they give alone."""
    import threading

    from torchgt_b200 import edge_position_bias, gated_feed_forward
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm_quantized

    def work(seed, rows, dtype):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        draw = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)   # noqa: E731
        x, r, dy = draw(rows, 192), draw(rows, 192), draw(rows, 192)
        w, wg, wu, wd = draw(192), draw(256, 192) / 14, draw(256, 192) / 14, draw(192, 256) / 16
        table = torch.randn(32, HEADS, generator=gen, device="cuda", requires_grad=True)
        edges = torch.randint(0, rows, (2, 6 * rows), generator=gen, device="cuda")
        dbias = torch.randn(6 * rows, HEADS, generator=gen, device="cuda")

        def step():
            leaves = [t.detach().requires_grad_() for t in (x, r, w, wg, wu, wd)]
            y, total = add_rms_norm(*leaves[:3], EPS)
            y = gated_feed_forward(y, *leaves[3:], "silu", total)
            with torch.no_grad():
                values, scales, _ = rms_norm_quantized(x, w, EPS, r)
                few = gated_feed_forward(x[:7], wg, wu, wd)
            return [y.detach(), *torch.autograd.grad(y, leaves, dy), values.view(torch.uint8), scales, few,
                    *torch.autograd.grad(edge_position_bias(table, edges), [table], dbias)]
        return step
    steps = [work(1, 1500, torch.bfloat16), work(2, 5000, torch.bfloat16), work(3, 3000, torch.float32)]
    wanted = [step() for step in steps]
    torch.cuda.synchronize()
    wrong = []

    def run(step, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not all(torch.equal(a, b) for a, b in zip(step(), want)):
                    wrong.append(step)
    threads = [threading.Thread(target=run, args=pair) for pair in zip(steps, wanted)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not wrong and not any(t.is_alive() for t in threads)
