"""The relative position bias of edges and the gradient of its table.  A row of bias is a copy of a table row, so it is equal
bit by bit; a sum of the gradient is at most a few hundred terms in a lane, and as many steps over lanes, warps and CTAs, for
the lists here: below 512 * 2^-24 of the sum of the magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SUM = 512 * 2.0 ** -24


def _bucket(offset, borders, both_ways):
    """Counted border by border."""
    distance = offset.abs() if both_ways else (-offset).clamp(min=0)
    bucket = sum((distance >= b).long() for b in borders) if len(borders) else torch.zeros_like(offset)
    return bucket + (offset > 0).long() * (len(borders) + 1) if both_ways else bucket


def _check(table, edges, positions, distance, both_ways, dbias):
    from torchgt_b200.position_bias import bucket_borders, edge_position_bias
    borders = bucket_borders(table.shape[0], distance, both_ways)
    leaf = table.detach().requires_grad_()
    bias = edge_position_bias(leaf, edges, positions, distance, both_ways)
    where = (positions if positions is not None else torch.arange(int(edges.max()) + 1 if edges.numel() else 1)).long().cpu()
    ends = where[edges.long().cpu()]
    bucket = _bucket(ends[0] - ends[1], borders, both_ways)
    assert torch.equal(bias.detach().cpu(), table.detach().cpu()[bucket])
    grad, = torch.autograd.grad(bias, [leaf], dbias)
    d = dbias.double().cpu()
    want = torch.zeros(table.shape, dtype=torch.float64).index_add_(0, bucket, d)
    size = torch.zeros(table.shape, dtype=torch.float64).index_add_(0, bucket, d.abs())
    off = (grad.double().cpu() - want).abs()
    assert bool((off <= SUM * size).all()), float((off / (SUM * size + 1e-300)).max())
    return bias, grad


CASES = [(1, 1, 32, 128, True), (31, 8, 32, 128, True), (33, 8, 32, 128, False), (5000, 1, 32, 128, True), (5000, 2, 16, 64, False),
         (4097, 3, 10, 50, True), (4097, 4, 64, 1000, True), (20000, 8, 32, 128, True), (3001, 12, 2, 2, False),
         (3000, 16, 4, 2, True), (2500, 32, 512, 100000, True), (2500, 40, 511, 1000, False), (999, 256, 128, 4096, True),
         (200000, 8, 32, 128, True), (777, 6, 3, 9, False)]


@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
@pytest.mark.parametrize("edges,heads,buckets,distance,both_ways", CASES)
def test_bias_and_gradient(edges, heads, buckets, distance, both_ways, ids):
    gen = torch.Generator().manual_seed(edges + heads)
    nodes = max(1, edges // 4)
    list_ = torch.randint(0, nodes, (2, edges), generator=gen)
    list_[:, : edges // 10] = 0                                    # many edges of one bucket
    table, dbias = torch.randn(buckets, heads, generator=gen).cuda(), torch.randn(edges, heads, generator=gen).cuda()
    _check(table, list_.to(ids).cuda(), None, distance, both_ways, dbias)
    positions = torch.randint(-2 * distance, 2 * distance, (nodes,), generator=gen)
    for kind in (torch.int64, torch.int32):
        _check(table, list_.to(ids).cuda(), positions.to(kind).cuda(), distance, both_ways, dbias)


@pytest.mark.parametrize("heads,buckets,ids,places", [(4, 128, torch.int64, torch.int64), (8, 64, torch.int64, torch.int32), (8, 4, torch.int32, torch.int64),
                                                      (16, 33, torch.int32, torch.int32), (8, 130, torch.int64, torch.int64)])
def test_many_edges(heads, buckets, ids, places):
    """Lists long enough for the table in shared memory, odd ones, with and without positions, some ids outside them."""
    from torchgt_b200.position_bias import bucket_borders, edge_position_bias
    gen = torch.Generator().manual_seed(heads * buckets)
    edges, nodes, both = 1310003 + heads, 5000, buckets % 2 == 0
    list_ = torch.randint(0, nodes, (2, edges), generator=gen)
    positions = torch.randint(-300, 300, (nodes,), generator=gen)
    table = torch.randn(buckets, heads, generator=gen)
    borders = bucket_borders(buckets, 200, both)
    for where in (None, positions):
        ends = list_ if where is None else where[list_]
        want = table[_bucket(ends[0] - ends[1], borders, both)]
        got = edge_position_bias(table.cuda(), list_.to(ids).cuda(), None if where is None else where.to(places).cuda(), 200, both)
        assert torch.equal(got.cpu(), want)
    wrong = list_.clone()
    wrong[0, 7], wrong[1, edges - 1], wrong[1, edges // 2] = -1, nodes, nodes + 100
    got = edge_position_bias(table.cuda(), wrong.to(ids).cuda(), positions.to(places).cuda(), 200, both).cpu()
    bad = torch.zeros(edges, dtype=torch.bool)
    bad[[7, edges - 1, edges // 2]] = True
    assert torch.equal(got[~bad], want[~bad]) and bool(got[bad].isnan().all())


def test_every_border_is_met_exactly():
    """Distances around every border, with one node at each place."""
    from torchgt_b200.position_bias import bucket_borders
    for buckets, distance, both_ways in ((32, 128, True), (32, 128, False), (64, 100000, True), (512, 2 ** 31 - 1, False)):
        borders = bucket_borders(buckets, distance, both_ways)
        at = sorted({max(0, b + k) for b in borders for k in (-1, 0, 1)})
        positions = torch.tensor([0] + at + [2 ** 40, -2 ** 62, 2 ** 63 - 1, -2 ** 63])
        n = len(positions)
        there = torch.stack([torch.arange(n - 4), torch.zeros(n - 4, dtype=torch.long)])
        edges = torch.cat([there, there.flip(0)], 1)
        table = torch.arange(buckets, dtype=torch.float32)[:, None].repeat(1, 4).cuda()
        _check(table, edges.cuda(), positions.cuda(), distance, both_ways, torch.ones(edges.shape[1], 4).cuda())
        # far beyond the last border, up to the ends of 64 bits
        from torchgt_b200.position_bias import edge_position_bias
        far = torch.tensor([[n - 4, n - 3, n - 2, n - 1, 0, n - 2], [0, 0, 0, 0, n - 4, n - 1]])
        got = edge_position_bias(table, far.cuda(), positions.cuda(), distance, both_ways)[:, 0].long().tolist()
        last, half = len(borders), len(borders) + 1
        assert got == ([half + last, last, half + last, last, last, half + last] if both_ways else [0, last, 0, last, last, 0])


def test_ids_outside_the_positions_are_nan_and_leave_the_rest():
    from torchgt_b200.position_bias import edge_position_bias
    gen = torch.Generator().manual_seed(3)
    edges = torch.randint(0, 50, (2, 200), generator=gen)
    table = torch.randn(32, 8, generator=gen).cuda().requires_grad_()
    positions = torch.randint(0, 300, (50,), generator=gen).cuda()
    want = edge_position_bias(table, edges.cuda(), positions)
    bad = edges.clone()
    bad[0, 7], bad[1, 33], bad[0, 150], bad[1, 151] = 50, -1, 2 ** 40, -2 ** 50
    broken = [7, 33, 150, 151]
    fine = [e for e in range(200) if e not in broken]
    got = edge_position_bias(table, bad.cuda(), positions)
    assert bool(got[broken].isnan().all()) and torch.equal(got[fine], want[fine])
    dbias = torch.randn(200, 8, generator=gen).cuda()
    dbias[broken] = float("nan")
    grad, = torch.autograd.grad(got, [table], dbias)
    zeroed = dbias.clone()
    zeroed[broken] = 0
    assert torch.equal(grad, torch.autograd.grad(want, [table], zeroed)[0])
    nobody = edge_position_bias(table, edges.cuda(), positions[:0])
    assert bool(nobody.isnan().all())


def test_no_edges_and_strided_lists():
    from torchgt_b200.position_bias import edge_position_bias
    table = torch.randn(32, 8, device="cuda", requires_grad=True)
    bias = edge_position_bias(table, torch.zeros(2, 0, dtype=torch.long, device="cuda"))
    assert bias.shape == (0, 8)
    grad, = torch.autograd.grad(bias, [table], torch.zeros(0, 8, device="cuda"))
    assert torch.equal(grad, torch.zeros_like(table))
    pairs = torch.randint(0, 500, (1000, 2), device="cuda")
    wide = torch.randn(32, 20, device="cuda")
    got = edge_position_bias(wide[:, 3:11], pairs.t())
    assert torch.equal(got, edge_position_bias(wide[:, 3:11].contiguous(), pairs.t().contiguous()))
    assert torch.equal(edge_position_bias(wide.t()[:8].t(), pairs.t()), edge_position_bias(wide[:, :8].contiguous(), pairs.t()))
    off = torch.zeros(32 * 8 + 1, device="cuda")
    off[1:] = wide[:, :8].flatten()
    assert torch.equal(edge_position_bias(off[1:].view(32, 8), pairs.t()), edge_position_bias(wide[:, :8].contiguous(), pairs.t()))
    expanded = torch.ones(1, 8, device="cuda").expand(1000, 8)
    table = wide[:, :8].contiguous().requires_grad_()
    grad, = torch.autograd.grad(edge_position_bias(table, pairs.t()), [table], expanded)
    assert float(grad.sum()) == 8000.0


def test_same_bits_on_other_streams_from_a_graph_and_second_order():
    from torchgt_b200.position_bias import edge_position_bias
    edges = torch.randint(0, 5000, (2, 60000), device="cuda")
    positions = torch.randperm(5000, device="cuda")
    table, dbias = torch.randn(32, 8, device="cuda"), torch.randn(60000, 8, device="cuda")
    def step():
        leaf = table.detach().requires_grad_()
        bias = edge_position_bias(leaf, edges, positions)
        return bias.detach(), torch.autograd.grad(bias, [leaf], dbias)[0]
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    positions.copy_(positions.flip(0))
    graph.replay()
    assert torch.equal(captured[0], step()[0])
    positions.copy_(positions.flip(0))
    graph.replay()
    for a, b, c in zip(want, other, captured):
        assert torch.equal(a, b) and torch.equal(a, c)
    leaf = table.detach().requires_grad_()
    d = dbias.detach().requires_grad_()
    grad, = torch.autograd.grad(edge_position_bias(leaf, edges, positions), [leaf], d, create_graph=True)
    back, = torch.autograd.grad(grad, [d], table)
    assert torch.equal(back, edge_position_bias(table, edges, positions))
    many, = torch.autograd.grad(edge_position_bias(leaf, edges, positions), [leaf], torch.stack([dbias, 2 * dbias]),
                                is_grads_batched=True)
    assert many.shape == (2, 32, 8)
    torch.testing.assert_close(many[0], want[1], rtol=1e-4, atol=1e-3)


def test_module_feeds_the_attention_and_learns():
    """Bias, attention and back: the table's gradient against the attention's own gradient of a per-edge bias."""
    from torchgt_b200 import RelativePositionBias, SparseGraph, sparse_graph_attention
    gen = torch.Generator().manual_seed(5)
    n, heads = 300, 8
    edges = torch.randint(0, n, (2, 2400), generator=gen).cuda()
    graph = SparseGraph(edges, n)
    module = RelativePositionBias(heads, 32, 128).cuda()
    assert list(module.state_dict()) == ["weight"]
    q, k, v, dout = (torch.randn(n, heads, 8, generator=gen).cuda() for _ in range(4))
    bias = module(edges)
    loose = bias.detach().requires_grad_()
    out = sparse_graph_attention(q, k, v, graph, bias)
    out.backward(dout)
    dbias, = torch.autograd.grad(sparse_graph_attention(q, k, v, graph, loose), [loose], dout)
    again, = torch.autograd.grad(module(edges), [module.weight], dbias)
    assert torch.equal(module.weight.grad, again)
