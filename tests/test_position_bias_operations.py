"""The relative position bias as torch's operations (what tracers, compilers and torch.func record) next to its definition in whole
numbers and to the kernels: the same rows of the table, bit by bit."""
import pytest
import torch


def _recorded(table, edges, positions, distance=128, both_ways=True):
    from torchgt_b200.position_bias import _as_operations, bucket_borders
    return _as_operations(table, edges, positions, bucket_borders(table.shape[0], distance, both_ways), both_ways)


def _defined(table, edges, positions, distance=128, both_ways=True):
    """Edge by edge in Python's numbers; NaN for an id outside the positions."""
    from torchgt_b200.position_bias import bucket_borders
    borders = bucket_borders(table.shape[0], distance, both_ways)
    rows = []
    for s, d in edges.t().tolist():
        if positions is not None:
            if not (0 <= s < len(positions) and 0 <= d < len(positions)):
                rows.append(torch.full(table.shape[1:], float("nan")))
                continue
            s, d = int(positions[s]), int(positions[d])
        reach = abs(s - d) if both_ways else max(0, d - s)
        rows.append(table[sum(reach >= b for b in borders) + (len(borders) + 1 if both_ways and s > d else 0)])
    return torch.stack(rows) if rows else table[:0]


def _same(a, b):
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def _list_with_ids_outside():
    gen = torch.Generator().manual_seed(3)
    edges = torch.randint(0, 50, (2, 200), generator=gen)
    edges[0, 7], edges[1, 33], edges[0, 150], edges[1, 151] = 50, -1, 2 ** 40, -2 ** 50
    return edges, torch.randint(0, 300, (50,), generator=gen), torch.randn(32, 8, generator=gen), torch.randn(200, 8, generator=gen)


@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
def test_ids_outside_the_positions_are_nan(ids):
    edges, positions, table, dbias = _list_with_ids_outside()
    if ids == torch.int32:
        edges = edges.clamp(-2 ** 31, 2 ** 31 - 1)
    broken = [7, 33, 150, 151]
    table.requires_grad_()
    got = _recorded(table, edges.to(ids), positions.to(ids))
    assert _same(got.detach(), _defined(table.detach(), edges, positions))
    dbias[broken] = float("nan")                             # of no consequence
    grad, = torch.autograd.grad(got, [table], dbias)
    keep = [e for e in range(200) if e not in broken]
    want, = torch.autograd.grad(_recorded(table, edges[:, keep], positions), [table], dbias[keep])
    torch.testing.assert_close(grad, want)
    nobody = _recorded(table.detach(), edges.to(ids), positions[:0].to(ids))
    assert nobody.shape == (200, 8) and bool(nobody.isnan().all())
    assert _recorded(table.detach(), edges[:, :0], positions[:0]).shape == (0, 8)


@pytest.mark.gpu
def test_ids_outside_the_positions_under_vmap():
    from torchgt_b200 import edge_position_bias
    edges, positions, table, _ = (t.cuda() for t in _list_with_ids_outside())
    want = edge_position_bias(table, edges, positions)
    got = torch.func.vmap(lambda t: edge_position_bias(t, edges, positions))(torch.stack([table, 2 * table]))
    assert _same(got[0], want) and _same(got[1], 2 * want)
    moved = torch.func.vmap(lambda p: edge_position_bias(table, edges, p))(torch.stack([positions, positions.flip(0)]))
    assert _same(moved[0], want) and _same(moved[1], edge_position_bias(table, edges, positions.flip(0)))
    torch.cuda.synchronize()


def _far_places():
    places = [0, 1, -1, 2 ** 40, -2 ** 40, 2 ** 62, -2 ** 62, -2 ** 62 - 1, 2 ** 63 - 1, -2 ** 63, -2 ** 63 + 1]
    n = len(places)
    return torch.cartesian_prod(torch.arange(n), torch.arange(n)).t().contiguous(), torch.tensor(places), torch.arange(32.)[:, None].repeat(1, 2)


@pytest.mark.parametrize("both_ways", [True, False])
def test_positions_at_the_ends_of_64_bits(both_ways):
    """Differences that 64 bits do not hold, and the one whose negative they do not."""
    edges, positions, table = _far_places()
    want = _defined(table, edges, positions, both_ways=both_ways)
    assert torch.equal(_recorded(table, edges, positions, both_ways=both_ways), want)
    assert torch.equal(_recorded(table, positions[edges], None, both_ways=both_ways), want)   # without positions an id is its place


@pytest.mark.gpu
@pytest.mark.parametrize("both_ways", [True, False])
def test_positions_at_the_ends_of_64_bits_in_the_kernels(both_ways):
    from torchgt_b200 import edge_position_bias
    edges, positions, table = _far_places()
    want = _defined(table, edges, positions, both_ways=both_ways)
    for ids, where in ((edges, positions.cuda()), (positions[edges], None)):
        got = edge_position_bias(table.cuda(), ids.cuda(), where, bidirectional=both_ways)
        assert torch.equal(got.cpu(), want)
        wrapped = torch.func.vmap(lambda t: edge_position_bias(t, ids.cuda(), where, bidirectional=both_ways))(table.cuda()[None])   # noqa: B023
        assert torch.equal(wrapped[0].cpu(), want)


def test_a_trace_takes_other_lists_and_positions():
    """Sizes of the traced call are not in the trace: more nodes, more edges, and an id outside the new ones."""
    table = torch.randn(32, 4)
    lists = lambda n, e, seed: (torch.randint(0, n, (2, e), generator=torch.Generator().manual_seed(seed)), torch.arange(n).flip(0) * 3)   # noqa: E731
    traced = torch.jit.trace(_recorded, (table, *lists(50, 200, 1)), check_trace=False)
    edges, positions = lists(80, 301, 2)
    edges[0, 3], edges[1, 9] = 80, -1
    assert _same(traced(table, edges, positions), _defined(table, edges, positions))
