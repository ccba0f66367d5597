"""The relative position bias under autocast: its table is fp32 and its ids are whole numbers, so it is the kernels there as well."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast_runs_the_kernels(dtype):
    from torchgt_b200 import RelativePositionBias
    gen = torch.Generator().manual_seed(1)
    edges, positions = torch.randint(0, 500, (2, 5001), generator=gen).cuda(), torch.randint(0, 400, (500,), generator=gen).cuda()
    edges[0, 5], edges[1, 9] = -1, 500                       # outside the positions
    module, dbias = RelativePositionBias(8).cuda(), torch.randn(5001, 8, generator=gen).cuda()

    def step(autocast):
        with torch.autocast("cuda", dtype=dtype, enabled=autocast):
            bias = module(edges, positions)
        grad, = torch.autograd.grad(bias, [module.weight], dbias)
        return bias.detach(), grad, bias.grad_fn.name()      # no eager graph of the weight lives when a step is captured
    want, want_grad, node = step(False)
    assert bool(want[5].isnan().all()) and bool(want[9].isnan().all())
    bias, grad, name = step(True)
    assert bias.dtype == torch.float32 and name == node
    assert torch.equal(bias.nan_to_num(), want.nan_to_num()) and torch.equal(grad, want_grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, held_grad, _ = step(True)
    graph.replay()
    assert torch.equal(held.nan_to_num(), want.nan_to_num()) and torch.equal(held_grad, want_grad)
