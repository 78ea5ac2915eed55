"""GPU: a step through a compressed layer, forward and backward, captured into a graph and replayed with other values and
eager work between."""
import pytest
import torch

import neuzip_amd
from neuzip_amd import nn

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("m,n,k", [(64, 96, 200), (2048, 4096, 512), (4096, 1024, 256), (9001, 1001, 64)])
def test_a_captured_step_of_a_compressed_layer(m, n, k, bits):
    """Whole numbers: the gradient of the bias is exact in any order.  A library's sum over many rows clears its counters
    with a node that replays do not keep to."""
    dtype = torch.bfloat16
    layer = nn.Linear(neuzip_amd.Manager(precision=7), torch.nn.Linear(k, n).to(dtype).to(DEV))
    layer.saved_bits = bits
    x = torch.randn(m, k, device=DEV).to(dtype)
    g = torch.zeros(m, n, dtype=dtype, device=DEV)

    def step():
        layer.weight._gradient = None
        a = x.detach().requires_grad_(True)
        y = layer(a)
        dx, db = torch.autograd.grad(y, (a, layer.bias), g)
        return y.detach(), dx, db, layer.weight._gradient

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        gen = torch.Generator(device=DEV).manual_seed(turn)
        x.copy_(torch.randn(m, k, device=DEV, generator=gen))
        g.copy_(torch.randint(-3, 4, (m, n), device=DEV, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(out[2], g.double().sum(0).to(torch.float32).to(dtype)), turn
        for a, b in zip(out, want):
            assert torch.equal(a, b), turn
