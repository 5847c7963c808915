"""GPU test of the server's optimiser step on a network with running
statistics: they take the clients' average, eagerly and in a graph."""
import math

import numpy as np
import pytest

from compressor_b200 import federated as fed
from compressor_b200 import workloads

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("bits", [32, 8])
def test_statistics_are_averaged(product_lib, bits):
    names, shapes = zip(*workloads.manifest("resnet18"))
    layout = fed.AggregateLayout.of(list(names), list(shapes))
    gen = torch.Generator("cuda").manual_seed(2)
    w = torch.rand(layout.total, device="cuda", generator=gen) * 1e-3
    agg = torch.randn(layout.total, device="cuda", generator=gen) * 1e-4
    stat = torch.zeros(layout.total, dtype=torch.bool)
    for n, s, o in zip(names, layout.shapes, layout.offsets):
        stat[o:o + int(np.prod(s))] = "running" in n
    stat = stat.cuda()
    server = fed.ServerAdamW(layout, w, agg, lr=1e-2, max_norm=1e-2, state_bits=bits)
    before = w.clone()
    clip = server.step()
    total = float(agg[~stat].double().square().sum().sqrt())
    assert abs(float(clip[0]) - total) <= 2.0 ** -23 * total
    assert torch.equal(w[stat], before[stat] + agg[stat])
    moved = (w - before)[~stat].abs()
    # a first step moves by about lr whatever the gradient: with 32 bits within a thousandth
    assert float(moved.max()) <= 1.01e-2 and (bits == 8 or float(moved.median()) > 0.99e-2)
    # a statistic that is not finite skips the whole step
    at = int(stat.nonzero()[5])
    kept = float(agg[at])
    agg[at] = math.inf
    before = w.clone()
    assert math.isnan(float(server.step()[1]))
    assert torch.equal(w, before) and int(server.opt.state["step"]) == 1
    agg[at] = kept
    # in a graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        server.step()
    for k in range(2):
        agg.mul_(-0.5)
        before = w.clone()
        graph.replay()
        assert torch.equal(w[stat], before[stat] + agg[stat]) and not torch.equal(w[~stat], before[~stat])
    assert int(server.opt.state["step"]) == 3
