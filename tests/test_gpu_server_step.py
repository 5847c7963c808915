"""GPU test of whole federated rounds with a server optimiser: clients'
updates compressed and decoded into the weighted aggregate by the codec, the
aggregate's norm clipped, an AdamW step on the global weights
(federated.ServerAdamW), several rounds, against the same AdamW in float64 on
the aggregates that came out."""
import ctypes
import math

import numpy as np
import pytest

from compressor_b200 import federated as fed
from compressor_b200.abi import Codec
from tests.helpers import seeded

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SHAPES = [("l1.conv.weight", (64, 32, 3, 3)), ("l1.bn.weight", (64,)), ("l1.bn.bias", (65,)),
          ("l2.conv.weight", (130, 64, 1, 1)), ("fc.weight", (10, 513)), ("fc.bias", (10,))]
LR, WD, MAX_NORM = 1e-2, 0.1, 0.05


def _round(encs, server, agg, layout, t):
    names = [n for n, _ in SHAPES]
    w = fed.uniform_weights(len(encs))
    for c, enc in enumerate(encs):
        xs = [seeded(s, 1000 * c + 10 * t + i) for i, (_, s) in enumerate(SHAPES)]
        ret, layers, errs = enc.compress_batch(names, xs)
        assert ret == 0, errs
        fed.set_client_weight(server.lib, server.h, agg.data_ptr(), layout.c_offsets(), len(names), w[c])
        fed.set_aggregate_store(server.lib, server.h, c == 0)
        assert server.decompress_batch(names, layers, client=f"c{c}")[0] == 0
    fed.allreduce_aggregate(agg)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("align", [1, 64])
def test_rounds_with_server_adamw(product_lib, bits, align):
    layout = fed.AggregateLayout.of([n for n, _ in SHAPES], [s for _, s in SHAPES], align=align)
    encs = [Codec(product_lib, client=f"c{c}", param_count_threshold=16) for c in range(2)]
    server = Codec(product_lib, client="server", param_count_threshold=16)
    gen = torch.Generator("cuda").manual_seed(0)
    weights = [torch.randn(layout.total, device="cuda", generator=gen) * 0.05]
    weights.append(weights[0].clone())
    agg = torch.zeros(layout.total, device="cuda")
    steps = [fed.ServerAdamW(layout, w, agg, lr=LR, weight_decay=WD, state_bits=bits, max_norm=MAX_NORM)
             for w in weights]
    start = weights[0].clone()
    spans = [(o, o + int(np.prod(s)), len(s) > 1) for o, (_, s) in zip(layout.offsets, SHAPES)]
    p = start.double().cpu().numpy()
    m, v = np.zeros_like(p), np.zeros_like(p)
    for t in range(1, 5):
        _round(encs, server, agg, layout, t)
        clips = [s.step() for s in steps]
        a = agg.double().cpu().numpy()
        norm = math.sqrt(sum(float((a[b:e] ** 2).sum()) for b, e, _ in spans))
        assert norm > MAX_NORM                       # the clipping is exercised
        got = clips[0].cpu().numpy()
        assert abs(got[0] - norm) <= 2.0 ** -23 * norm and abs(got[1] - MAX_NORM / norm) <= 2.0 ** -23
        for b, e, decays in spans:
            g = -a[b:e] * (MAX_NORM / norm)
            m[b:e] = 0.9 * m[b:e] + 0.1 * g
            v[b:e] = 0.999 * v[b:e] + 0.001 * g * g
            p[b:e] *= 1 - LR * WD * decays
            p[b:e] -= LR * (m[b:e] / (1 - 0.9 ** t)) / (np.sqrt(v[b:e] / (1 - 0.999 ** t)) + 1e-8)
    torch.cuda.synchronize()
    assert torch.equal(weights[0], weights[1])       # equal copies stay equal, bit for bit
    moved = np.linalg.norm(p - start.double().cpu().numpy())
    off = np.linalg.norm(weights[0].double().cpu().numpy() - p)
    # 32 bits: four roundings of the weights and a few of each update; 8 bits:
    # a stored moment is off by an eighth at most, an update by about as much
    assert off <= (4 * 2.0 ** -24 * math.sqrt(layout.total) + 1e-5 * moved if bits == 32 else 0.13 * moved), (off, moved)
    inside = np.zeros(layout.total, bool)
    for b, e, _ in spans:
        inside[b:e] = True
    assert torch.equal(weights[0][torch.from_numpy(~inside)], start[torch.from_numpy(~inside)])   # padding stays
    for s in steps:
        s.close()
    for c in encs + [server]:
        c.close()


def test_non_finite_round_is_skipped(product_lib):
    layout = fed.AggregateLayout.of(["a", "b"], [(100, 7), (31,)])
    w = torch.randn(layout.total, device="cuda")
    agg = torch.randn(layout.total, device="cuda")
    s = fed.ServerAdamW(layout, w, agg, max_norm=1.0, names=["a"])
    agg[720] = math.nan                              # in "b", which takes no part
    before = w.clone()
    s.step()
    assert not torch.equal(w[:700], before[:700]) and torch.equal(w[700:], before[700:])
    agg[3] = math.inf
    before = w.clone()
    assert torch.isnan(s.step()[1])
    assert torch.equal(w, before) and int(s.opt.state["step"]) == 1
    s.close()
