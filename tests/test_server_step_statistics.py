"""Running statistics in the server's optimiser step: averaged, not stepped
on.  On the CPU with a stand-in for the GPU operators."""
import math

import pytest

from compressor_b200 import federated as fed
from compressor_b200 import workloads

torch = pytest.importorskip("torch")

LAYOUT = fed.AggregateLayout.of(["conv.weight", "bn.weight", "bn.running_mean", "bn.running_var", "fc.bias"],
                                [(4, 3), (4,), (4,), (4,), (2,)], align=8)
PLACES = list(zip(LAYOUT.names, LAYOUT.offsets, LAYOUT.shapes))


@pytest.fixture
def seen(monkeypatch):
    from compressor_b200 import optim
    calls = {"coefficient": 0.5}

    class Norm:
        def __init__(self, tensors, lib_path=None):
            calls["norm"] = tensors

        def __call__(self, **kw):
            return torch.tensor([2.0, calls["coefficient"]])

    class Adam:
        def __init__(self, params, grads, **kw):
            calls["params"], calls["grads"], calls["kw"] = params, grads, kw

        def step(self, **kw):
            calls["step"] = kw

    monkeypatch.setattr(optim, "GradNorm", Norm)
    monkeypatch.setattr(optim, "AdamW", Adam)
    return calls


def _flat():
    gen = torch.Generator().manual_seed(1)
    return torch.randn(LAYOUT.total, generator=gen), torch.randn(LAYOUT.total, generator=gen)


def test_statistics_get_the_aggregate_and_nothing_else(seen):
    w, a = _flat()
    before = w.clone()
    s = fed.ServerAdamW(LAYOUT, w, a, weight_decay=0.1, max_norm=1.0)
    assert s.names == ["conv.weight", "bn.weight", "fc.bias"] and s.averaged == ["bn.running_mean", "bn.running_var"]
    stepped = [LAYOUT.offsets[i] for i in (0, 1, 4)]
    assert [p.data_ptr() for p in seen["params"]] == [w[o:].data_ptr() for o in stepped]
    assert [g.data_ptr() for g in seen["norm"]] == [a[o:].data_ptr() for o in stepped]    # nor do they clip
    assert seen["kw"]["weight_decay"] == [0.1, 0.0, 0.0]
    clip = s.step()
    assert clip.tolist() == [2.0, 0.5] and seen["step"]["clip"].tolist() == [2.0, 0.5]
    inside = torch.zeros(LAYOUT.total, dtype=torch.bool)
    for name, o, shape in PLACES:
        if "running" in name:
            inside[o:o + math.prod(shape)] = True
    assert torch.equal(w[inside], before[inside] + a[inside]) and torch.equal(w[~inside], before[~inside])


@pytest.mark.parametrize("grad_scale", [-0.25, 1.0])
def test_statistics_follow_the_sign_and_the_scale(seen, grad_scale):
    w, a = _flat()
    before = w.clone()
    s = fed.ServerAdamW(LAYOUT, w, a, grad_scale=grad_scale)
    assert s.step() is None
    o = LAYOUT.offsets[3]
    assert torch.allclose(w[o:o + 4], before[o:o + 4] - grad_scale * a[o:o + 4], rtol=0, atol=2.0 ** -21)


@pytest.mark.parametrize("where", ["weights", "statistics"])
def test_a_round_that_is_not_finite_is_skipped_whole(seen, where):
    w, a = _flat()
    before = w.clone()
    s = fed.ServerAdamW(LAYOUT, w, a, max_norm=1.0)
    if where == "weights":
        seen["coefficient"] = math.nan
    else:
        a[LAYOUT.offsets[2] + 1] = math.inf
    assert math.isnan(s.step()[1]) and math.isnan(seen["step"]["clip"][1])
    assert torch.equal(w, before)


def test_names_and_a_choice_of_ones_own(seen):
    w, a = _flat()
    s = fed.ServerAdamW(LAYOUT, w, a, names=["conv.weight", "bn.running_var"])
    assert s.names == ["conv.weight"] and s.averaged == ["bn.running_var"]
    s = fed.ServerAdamW(LAYOUT, w, a, averaged=lambda name, shape: name == "fc.bias")
    assert s.averaged == ["fc.bias"] and "bn.running_var" in s.names
    before = w.clone()
    s.step()
    assert torch.equal(w[-2:], before[-2:] + a[-2:]) and torch.equal(w[:-2], before[:-2])


@pytest.mark.parametrize("model,count", [("resnet18", 40), ("resnet50", 106)])
def test_the_models_statistics_are_found(seen, model, count):
    names, shapes = zip(*workloads.manifest(model))
    layout = fed.AggregateLayout.of(list(names), list(shapes))
    s = fed.ServerAdamW(layout, torch.zeros(layout.total), torch.zeros(layout.total))
    assert len(s.averaged) == count and not any("running" in n for n in s.names)
    assert len(s.names) + count == len(names)


def test_errors_of_the_step_are_reported(seen):
    w, a = _flat()
    s = fed.ServerAdamW(LAYOUT, w, a)
    s.opt.errors = lambda: 1
    assert s.errors() == 1


def test_a_refused_step_leaves_the_statistics(seen):
    w, a = _flat()
    before = w.clone()
    s = fed.ServerAdamW(LAYOUT, w, a, max_norm=1.0)

    def refuse(**kw):
        raise ValueError("lr")

    s.opt.step = refuse
    with pytest.raises(ValueError):
        s.step(lr=-1.0)
    assert torch.equal(w, before)
