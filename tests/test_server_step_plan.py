"""What federated.ServerAdamW hands to the optimiser: slices, decays, scale
and refusals, on the CPU with a stand-in for the GPU operators."""
import pytest

from compressor_b200 import federated as fed

torch = pytest.importorskip("torch")


@pytest.fixture
def seen(monkeypatch):
    from compressor_b200 import optim
    calls = {}

    class Norm:
        def __init__(self, tensors, lib_path=None):
            calls["norm"] = tensors

        def __call__(self, **kw):
            calls["norm_call"] = kw
            return "clip"

    class Adam:
        def __init__(self, params, grads, **kw):
            calls["params"], calls["grads"], calls["kw"] = params, grads, kw

        def step(self, **kw):
            calls["step"] = kw

    monkeypatch.setattr(optim, "GradNorm", Norm)
    monkeypatch.setattr(optim, "AdamW", Adam)
    return calls


LAYOUT = fed.AggregateLayout.of(["w", "b", "u"], [(4, 3), (5,), (2, 2)], align=8)


def test_slices_decay_and_scale(seen):
    w, a = torch.arange(30.0), torch.arange(30.0) + 100
    s = fed.ServerAdamW(LAYOUT, w, a, lr=0.5, weight_decay=0.1, max_norm=2.0, state_bits=8, seed=3)
    assert [p.tolist() for p in seen["params"]] == [list(range(0, 12)), list(range(16, 21)), list(range(24, 28))]
    assert all(g[0] == p[0] + 100 and g.numel() == p.numel() for p, g in zip(seen["params"], seen["grads"]))
    assert all(p.data_ptr() == w[int(p[0]):].data_ptr() for p in seen["params"])      # views, not copies
    assert seen["kw"]["weight_decay"] == [0.1, 0.0, 0.1]
    assert seen["kw"]["lr"] == 0.5 and seen["kw"]["state_bits"] == 8 and seen["kw"]["seed"] == 3
    assert s.step(lr=0.25) == "clip"
    assert seen["norm_call"] == {"max_norm": 2.0, "grad_scale": -1.0}
    assert seen["step"] == {"lr": 0.25, "grad_scale": -1.0, "clip": "clip"}


def test_names_decays_and_no_clipping(seen):
    s = fed.ServerAdamW(LAYOUT, torch.zeros(28), torch.zeros(28), weight_decay=0.1, names=["u", "b"],
                        decays=lambda n, shape: n == "b", grad_scale=1.0)
    assert s.names == ["b", "u"] and seen["kw"]["weight_decay"] == [0.1, 0.0]
    assert "norm" not in seen and s.step() is None and seen["step"]["grad_scale"] == 1.0


def test_refusals(seen):
    ok = torch.zeros(28)
    for w, a in [(torch.zeros(27), ok), (ok, torch.zeros(27)), (ok.view(4, 7), ok), (ok, torch.zeros(56)[::2])]:
        with pytest.raises(ValueError):
            fed.ServerAdamW(LAYOUT, w, a)
    with pytest.raises(ValueError):
        fed.ServerAdamW(LAYOUT, ok, ok.clone(), names=["w", "x"])
