"""AdamW.state: the plan writes these tensors' memory, so nothing else takes
their place (on the CPU, without a plan)."""
import copy
import io

import pytest

torch = pytest.importorskip("torch")


def test_states_are_loaded_not_assigned():
    from compressor_b200 import optim
    o = object.__new__(optim.AdamW)
    o._h = None
    o._state = {"m": torch.zeros(3), "v": torch.zeros(3), "step": torch.zeros(1, dtype=torch.int64)}
    first = dict(o._state)
    with pytest.raises(AttributeError):
        o.state = {k: t.clone() for k, t in o.state.items()}
    o.state["m"] = torch.ones(3)
    del o.state["v"]
    assert o.state.keys() == first.keys() and all(o.state[k] is t for k, t in first.items())
    o.state["v"].fill_(2.0)                        # in place is what counts
    assert o.state["v"].tolist() == [2.0] * 3
    file = io.BytesIO()
    torch.save(o.state, file)
    file.seek(0)
    assert torch.load(file)["v"].tolist() == [2.0] * 3
    assert copy.deepcopy(o.state)["v"] is not o.state["v"]
    saved = {**o.state, "m": torch.ones(3), "step": torch.full((1,), 7)}
    o.load_state(saved)
    assert o.state["m"].tolist() == [1.0] * 3 and int(o.state["step"]) == 7 and o.state["m"] is not saved["m"]
    with pytest.raises(ValueError):
        o.load_state({"m": torch.ones(3)})
