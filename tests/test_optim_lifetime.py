"""What captured graphs use stays in place while they live: the plans' tables
(C entry points, through the kernel emulator) and what the torch classes own
(with a stand-in for the library)."""
import ctypes

import numpy as np
import pytest

from compressor_b200 import abi
from tests import optim_cases as oc
from tests.test_optim_emulation import _norm_create, emu  # noqa: F401


@pytest.fixture
def lib(emu):  # noqa: F811
    lib = emu.lib
    lib.emu_device_count.restype = ctypes.c_size_t
    yield lib
    lib.emu_optim_capture(0)
    lib.emu_optim_graph_gone()


def _norm_plan(emu, x, capture):  # noqa: F811
    plan = _norm_create(emu.lib, [x.ptr], [x.n], [0])
    work = oc.Placed(emu, np.zeros(emu.lib.falcom_norm_work_bytes(plan), np.uint8))
    out = oc.Placed(emu, np.zeros(2, np.float32))
    emu.lib.emu_optim_capture(capture)
    for _ in range(2):
        assert emu.lib.falcom_norm_run(plan, 1.0, 1.0, out.ptr, work.ptr, None) == 0
    emu.lib.emu_optim_capture(0)
    return plan, emu.lib.falcom_norm_destroy


def _adamw_plan(emu, x, capture):  # noqa: F811
    step = oc.Placed(emu, np.zeros(1, np.int64))
    t = oc.Tensor(emu, np.random.default_rng(0), 700, "f32", "f32", 8, 0.1)
    plan = emu.lib.falcom_adamw_create(oc.c_array(abi.AdamWTensorC, [t.c()]), 1, 8, step.ptr)
    emu.lib.emu_optim_capture(capture)
    assert emu.lib.falcom_adamw_step(plan, ctypes.byref(oc.make_args()), None) == 0
    emu.lib.emu_optim_capture(0)
    return plan, emu.lib.falcom_adamw_destroy


@pytest.mark.parametrize("make", [_norm_plan, _adamw_plan])
def test_a_graphs_plan_outlives_destroy(emu, lib, make):  # noqa: F811
    x = oc.Placed(emu, np.ones(5000, np.float32))
    base = lib.emu_device_count()
    plan, destroy = make(emu, x, 0)
    destroy(plan)
    assert lib.emu_device_count() == base
    plan, destroy = make(emu, x, 1)
    destroy(plan)
    assert lib.emu_device_count() == base + 1      # the table that the graph reads
    other, _ = make(emu, x, 0)
    destroy(other)
    assert lib.emu_device_count() == base + 1
    lib.emu_optim_graph_gone()
    other, _ = make(emu, x, 0)                     # later plans free what no graph uses any longer
    destroy(other)
    assert lib.emu_device_count() == base


def test_graphs_are_counted(emu, lib):  # noqa: F811
    x = oc.Placed(emu, np.ones(5000, np.float32))
    plan, destroy = _norm_plan(emu, x, 1)
    assert lib.falcom_norm_graphs(plan) == 2       # one use for each captured call
    lib.emu_optim_graph_gone()
    assert lib.falcom_norm_graphs(plan) == 0 and lib.falcom_norm_graphs(None) == 0
    destroy(plan)
    plan, destroy = _adamw_plan(emu, x, 1)
    assert lib.falcom_adamw_graphs(plan) == 1 and lib.falcom_adamw_graphs(None) == 0
    lib.emu_optim_graph_gone()
    assert lib.falcom_adamw_graphs(plan) == 0
    destroy(plan)


class FakeLibrary:
    def __init__(self):
        self.graphs, self.destroyed = {}, []

    def falcom_norm_graphs(self, h):
        return self.graphs.get(h, 0)

    falcom_adamw_graphs = falcom_norm_graphs

    def falcom_norm_destroy(self, h):
        self.destroyed.append(h)

    falcom_adamw_destroy = falcom_norm_destroy


@pytest.mark.parametrize("kind", ["GradNorm", "AdamW"])
@pytest.mark.parametrize("how", ["close", "del"])
def test_classes_leave_graphs_their_memory(kind, how):
    torch = pytest.importorskip("torch")
    import weakref
    from compressor_b200 import optim

    def make(h):
        o = object.__new__(getattr(optim, kind))
        o._h, o.lib = h, lib
        o._held = [torch.zeros(1)]
        o._work, o._captured, o._state = {}, [torch.zeros(1)], {"m": torch.zeros(1)}
        return o, [weakref.ref(t) for t in (o._held[0], o._captured[0] if kind == "GradNorm" else o._state["m"])]

    def drop(o):
        if how == "close":
            o.close()
            with pytest.raises(RuntimeError, match="closed"):
                o() if kind == "GradNorm" else o.step()

    lib = FakeLibrary()
    o, memory = make(1)
    drop(o)
    del o
    assert lib.destroyed == [1] and not any(r() is not None for r in memory)
    lib.graphs[2] = 1
    o, memory = make(2)
    drop(o)
    del o
    o, _ = make(3)
    drop(o)
    del o
    assert lib.destroyed == [1, 3] and all(r() is not None for r in memory)
    lib.graphs[2] = 0
    o, _ = make(4)
    drop(o)
    del o
    assert sorted(lib.destroyed) == [1, 2, 3, 4] and not any(r() is not None for r in memory)
