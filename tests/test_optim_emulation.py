"""The optimiser kernels (mc_optim.cu) and their host side on the CPU, through
the kernel emulator, against plain 64-bit formulas (tests/optim_cases.py):
indexing, short blocks, misaligned arrays, mixed types, the 8-bit states'
rounding, refusals.  tests/test_gpu_optim.py runs the same checks on a GPU."""
import ctypes
import math

import numpy as np
import pytest

from compressor_b200 import abi
from tests import optim_cases as oc


class Emu:
    stream = None

    class Mem:
        def __init__(self, lib, raw):
            self.lib, self.size = lib, raw.size
            self.ptr = lib.emu_device_alloc(raw.size)
            ctypes.memmove(self.ptr, raw.ctypes.data, raw.size)

        def __del__(self):
            self.lib.emu_device_free(self.ptr)

    def __init__(self, path):
        self.lib = ctypes.CDLL(path)
        abi.bind_optim(self.lib)
        self.lib.emu_device_alloc.argtypes = [ctypes.c_size_t]
        self.lib.emu_device_alloc.restype = ctypes.c_void_p
        self.lib.emu_device_free.argtypes = [ctypes.c_void_p]
        self.lib.emu_device_free.restype = None

    def upload(self, raw):
        return Emu.Mem(self.lib, raw)

    def download(self, h):
        return np.frombuffer(ctypes.string_at(h.ptr, h.size), np.uint8)

    def sync(self):
        pass


@pytest.fixture(scope="module")
def emu():
    from tests.emu import build_optim
    return Emu(build_optim.build())


@pytest.mark.parametrize("name", list(oc.NORM_CASES))
def test_norm(emu, name):
    ns, kinds, shifts = oc.NORM_CASES[name]
    rng = np.random.default_rng(1)
    xs = [rng.standard_normal(n) * 10.0 ** rng.integers(-4, 2) for n in ns]
    oc.check_norm(emu, xs, kinds, shifts, scale=-0.5, max_norm=0.75)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pk,gk", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "f16")])
def test_adamw_types(emu, bits, pk, gk):
    oc.run_adamw(emu, oc.case_tensors(emu, "odd", bits, pk, gk), bits, steps=2, start=5)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("name", ["one", "units", "shifted"])
def test_adamw_shapes(emu, bits, name):
    oc.run_adamw(emu, oc.case_tensors(emu, name, bits, "f32", "f32", start=False), bits, steps=2, clip=0.25,
                 grad_scale=-1.0)


@pytest.mark.parametrize("pk,gk", [("bf16", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("name", ["units", "shifted"])
def test_adamw8_narrow_units(emu, name, pk, gk):
    """Units of 16 blocks, whole, cut short and off their alignment."""
    oc.run_adamw(emu, oc.case_tensors(emu, name, 8, pk, gk), 8, steps=2)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_mixed_types(emu, bits):
    rng = np.random.default_rng(2)
    kinds = [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32")]
    ts = [oc.Tensor(emu, rng, 300 + 100 * i, pk, gk, bits, 0.1) for i, (pk, gk) in enumerate(kinds)]
    oc.run_adamw(emu, ts, bits, steps=2, lr_device=3e-3)


# ------------------------------------------------------------------ refusals
def _norm_create(lib, ptrs, ns, kinds):
    return lib.falcom_norm_create(oc.c_array(ctypes.c_void_p, ptrs), oc.c_array(ctypes.c_size_t, ns),
                                  oc.c_array(ctypes.c_int, kinds), len(ptrs))


def test_norm_refusals(emu, capfd):
    lib = emu.lib
    x = oc.Placed(emu, np.ones(64, np.float32))
    host = np.ones(64, np.float32)
    assert not _norm_create(lib, [x.ptr], [64], [3])
    assert not _norm_create(lib, [x.ptr], [64], [-1])
    assert not _norm_create(lib, [0], [64], [0])
    assert not _norm_create(lib, [x.ptr + 2], [8], [0])
    assert not _norm_create(lib, [host.ctypes.data], [64], [0])
    assert not _norm_create(lib, [x.ptr], [1 << 62], [0])
    assert not _norm_create(lib, [x.ptr], [4096], [0])                 # ends past its memory
    assert not lib.falcom_norm_create(None, None, None, 1)
    plan = _norm_create(lib, [x.ptr], [64], [0])
    work = oc.Placed(emu, np.zeros(lib.falcom_norm_work_bytes(plan), np.uint8))
    out = oc.Placed(emu, np.zeros(2, np.float32))
    for scale, most, o, w in [(math.nan, 1, out.ptr, work.ptr), (math.inf, 1, out.ptr, work.ptr),
                              (1, 0, out.ptr, work.ptr), (1, -1, out.ptr, work.ptr), (1, math.nan, out.ptr, work.ptr),
                              (1, 1, None, work.ptr), (1, 1, out.ptr, None), (1, 1, host.ctypes.data, work.ptr),
                              (1, 1, out.ptr, host.ctypes.data), (1, 1, out.ptr, work.ptr + 4)]:
        assert lib.falcom_norm_run(plan, scale, most, o, w, None) == -4
    assert lib.falcom_norm_run(None, 1, 1, out.ptr, work.ptr, None) == -4
    assert lib.falcom_norm_work_bytes(None) == 0
    assert not out.get().any()
    assert lib.falcom_norm_run(plan, 1, 1, out.ptr, work.ptr, None) == 0 and out.get()[0] == 8.0
    lib.falcom_norm_destroy(plan)
    lib.falcom_norm_destroy(None)
    assert "[ERROR] falcom_norm" in capfd.readouterr().err


def _adamw_create(emu, tensors, bits=32, step=None, edit=None):
    cs = [x.c() for x in tensors]
    if edit:
        edit(cs)
    return emu.lib.falcom_adamw_create(oc.c_array(abi.AdamWTensorC, cs), len(cs), bits, step)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_refusals(emu, bits, capfd):
    rng = np.random.default_rng(3)
    ts = [oc.Tensor(emu, rng, 300, "f32", "f32", bits, 0.1), oc.Tensor(emu, rng, 600, "bf16", "f16", bits, 0.0)]
    step = oc.Placed(emu, np.zeros(1, np.int64))
    host = np.zeros(4096, np.uint8)

    def edits():
        def setter(field, value, i=0):
            return lambda cs: setattr(cs[i], field, value)
        for field in ("param", "grad", "m", "v") + (("m_scale", "v_scale") if bits == 8 else ()):
            yield setter(field, None)
            yield setter(field, host.ctypes.data)
            if field in ("param", "grad") or "scale" in field or bits == 32:
                yield lambda cs, f=field: setattr(cs[0], f, getattr(cs[0], f) + 1)
            if field != "grad":
                yield lambda cs, f=field: setattr(cs[1], f, getattr(cs[0], f))      # the same memory twice
        yield setter("n", 100_000)                                                   # ends past its memory
        yield setter("n", 1 << 60)
        yield setter("param_type", 3)
        yield setter("grad_type", -1)
        yield setter("weight_decay", -0.1)
        yield setter("weight_decay", math.nan)
        yield setter("weight_decay", math.inf)
        yield lambda cs: setattr(cs[0], "grad", cs[0].param)                         # read and written
        yield lambda cs: setattr(cs[1], "grad", cs[0].m)

    for edit in edits():
        assert not _adamw_create(emu, ts, bits, step.ptr, edit)
    assert not _adamw_create(emu, ts, 16, step.ptr)
    assert not _adamw_create(emu, ts, bits, None)
    assert not _adamw_create(emu, ts, bits, step.ptr + 4)
    assert not _adamw_create(emu, ts, bits, host.ctypes.data)
    assert not _adamw_create(emu, ts, bits, ts[0].dp.ptr)
    assert not emu.lib.falcom_adamw_create(None, 2, bits, step.ptr)
    # two parameters may share one gradient: it is only read
    plan = _adamw_create(emu, ts, bits, step.ptr, lambda cs: (setattr(cs[1], "grad", cs[0].grad), setattr(cs[1], "n", 300)))
    assert plan
    emu.lib.falcom_adamw_destroy(plan)
    plan = _adamw_create(emu, ts, bits, step.ptr)
    f = oc.Placed(emu, np.ones(2, np.float32))
    assert f.ptr
    for bad in (dict(lr=-1.0), dict(lr=math.nan), dict(lr=math.inf), dict(beta1=1.0), dict(beta1=-0.1),
                dict(beta2=1.0), dict(beta2=math.nan), dict(eps=0.0), dict(eps=1e-60), dict(eps=math.inf),
                dict(eps=-1.0), dict(grad_scale=math.nan), dict(grad_scale=1e39), dict(clip=host.ctypes.data),
                dict(lr_device=host.ctypes.data), dict(clip=f.ptr + 2)):
        assert emu.lib.falcom_adamw_step(plan, ctypes.byref(oc.make_args(**bad)), None) == -4, bad
    assert emu.lib.falcom_adamw_step(None, ctypes.byref(oc.make_args()), None) == -4
    assert emu.lib.falcom_adamw_step(plan, None, None) == -4
    assert step.get()[0] == 0
    emu.lib.falcom_adamw_destroy(plan)
    emu.lib.falcom_adamw_destroy(None)
    old = [(x.p, x.m, x.v) for x in ts]
    for x, o in zip(ts, old):
        x.refresh()
        assert all((a == b).all() for a, b in zip((x.p, x.m, x.v), o))
    assert "[ERROR] falcom_adamw" in capfd.readouterr().err
