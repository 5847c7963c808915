"""Device arguments of the optimiser calls that are shorter than what the
kernels read and write, through the kernel emulator (which knows every
allocation's length)."""
import ctypes

import numpy as np
import pytest

from compressor_b200 import abi
from tests import optim_cases as oc
from tests.test_optim_emulation import _norm_create, emu  # noqa: F401


class Block:
    """Device memory of n bytes, n a multiple of 256: it starts and ends on 256-byte boundaries."""

    def __init__(self, emu, n):  # noqa: F811
        self.lib, self.n = emu.lib, n
        self.ptr = emu.lib.emu_device_alloc(n)
        assert self.ptr % 256 == 0
        ctypes.memset(self.ptr, 0, n)

    def __del__(self):
        self.lib.emu_device_free(self.ptr)


def test_short_scratch_is_refused(emu):  # noqa: F811
    lib = emu.lib
    x = oc.Placed(emu, np.ones(100_000, np.float32))
    plan = _norm_create(lib, [x.ptr], [x.n], [0])
    need = lib.falcom_norm_work_bytes(plan)
    assert 64 < need <= 256
    out, b = oc.Placed(emu, np.zeros(2, np.float32)), Block(emu, 1024)
    end = b.ptr + b.n
    for short in (8, need // 2 & ~7, need - 8):
        assert lib.falcom_norm_run(plan, 1.0, 1.0, out.ptr, end - short, None) == abi.ERROR_INVALID_PARAM
    assert lib.falcom_norm_run(plan, 1.0, 1.0, end - 4, b.ptr, None) == abi.ERROR_INVALID_PARAM
    assert not out.get().any()
    assert lib.falcom_norm_run(plan, 1.0, 1.0, out.ptr, end - need, None) == 0
    assert abs(out.get()[0] - 100_000 ** 0.5) < 1e-4
    assert lib.falcom_norm_run(plan, 1.0, 1.0, end - 8, b.ptr, None) == 0
    lib.falcom_norm_destroy(plan)


@pytest.mark.parametrize("bits", [32, 8])
def test_short_coefficient_is_refused(emu, bits):  # noqa: F811
    t = oc.Tensor(emu, np.random.default_rng(0), 700, "f32", "f32", bits, 0.1)
    step = oc.Placed(emu, np.zeros(1, np.int64))
    plan = emu.lib.falcom_adamw_create(oc.c_array(abi.AdamWTensorC, [t.c()]), 1, bits, step.ptr)
    b = Block(emu, 256)
    ctypes.memset(b.ptr, 0, 256)
    end = b.ptr + b.n
    assert emu.lib.falcom_adamw_step(plan, ctypes.byref(oc.make_args(clip=end - 4)), None) == abi.ERROR_INVALID_PARAM
    assert step.get()[0] == 0
    for kw in (dict(clip=end - 8), dict(lr_device=end - 4)):
        assert emu.lib.falcom_adamw_step(plan, ctypes.byref(oc.make_args(**kw)), None) == 0
    assert step.get()[0] == 2
    emu.lib.falcom_adamw_destroy(plan)
