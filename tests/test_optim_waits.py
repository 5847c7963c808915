"""Waits of the 8-bit AdamW kernel that run out, on the CPU through the kernel
emulator, which makes chosen waits report so."""
import ctypes

import numpy as np
import pytest

from compressor_b200 import abi
from tests import optim_cases as oc
from tests.test_optim_emulation import emu  # noqa: F401


@pytest.fixture
def late(emu):  # noqa: F811
    yield emu.lib.emu_optim_late_waits
    emu.lib.emu_optim_late_waits(0)


def _step(emu, late, n):  # noqa: F811
    """One step with n waits that run out; returns (tensor, error word, counter)."""
    x = oc.Tensor(emu, np.random.default_rng(1), 2048 * 8, "f32", "f32", 8, 0.1)
    step = oc.Placed(emu, np.zeros(1, np.int64))
    plan = emu.lib.falcom_adamw_create(oc.c_array(abi.AdamWTensorC, [x.c()]), 1, 8, step.ptr)
    assert plan and emu.lib.falcom_adamw_errors(plan) == 0
    late(n)
    assert emu.lib.falcom_adamw_step(plan, ctypes.byref(oc.make_args()), None) == 0
    late(0)
    errors = emu.lib.falcom_adamw_errors(plan)
    emu.lib.falcom_adamw_destroy(plan)
    return x, errors, int(step.get()[0])


def test_copies_that_arrive_in_the_second_wait_are_used(emu, late):  # noqa: F811
    x, errors, step = _step(emu, late, 1)
    assert errors == 0 and step == 1
    oc.check_step([x], 1, oc.HYPER)


def test_copies_that_never_arrive_are_reported(emu, late):  # noqa: F811
    x, errors, step = _step(emu, late, 1 << 30)
    assert errors == 1 and step == 1
