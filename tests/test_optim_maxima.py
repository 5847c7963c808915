"""8-bit AdamW states whose block maxima are far apart, on the CPU through
the kernel emulator (tests/optim_bits.py; tests/test_gpu_optim_maxima.py runs
the same on a GPU)."""
import pytest

from tests import optim_bits as ob
from tests.test_optim_emulation import emu  # noqa: F401


@pytest.mark.parametrize("layout", list(ob.LAYOUTS))
def test_maxima(emu, layout):  # noqa: F811
    ob.check_maxima(emu, *ob.LAYOUTS[layout])


@pytest.mark.parametrize("gradient", ob.VANISHING)
@pytest.mark.parametrize("layout", ["two runs of four", "runs of eight", "shifted", "ragged"])
def test_smallest_roots_keep_a_code(emu, layout, gradient):  # noqa: F811
    ob.check_maxima(emu, *ob.LAYOUTS[layout], gradient=gradient)
