"""8-bit AdamW states whose block maxima are far apart, bit for bit on a GPU
(tests/optim_bits.py)."""
import pytest

from tests import optim_bits as ob

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")
from tests.test_gpu_optim import gpu  # noqa: E402,F401


@pytest.mark.parametrize("layout", list(ob.LAYOUTS))
def test_maxima(gpu, layout):  # noqa: F811
    ob.check_maxima(gpu, *ob.LAYOUTS[layout])


@pytest.mark.parametrize("gradient", ob.VANISHING)
@pytest.mark.parametrize("layout", ["two runs of four", "runs of eight", "shifted", "ragged"])
def test_smallest_roots_keep_a_code(gpu, layout, gradient):  # noqa: F811
    ob.check_maxima(gpu, *ob.LAYOUTS[layout], gradient=gradient)
