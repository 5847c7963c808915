"""What the optimiser operators refuse before they touch a GPU: the product
library's own checks on host memory and bad arguments, and the torch classes'
checks of their lists (the same on a machine with and without a GPU)."""
import ctypes

import numpy as np
import pytest

from compressor_b200 import abi
from tests import optim_cases as oc


@pytest.fixture(scope="module")
def lib(product_lib):
    lib = ctypes.CDLL(product_lib)
    abi.bind_optim(lib)
    return lib


def test_library_refuses_host_memory(lib, capfd):
    x = np.ones(1024, np.float32)
    ptrs = oc.c_array(ctypes.c_void_p, [x.ctypes.data])
    assert not lib.falcom_norm_create(ptrs, oc.c_array(ctypes.c_size_t, [1024]), oc.c_array(ctypes.c_int, [0]), 1)
    t = abi.AdamWTensorC(param=x.ctypes.data, grad=x.ctypes.data, m=x.ctypes.data, v=x.ctypes.data, n=16)
    for bits in (32, 8, 16):
        assert not lib.falcom_adamw_create(oc.c_array(abi.AdamWTensorC, [t]), 1, bits, x.ctypes.data)
    assert lib.falcom_norm_run(None, 1.0, 1.0, None, None, None) == abi.ERROR_INVALID_PARAM
    assert lib.falcom_adamw_step(None, ctypes.byref(oc.make_args()), None) == abi.ERROR_INVALID_PARAM
    assert lib.falcom_adamw_errors(None) == abi.ERROR_INVALID_PARAM
    lib.falcom_norm_destroy(None)
    lib.falcom_adamw_destroy(None)
    assert (x == 1).all() and "[ERROR] falcom_adamw_create" in capfd.readouterr().err


def test_struct_layouts_match_the_header():
    """Offsets as a C compiler lays the header's structs out on this ABI."""
    t, a = abi.AdamWTensorC, abi.AdamWArgsC
    assert [getattr(t, f).offset for f, _ in t._fields_] == [0, 8, 16, 24, 32, 40, 48, 56, 60, 64]
    assert ctypes.sizeof(t) == 72
    assert [getattr(a, f).offset for f, _ in a._fields_] == [0, 8, 16, 24, 32, 40, 48, 56]
    assert ctypes.sizeof(a) == 64


def test_classes_refuse_lists(product_lib):
    torch = pytest.importorskip("torch")
    from compressor_b200 import optim
    x, y = torch.zeros(8, 8), torch.zeros(8, 8)
    for bad in ([x], [x.double()], [x.int()], [x.to_sparse()]):
        with pytest.raises(ValueError):
            optim.GradNorm(bad)
        with pytest.raises(ValueError):
            optim.AdamW(bad, [y])
    with pytest.raises(TypeError):
        optim.GradNorm([np.zeros(3)])
    assert optim._dense_strides(x) == optim._dense_strides(x.clone()) and optim._dense_strides(x[:, ::2]) is None
    assert optim._dense_strides(x.t()) != optim._dense_strides(x) and optim._dense_strides(x.expand(3, 8, 8)) is None
    assert optim._dense_strides(torch.zeros(4, 1, 6)[:, :, :]) == optim._dense_strides(torch.zeros(4, 6))
