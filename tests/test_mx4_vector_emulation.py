"""A 4-bit vector as one run of bytes (falcom_mx4_encode_vector) on the CPU,
through the kernel emulator: every byte is written, nothing beside it."""
import ctypes

import pytest

from compressor_b200 import abi

torch = pytest.importorskip("torch")

from tests.test_mx4_emulation import KIND, Mem, held, lib, wild  # noqa: E402, F401


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 256, 257, 1000, 5130])
@pytest.mark.parametrize("dtype,shift,based,random", [(torch.float32, 0, True, False), (torch.bfloat16, 1, False, True),
                                                      (torch.float16, 0, False, False), (torch.float32, 1, True, True)])
def test_every_byte_of_a_vector(lib, n, dtype, shift, based, random):  # noqa: F811
    x, base = wild(1, n, dtype, 2)[0], wild(1, n, torch.float32, 3)[0]
    rnd = ctypes.byref(abi.RandomC(9, None)) if random else None
    xm, one, other = held(lib, x, shift), held(lib, base, shift), held(lib, base, shift)
    codes, scales = Mem(lib, (n + 1) // 2), Mem(lib, -(-n // 32))
    size, begin = lib.falcom_mx4_vector_bytes(n), -(-((n + 1) // 2) // 16) * 16
    assert size == begin + -(-n // 32)
    whole = Mem(lib, size)   # (filled with something else)
    assert lib.falcom_mx4_encode(xm.at, KIND[dtype], n, one.at if based else None, rnd, codes.at, scales.at, None) == 0
    assert lib.falcom_mx4_encode_vector(xm.at, KIND[dtype], n, other.at if based else None, rnd, whole.at, None) == 0
    got = whole.read()
    assert torch.equal(got[:(n + 1) // 2], codes.read()) and torch.equal(got[begin:], scales.read())
    assert not got[(n + 1) // 2:begin].any()
    assert torch.equal(one.read(torch.float32), other.read(torch.float32))


def test_sizes_and_refusals(lib):  # noqa: F811
    from compressor_b200.mx4 import Mx4Vector
    for n in (0, 1, 31, 32, 33, 1000, 1 << 40):
        assert lib.falcom_mx4_vector_bytes(n) == Mx4Vector.size_of(n)
    assert lib.falcom_mx4_vector_bytes((1 << 40) + 1) == 0
    x, v, r = held(lib, torch.ones(64)), Mem(lib, 34), abi.ERROR_INVALID_PARAM
    assert lib.falcom_mx4_encode_vector(x.at, 0, 64, None, None, v.at, None) == 0
    assert lib.falcom_mx4_encode_vector(x.at, 0, 64, None, None, None, None) == r
    assert lib.falcom_mx4_encode_vector(x.at, 0, 64, None, None, v.at + 8, None) == r        # alignment
    assert lib.falcom_mx4_encode_vector(x.at, 0, 64, None, None, x.at, None) == r            # over x
    assert lib.falcom_mx4_encode_vector(x.at, 3, 64, None, None, v.at, None) == r
    assert lib.falcom_mx4_encode_vector(x.at, 0, (1 << 40) + 1, None, None, v.at, None) == r
    assert lib.falcom_mx4_encode(x.at, 0, 64, None, None, v.at, None, None) == r             # no scales
    assert lib.falcom_mx4_encode_vector(None, 0, 0, None, None, None, None) == 0
    x.read(), v.read()
