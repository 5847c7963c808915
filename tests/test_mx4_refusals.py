"""What the 4-bit operators and dropout refuse before they touch a GPU, and
their host-side sizes (the same on a machine with and without a GPU)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from compressor_b200 import abi

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(product_lib):
    lib = ctypes.CDLL(product_lib)
    abi.bind_mx4(lib)
    return lib


def refused(rc):
    return rc == abi.ERROR_INVALID_PARAM


def test_struct_layouts_match_the_header(tmp_path):
    names = {"falcom_random": abi.RandomC, "falcom_dropout_args": abi.DropoutArgsC, "falcom_mx4_matrix": abi.Mx4MatrixC,
             "falcom_mx4_linear": abi.Mx4LinearC}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "falcom_b200.h"', "int main(void) {"]
    for c, py in names.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    (tmp_path / "probe.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-I", "/usr/local/cuda/include", "probe.c", "-o", "probe"],
                   cwd=tmp_path, check=True)
    got = [int(v) for v in subprocess.run(["./probe"], cwd=tmp_path, capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in names.values():
        want += [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want


def test_sizes(lib):
    from compressor_b200.mx4 import Mx4Matrix, Mx4Vector
    for rows, cols in [(1, 1), (8, 256), (9, 257), (128, 32), (129, 1000), (0, 5), (5, 0), (50257, 1024)]:
        codes, scales = lib.falcom_mx4_codes_bytes(rows, cols), lib.falcom_mx4_scales_bytes(rows, cols)
        assert (codes, scales) == Mx4Matrix.sizes_of(rows, cols)
        assert lib.falcom_mx4_work_bytes(rows, cols) == (0 if rows <= 16 and cols <= 4096 and rows * cols <= 32768 else codes + scales)
        # 4 bits an element and one byte per 32, filled up to 8 rows (scales: 128) and 256 columns
        if rows and cols:
            assert codes == -(-cols // 256) * 256 * -(-rows // 8) * 8 // 2
            assert scales == -(-cols // 256) * 8 * -(-rows // 128) * 128
    assert lib.falcom_mx4_codes_bytes(2 ** 31 + 1, 1) == 0 == lib.falcom_mx4_scales_bytes(1, 2 ** 31 + 1)
    for n in (0, 1, 31, 32, 33, 1000):
        assert Mx4Vector.size_of(n) == -(-(-(-n // 2)) // 16) * 16 + -(-n // 32)
    layer = abi.Mx4LinearC(rows=7, cols=300, outs=20, want_dx=1, want_dw=0)
    assert lib.falcom_mx4_linear_kept_bytes(ctypes.byref(layer)) == sum(Mx4Matrix.sizes_of(300, 20))
    assert lib.falcom_mx4_linear_work_bytes(ctypes.byref(layer), 0) == sum(Mx4Matrix.sizes_of(7, 300)) + sum(Mx4Matrix.sizes_of(20, 300))
    assert lib.falcom_mx4_linear_work_bytes(ctypes.byref(layer), 1) == sum(Mx4Matrix.sizes_of(7, 20))


def test_library_refuses_host_memory_and_bad_arguments(lib, capfd):
    x = np.ones(4096, np.float32)
    at = x.ctypes.data
    m = abi.Mx4MatrixC(at, at, 4, 8)
    r = ctypes.byref
    none = abi.DropoutArgsC(1.0, abi.RandomC(0, None))
    some = abi.DropoutArgsC(0.5, abi.RandomC(0, None))
    assert refused(lib.falcom_mx4_encode(at, 0, 32, None, None, at, at, None))
    assert refused(lib.falcom_mx4_encode(None, 0, 32, None, None, None, None, None))
    assert refused(lib.falcom_mx4_encode(at, 7, 32, None, None, at, at, None))
    assert refused(lib.falcom_mx4_decode(at, at, 32, 1.0, 0, at, 0, None))
    assert refused(lib.falcom_mx4_decode(at, at, 32, float("nan"), 0, at, 0, None))
    assert refused(lib.falcom_mx4_quantize(at, 0, 4, 8, 8, None, None, r(m), None, None))
    assert refused(lib.falcom_mx4_quantize(at, 0, 4, 8, 7, None, None, r(m), None, None))           # rows overlap
    assert refused(lib.falcom_mx4_quantize(at, 0, 4, 9, 9, None, None, r(m), None, None))           # another size
    assert refused(lib.falcom_mx4_quantize(at, 0, 4, 8, 8, None, None, None, r(m), None))           # not transposed
    assert refused(lib.falcom_mx4_quantize(at, 0, 4, 8, 8, None, r(none), r(m), None, None))        # p = 1
    assert refused(lib.falcom_mx4_quantize(at, 0, 1 << 31, 1 << 31, 1 << 40, None, None, r(m), None, None))
    assert refused(lib.falcom_mx4_dequantize(r(m), at, 0, 8, None))
    assert refused(lib.falcom_mx4_dequantize(None, at, 0, 8, None))
    assert refused(lib.falcom_mx4_product(r(m), r(m), at, 0, 4, None, None))
    assert refused(lib.falcom_mx4_product(r(m), r(m), at, 0, 3, None, None))
    assert refused(lib.falcom_mx4_product(r(m), r(abi.Mx4MatrixC(at, at, 4, 9)), at, 0, 4, None, None))
    assert refused(lib.falcom_mx4_product(None, r(m), at, 0, 4, None, None))
    assert refused(lib.falcom_mx4_product_of(at, 0, 4, 8, r(m), at, 0, 4, at, None))
    assert refused(lib.falcom_mx4_product_of(at, 3, 4, 8, r(m), at, 0, 4, at, None))
    layer = abi.Mx4LinearC(rows=4, cols=8, outs=4, want_dx=1)
    assert refused(lib.falcom_mx4_linear_forward(r(layer), at, 8, at, 8, at, at, at, None))
    assert refused(lib.falcom_mx4_linear_forward(None, at, 8, at, 8, at, at, at, None))
    assert refused(lib.falcom_mx4_linear_backward(r(layer), at, 4, at, at, None, at, None))
    assert refused(lib.falcom_mx4_linear_backward(r(layer), at, 4, at, None, at, at, None))         # dw was not wanted
    assert refused(lib.falcom_dropout(at, None, at, 0, 4, 8, r(some), None))
    assert refused(lib.falcom_dropout(at, None, at, 0, 4, 8, None, None))
    assert refused(lib.falcom_dropout(at, None, at, 0, 4, 8, r(none), None))
    assert refused(lib.falcom_dropout(at, None, at, 0, 1 << 31, 1 << 31, r(some), None))
    # nothing to do is no error, whatever the addresses
    assert lib.falcom_mx4_encode(None, 0, 0, None, None, None, None, None) == 0
    assert lib.falcom_mx4_quantize(None, 0, 0, 8, 8, None, None, None, None, None) == 0
    assert lib.falcom_dropout(None, None, None, 0, 0, 8, r(some), None) == 0
    assert (x == 1).all() and "[ERROR] falcom_mx4_product" in capfd.readouterr().err


def test_functions_refuse_tensors(product_lib):
    from compressor_b200 import dropout, mx4
    x = torch.zeros(8, 32)
    for bad in (x, x.double(), x.int(), x.to_sparse()):
        for call in (lambda: mx4.encode(bad), lambda: mx4.quantize(bad), lambda: mx4.linear(bad, bad), lambda: dropout.dropout(bad)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: mx4.encode([1.0]), lambda: mx4.product(x, x), lambda: dropout.dropout(3)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError, match="along"):
        mx4.quantize(x, along="diagonal")
    with pytest.raises(ValueError, match="accumulate"):
        mx4.decode(mx4.Mx4Vector.empty(32, "cpu"), accumulate=True)
    with pytest.raises(ValueError, match="CUDA device is wanted"):
        mx4.decode(mx4.Mx4Vector.empty(32, "cpu"))
    with pytest.raises(ValueError, match="bytes"):
        mx4.Mx4Vector(33, torch.zeros(17, dtype=torch.uint8))
    with pytest.raises(ValueError, match="bytes"):
        mx4.Mx4Matrix(1, 1, torch.zeros(5, dtype=torch.uint8))
    for bad in (-0.1, 1.0, 0.9999999, float("nan")):
        with pytest.raises(ValueError, match="p must"):
            mx4._check_p(bad)
    with pytest.raises(ValueError, match="64 bits"):
        mx4._seeded(-1, None, torch.device("cpu"))
    with pytest.raises(ValueError, match="counter"):
        mx4._seeded(1, torch.zeros(2, dtype=torch.int64), torch.device("cpu"))
    with pytest.raises(ValueError, match="rounding"):
        mx4._random("up", 1, None, torch.device("cpu"))


def test_reference_rounding_is_unbiased_and_complete():
    """The comparison's own definition: exact values stay, ties go to even
    codes, random rounding is right on average."""
    from tests import mx4_reference as ref
    grid = torch.cat([ref.VALUES, -ref.VALUES, torch.tensor([6.0])]).float()[None]
    assert torch.equal(ref.values(grid), grid.double())
    ties = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, 6.0]])
    assert ref.values(ties)[0].tolist() == [0, 1, 1, 2, 2, 4, 4, -4, 6]
    n = 1 << 15
    x = torch.full((1, n), 2.3)
    x[:, ::32] = 6.0
    bits = ref.random_bits(ref.places(1, n), ref.ROUNDING, 5)
    v = ref.values(x, bits)[0].view(-1, 32)[:, 1:]
    assert set(v.unique().tolist()) == {2.0, 3.0}
    # 31 n / 32 draws of chance 0.3: five standard deviations
    assert abs(v.mean().item() - 2.3) < 5 * (0.21 / v.numel()) ** 0.5
    top = torch.tensor([[2.0 ** 127 * 1.75, 1.0], [2.0 ** -149, 0.0], [float("inf"), 1.0], [1.0, float("nan")]])
    e, fine = ref.scales(top.double())
    assert e[:2, 0].tolist() == [126, -127] and fine[:, 0].tolist() == [True, True, False, False]
