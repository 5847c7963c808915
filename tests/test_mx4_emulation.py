"""The kernels of the 4-bit operators (but for the product's, which are tensor
core instructions) and of dropout on the CPU, through the kernel emulator,
against their definition in 64 bits: indexing, short blocks, misaligned rows,
padding, what lies beside the arrays; and the layer's two calls around a plain
product."""
import ctypes

import numpy as np
import pytest

from compressor_b200 import abi

torch = pytest.importorskip("torch")

from tests import mx4_reference as ref  # noqa: E402

KIND = {torch.float32: abi.TYPE_F32, torch.bfloat16: abi.TYPE_BF16, torch.float16: abi.TYPE_F16}
TYPES = list(KIND)
GUARD = 64


@pytest.fixture(scope="module")
def lib():
    from tests.emu import build_mx4
    lib = ctypes.CDLL(build_mx4.build())
    abi.bind_mx4(lib)
    lib.emu_device_alloc.argtypes = [ctypes.c_size_t]
    lib.emu_device_alloc.restype = ctypes.c_void_p
    lib.emu_device_free.argtypes = [ctypes.c_void_p]
    lib.emu_device_free.restype = None
    return lib


class Mem:
    """Bytes that the library takes for device memory, between guards."""

    def __init__(self, lib, size, tensor=None, shift=0):
        self.lib, self.size = lib, size
        self.base = lib.emu_device_alloc(size + shift + 2 * GUARD)
        ctypes.memset(self.base, 0xA5, size + shift + 2 * GUARD)
        self.at, self.end = self.base + GUARD + shift, self.base + GUARD + shift + size
        if tensor is not None:
            raw = tensor.contiguous().view(torch.uint8).numpy()
            ctypes.memmove(self.at, raw.ctypes.data, size)

    def read(self, dtype=torch.uint8):
        assert ctypes.string_at(self.base, self.at - self.base) == b"\xa5" * (self.at - self.base)
        assert ctypes.string_at(self.end, GUARD) == b"\xa5" * GUARD
        return torch.frombuffer(bytearray(ctypes.string_at(self.at, self.size)), dtype=dtype)

    def __del__(self):
        self.lib.emu_device_free(self.base)


def held(lib, t, shift=0):
    return Mem(lib, t.numel() * t.element_size(), t, shift * t.element_size())


def matrix(lib, rows, cols):
    m = Mem(lib, lib.falcom_mx4_codes_bytes(rows, cols)), Mem(lib, lib.falcom_mx4_scales_bytes(rows, cols))
    return m, abi.Mx4MatrixC(m[0].at, m[1].at, rows, cols)


def wild(rows, cols, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-6, 6, (rows, 1), generator=g).float())
    flat = x.view(-1)
    flat[::5] = torch.round(flat[::5] * 8) / 8
    flat[3::17] = 0.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,beside", [(1, 1, 0), (3, 33, 0), (9, 300, 1), (130, 40, 0), (129, 400, 3)])
@pytest.mark.parametrize("random", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_quantize(lib, rows, cols, beside, dtype, random, p):
    x = wild(rows, cols, dtype, 1)
    if cols > 40:
        x[0, 35], x[-1, 0] = float("nan"), float("-inf")
    room = torch.full((rows, cols + beside), 3.0, dtype=dtype)
    room[:, :cols] = x
    mem = held(lib, room)
    rnd, drop = abi.RandomC(77, None), abi.DropoutArgsC(p, abi.RandomC(5, None))
    (rm, r), (cm, c) = matrix(lib, rows, cols), matrix(lib, cols, rows)
    rc = lib.falcom_mx4_quantize(mem.at, KIND[dtype], rows, cols, cols + beside, ctypes.byref(rnd) if random else None,
                                 ctypes.byref(drop), ctypes.byref(r), ctypes.byref(c), None)
    assert rc == 0
    d = ref.dropped(x, p, 5).float() if p else x
    bits = ref.random_bits(ref.places(rows, cols), ref.ROUNDING, 77) if random else None
    for got, want in ((rm, ref.codes(d, bits)), (cm, ref.codes(d.t(), bits.t() if random else None))):
        codes, scales = ref.pack(*want)
        assert torch.equal(got[0].read(), codes) and torch.equal(got[1].read(), scales)
    out = Mem(lib, rows * cols * 4)
    assert lib.falcom_mx4_dequantize(ctypes.byref(r), out.at, abi.TYPE_F32, cols, None) == 0
    assert torch.equal(out.read(torch.float32).view(rows, cols).nan_to_num(9.5), ref.values(d, bits).float().nan_to_num(9.5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 33, 256, 1000, 5130])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("random", [False, True])
def test_encode_and_decode(lib, n, dtype, shift, random):
    x, base, out = wild(1, n, dtype, 2)[0], wild(1, n, torch.float32, 3)[0], wild(1, n, dtype, 4)[0]
    xm, bm, om = held(lib, x, shift), held(lib, base, shift), held(lib, out, shift)
    codes, scales, counter = Mem(lib, (n + 1) // 2), Mem(lib, -(-n // 32)), held(lib, torch.tensor([3]))
    rnd = abi.RandomC(9, counter.at)
    assert lib.falcom_mx4_encode(xm.at, KIND[dtype], n, bm.at, ctypes.byref(rnd) if random else None, codes.at, scales.at, None) == 0
    bits = ref.random_bits(ref.places(1, n), ref.ROUNDING, 9, 3) if random else None
    code, e, fine = ref.codes((x.float() - base)[None], bits)
    padded = torch.nn.functional.pad(code[0], (0, n % 2))
    assert torch.equal(codes.read(), (padded[::2] | padded[1::2] << 4).to(torch.uint8))
    assert torch.equal(scales.read(), (e[0] + 127).to(torch.uint8))
    v = ref.values((x.float() - base)[None], bits)[0].float()
    assert torch.equal(bm.read(torch.float32), base + v)
    assert lib.falcom_mx4_decode(codes.at, scales.at, n, 0.3, 1, om.at, KIND[dtype], None) == 0
    assert torch.equal(om.read(dtype), (out.float() + torch.tensor(0.3) * v).to(dtype))
    assert lib.falcom_mx4_decode(codes.at, scales.at, n, 1.0, 0, om.at, KIND[dtype], None) == 0
    assert torch.equal(om.read(dtype), v.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 8), (5, 33), (4, 64), (1, 1000)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_dropout(lib, rows, cols, dtype, residual, shift):
    x, r = wild(rows, cols, dtype, 5), wild(rows, cols, dtype, 6)
    xm, rm, ym = held(lib, x, shift), held(lib, r), Mem(lib, x.numel() * x.element_size())
    drop = abi.DropoutArgsC(0.4, abi.RandomC((1 << 40) + 3, None))
    assert lib.falcom_dropout(xm.at, rm.at if residual else None, ym.at, KIND[dtype], rows, cols, ctypes.byref(drop), None) == 0
    want = ref.dropped(x, 0.4, (1 << 40) + 3).float()
    assert torch.equal(ym.read(dtype).view(rows, cols), (want + r.float() if residual else want).to(dtype))
    # in place
    assert lib.falcom_dropout(xm.at, None, xm.at, KIND[dtype], rows, cols, ctypes.byref(drop), None) == 0
    assert torch.equal(xm.read(dtype).view(rows, cols), want.to(dtype))


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("t,k,n", [(1, 32, 8), (20, 70, 40), (3, 260, 1)])
@pytest.mark.parametrize("want_dx,want_dw", [(1, 1), (1, 0), (0, 1)])
def test_layer(lib, t, k, n, p, want_dx, want_dw):
    x, w, dy = wild(t, k, torch.bfloat16, 7), wild(n, k, torch.float32, 8), wild(t, n, torch.bfloat16, 9)
    counter = held(lib, torch.tensor([6]))
    layer = abi.Mx4LinearC(t, k, n, abi.TYPE_BF16, abi.TYPE_F32, want_dx, want_dw, p, abi.RandomC(11, counter.at))
    ref_ = ctypes.byref(layer)
    xm, wm, gm, y = held(lib, x), held(lib, w), held(lib, dy), Mem(lib, t * n * 2)
    kept = Mem(lib, lib.falcom_mx4_linear_kept_bytes(ref_))
    work = Mem(lib, lib.falcom_mx4_linear_work_bytes(ref_, 0))
    assert lib.falcom_mx4_linear_forward(ref_, xm.at, k, wm.at, k, y.at, kept.at, work.at, None) == 0
    d = ref.dropped(x, p, 11, 6)
    bits = ref.random_bits(ref.places(t, n), ref.ROUNDING, 11, 6)

    def near(got, a, b, dtype, factor=1.0):
        want = (a @ b.t()) * factor
        return ((got.double() - want).abs() <= 2 * ref.sum_bound(a, b, dtype) + 2.0 ** -22 * want.abs()).all()

    assert near(y.read(torch.bfloat16).view(t, n), ref.values(d), ref.values(w), torch.bfloat16)
    kept.read(), work.read()
    dx, dw = Mem(lib, t * k * 2), Mem(lib, n * k * 4)
    work = Mem(lib, lib.falcom_mx4_linear_work_bytes(ref_, 1))
    assert lib.falcom_mx4_linear_backward(ref_, gm.at, n, kept.at, dx.at if want_dx else None, dw.at if want_dw else None,
                                          work.at, None) == 0
    work.read()
    if want_dx:
        mask = ref.dropped(torch.ones(t, k), p, 11, 6)
        assert near(dx.read(torch.bfloat16).view(t, k), ref.values(dy, bits), ref.values(w.t()), torch.bfloat16, mask)
    if want_dw:
        assert near(dw.read(torch.float32).view(n, k), ref.values(dy.t(), bits.t()), ref.values(d.t()), torch.float32)


def test_calls_are_refused_where_arrays_overlap_or_end(lib):
    x = held(lib, wild(4, 32, torch.float32, 1))
    (m, c), r = matrix(lib, 4, 32), abi.ERROR_INVALID_PARAM
    ref_ = ctypes.byref(c)
    assert lib.falcom_mx4_encode(x.at, 0, 128, x.at, None, m[0].at, m[1].at, None) == r          # base is x
    assert lib.falcom_mx4_encode(x.at, 0, 128, None, None, x.at, m[1].at, None) == r             # codes over x
    assert lib.falcom_mx4_encode(x.at, 0, 1 << 20, None, None, m[0].at, m[1].at, None) == r      # x ends before
    assert lib.falcom_mx4_encode(x.at + 2, 0, 8, None, None, m[0].at, m[1].at, None) == r        # alignment
    assert lib.falcom_mx4_encode(x.at, 0, 8, None, None, m[0].at + 8, m[1].at, None) == r
    assert lib.falcom_mx4_encode(x.at, 0, 8, None, ctypes.byref(abi.RandomC(1, x.at + 4)), m[0].at, m[1].at, None) == r
    assert lib.falcom_mx4_quantize(x.at, 0, 4, 32, 32, None, None, ref_, ctypes.byref(abi.Mx4MatrixC(m[0].at, m[1].at, 32, 4)), None) == r
    assert lib.falcom_mx4_product(ref_, ref_, m[0].at, 0, 4, None, None) == r                    # out over a factor
    assert lib.falcom_dropout(x.at, None, x.at + 4, 0, 1, 100, ctypes.byref(abi.DropoutArgsC(0.5, abi.RandomC(1, None))), None) == r
    assert lib.falcom_mx4_errors() == 0
    x.read()
