"""The 4-bit product's kernels on the CPU, through an emulation of clusters,
copies, tensor memory and matrix instructions: every form, with more panels
than stages, more tiles than SMs, rows of results at all offsets; compared
without a tolerance."""
import ctypes

import pytest

from compressor_b200 import abi

torch = pytest.importorskip("torch")

from tests import mx4_exact as exact  # noqa: E402
from tests import mx4_reference as ref  # noqa: E402

KIND = {torch.float32: abi.TYPE_F32, torch.bfloat16: abi.TYPE_BF16, torch.float16: abi.TYPE_F16}


class Launch(ctypes.Structure):
    """mx_product_launch of mc_mx4.h."""
    _fields_ = [("a_codes", ctypes.c_void_p), ("a_scales", ctypes.c_void_p), ("a_rows", ctypes.c_int64), ("a_cols", ctypes.c_int64),
                ("b_codes", ctypes.c_void_p), ("b_scales", ctypes.c_void_p), ("b_rows", ctypes.c_int64), ("b_cols", ctypes.c_int64),
                ("out", ctypes.c_void_p), ("ld", ctypes.c_int64),
                ("key", ctypes.c_uint32), ("on", ctypes.c_int32), ("counter", ctypes.c_void_p), ("key_a", ctypes.c_uint32),
                ("key_b", ctypes.c_uint32), ("threshold", ctypes.c_uint32), ("factor", ctypes.c_float),
                ("x", ctypes.c_void_p), ("ld_x", ctypes.c_int64), ("x_type", ctypes.c_int32), ("vectors", ctypes.c_int32)]


@pytest.fixture(scope="module")
def lib():
    from tests.emu import build_product
    lib = ctypes.CDLL(build_product.build())
    lib.emu_product.argtypes = [ctypes.POINTER(Launch), ctypes.c_double, ctypes.c_uint64, ctypes.c_int, ctypes.c_int]
    lib.emu_product_lose.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_double]
    lib.emu_product_lose.restype = None
    return lib


def aligned(t):
    """t in memory on a 16-byte boundary."""
    raw = t.contiguous().view(torch.uint8)
    room = torch.zeros(raw.numel() + 16, dtype=torch.uint8)
    at = -room.data_ptr() % 16
    room[at:at + raw.numel()] = raw.view(-1)
    return room[at:at + raw.numel()]


def call(lib, a, b, dtype, sms, p=0.0, seed=5, x=None, shift=0, beside=0):
    """The product of two matrices that 4 bits hold (or of x, rounded inside);
    (out, whether what lies beside it was left alone)."""
    (t, k), n = a.shape if x is None else x.shape, b.shape[0]
    keep = [aligned(part) for part in ref.pack(*ref.codes(b))]
    launch = Launch(a_rows=t, a_cols=k, b_codes=keep[0].data_ptr(), b_scales=keep[1].data_ptr(), b_rows=n, b_cols=k, ld=n + beside)
    if x is None:
        keep += [aligned(part) for part in ref.pack(*ref.codes(a))]
        launch.a_codes, launch.a_scales = keep[2].data_ptr(), keep[3].data_ptr()
    else:
        keep.append(aligned(x))
        launch.x, launch.ld_x, launch.x_type = keep[2].data_ptr(), k, KIND[x.dtype]
        launch.vectors = k * x.element_size() % 16 == 0
    room = torch.full((t * (n + beside) + shift + 8,), 7.0, dtype=dtype)
    room = room[-room.data_ptr() // room.element_size() % (16 // room.element_size()):]
    out = room[shift:shift + t * (n + beside)]
    launch.out = out.data_ptr()
    assert lib.emu_product(ctypes.byref(launch), p, seed, KIND[dtype], sms) == 0
    out = out.view(t, n + beside)
    return out[:, :n], bool((room[:shift] == 7).all() and (room[shift + t * (n + beside):] == 7).all() and (out[:, n:] == 7).all())


# (t, n, k), SMs: what it is for
NARROW = [
    ((1, 1, 1), 4, "the smallest"),
    ((1, 300, 2600), 2, "16 rows a tile, more panels than the 7 stages"),
    ((16, 130, 2100), 1, "no cluster, 9 panels"),
    ((3, 100, 2400), 8, "a cluster of 8, whose ranks have 1 or 2 panels"),
    ((5, 200, 5000), 4, "a cluster of 2, 10 panels each"),
    ((24, 140, 2000), 2, "32 rows a tile, more panels than stages"),
    ((40, 520, 1300), 1, "64 rows a tile, more CTAs than SMs: fewer stages"),
    ((64, 100, 1300), 2, "a cluster of 2"),
    ((100, 130, 1800), 1, "128 rows a tile, 8 panels of 5 stages"),
    ((128, 390, 1100), 1, "128 rows a tile, 4 CTAs on an SM"),
    ((129, 100, 1400), 1, "256 rows a tile, 6 panels of 4 stages"),
    ((600, 60, 900), 1, "256 rows a tile, 3 CTAs for an SM: one stage"),
    ((260, 120, 2400), 4, "256 rows a tile in clusters"),
]
WIDE = [
    ((129, 300, 64), 2, "one pair, two tiles of one panel of one step"),
    ((300, 520, 700), 2, "one pair, 6 tiles of 3 panels: sums overlap, stages wrap"),
    ((300, 260, 1500), 4, "two pairs, more panels than stages"),
    ((513, 257, 200), 2, "last rows and columns of one element"),
]


@pytest.mark.parametrize("size,sms,why", NARROW + WIDE)
def test_products_are_exact(lib, size, sms, why):
    t, n, k = size
    a, b = exact.matrix(t, k, 1), exact.matrix(n, k, 2)
    want = exact.product(a, b)
    for dtype, shift, beside in ((torch.float32, 0, 0), (torch.bfloat16, 3, 0), (torch.float16, 1, 5)):
        y, alone = call(lib, a, b, dtype, sms, shift=shift, beside=beside)
        assert torch.equal(y, want.to(dtype)) and alone
        if t * n * k > 3e7:
            break
    assert lib.emu_product_errors() == 0


@pytest.mark.parametrize("size,sms", [((5, 40, 1900), 1), ((3, 100, 2400), 8), ((40, 130, 300), 1), ((300, 260, 100), 2)])
def test_dropout_of_results(lib, size, sms):
    t, n, k = size
    a, b = exact.matrix(t, k, 3), exact.matrix(n, k, 4)
    y, _ = call(lib, a, b, torch.float32, sms, p=0.25, seed=11)
    assert torch.equal(y, ref.dropped(exact.product(a, b).float(), 0.25, 11).float())


@pytest.mark.parametrize("dtype", list(KIND))
@pytest.mark.parametrize("size,sms", [((1, 40, 1), 2), ((1, 130, 4096), 1), ((5, 100, 2400), 8), ((16, 300, 2048), 1), ((7, 130, 999), 2)])
def test_rounding_inside(lib, size, sms, dtype):
    t, n, k = size
    g = torch.Generator().manual_seed(1)
    x, b = torch.randn(t, k, generator=g).to(dtype), exact.matrix(n, k, 2)
    # (rounded values times a power of two for each row stay within what float32 sums exactly)
    x = (exact.matrix(t, k, 5) + 0.01 * x.float()).to(dtype)
    want = exact.product(ref.values(x).float(), b)
    y, _ = call(lib, None, b, torch.float32, sms, x=x)
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("size,sms", [((4, 60, 300), 1), ((260, 140, 300), 2)])
def test_nan_stays_in_its_rows(lib, size, sms):
    t, n, k = size
    a, b = exact.matrix(t, k, 1), exact.matrix(n, k, 2)
    want = exact.product(a, b).float()
    a[1, 40], b[3, k - 1] = float("nan"), float("inf")
    y, _ = call(lib, a, b, torch.float32, sms)
    want[1], want[:, 3] = float("nan"), float("nan")
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(0.5), want.nan_to_num(0.5))


# ((t, n, k), SMs, the rank that loses its copies, from which one on)
LATE = [
    ((5, 200, 600), 1, 0, 0),        # no cluster: nothing arrives
    ((5, 200, 600), 1, 0, 4),        # the second panel does not
    ((100, 130, 1800), 1, 0, 24),    # after the stages went round
    ((3, 100, 2400), 8, 5, 0),       # one rank of a cluster of 8
    ((40, 100, 1300), 2, 0, 4),      # of 2
    ((260, 120, 2400), 4, 1, 8),
    ((300, 520, 700), 2, 0, 0),      # a pair, either CTA: from its first tile on
    ((300, 520, 700), 2, 1, 0),
    ((300, 520, 700), 2, 1, 12),     # from its second one
    ((300, 520, 700), 2, 0, 42),     # in the middle of its fourth
]


@pytest.mark.parametrize("size,sms,rank,first", LATE)
def test_sums_that_are_not_complete_are_nan(lib, size, sms, rank, first):
    """Copies that never arrive: the waits end, each result is right or NaN, and
    what depends on the lost copies is NaN; none is left unwritten."""
    t, n, k = size
    a, b = exact.matrix(t, k, 1), exact.matrix(n, k, 2)
    want = exact.product(a, b)
    assert lib.emu_product_errors() == 0
    lib.emu_product_lose(rank, first, 0.02)
    try:
        y, alone = call(lib, a, b, torch.float32, sms, shift=1)
    finally:
        lib.emu_product_lose(-1, 0, 0.0)
    assert alone and lib.emu_product_errors() > 0 and lib.emu_product_errors() == 0
    assert (y.isnan() | (y.double() == want)).all()
    whole = 0   # tiles of 256 x 256, row by row, whose copies all arrived (a pair's panel is 4 copies)
    if t > 128 and n > 128:
        whole = first // (4 * -(-k // 256))
    for i, (r, c) in enumerate((r, c) for r in range(0, t, 256) for c in range(0, n, 256)):
        tile = y[r:r + 256, c:c + 256]
        assert i < whole or tile.isnan().all()
    y, _ = call(lib, a, b, torch.float32, sms)   # and the next call is as ever
    assert torch.equal(y.double(), want) and lib.emu_product_errors() == 0


def test_rounding_inside_with_late_copies(lib):
    b = exact.matrix(40, 600, 2)
    lib.emu_product_lose(0, 2, 0.02)
    try:
        y, _ = call(lib, None, b, torch.bfloat16, 1, x=exact.matrix(3, 600, 1))
    finally:
        lib.emu_product_lose(-1, 0, 0.0)
    assert y.isnan().all() and lib.emu_product_errors() > 0


def test_errors_are_reported_once():
    """falcom_mx4_errors: what gave up since the last call that said so."""
    from tests.emu import build_mx4
    lib = ctypes.CDLL(build_mx4.build())
    abi.bind_mx4(lib)
    count = ctypes.c_uint32.in_dll(lib, "emu_mx4_gave_up")
    start = count.value
    assert lib.falcom_mx4_errors() == 0
    for more in (1, 5, 2 ** 31 - 1, 2 ** 31 - 1, 3):   # (the count may go round)
        count.value += more
        assert lib.falcom_mx4_errors() == 1 and lib.falcom_mx4_errors() == 0
    assert count.value != start
    count.value = 0   # a device that was reset counts anew
    assert lib.falcom_mx4_errors() == 0
    count.value = 1
    assert lib.falcom_mx4_errors() == 1 and lib.falcom_mx4_errors() == 0
