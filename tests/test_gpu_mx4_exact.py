"""GPU tests of the 4-bit product without a tolerance: values whose sums float32
holds in any order, so that a missing or doubled term of the longest sum shows.
Sizes by what they reach on 148 SMs: more panels for a CTA than it has stages, at
every width; more CTAs than SMs; clusters; pairs with many tiles.  And the forms
of the C calls that nothing in Python makes."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from compressor_b200 import abi  # noqa: E402
from tests import mx4_exact as exact  # noqa: E402
from tests import mx4_reference as ref  # noqa: E402
from tests.test_gpu_mx4 import wild  # noqa: E402


@pytest.fixture(scope="module")
def mx4(product_lib):
    from compressor_b200 import mx4
    return mx4


SIZES = [
    (1, 50257, 1024), (8, 20000, 4096), (16, 70000, 2500),                   # 16 rows a tile
    (24, 20000, 4096), (32, 300, 20000),                                     # 32
    (64, 20000, 2048), (40, 50257, 1500),                                    # 64
    (100, 40000, 1024), (128, 20000, 4096), (77, 10, 9000),                  # 128
    (20000, 100, 4096), (40000, 100, 2048), (80001, 33, 700), (300, 90, 50257),   # 256
    (2048, 4096, 64), (1500, 5001, 300), (300, 20010, 256), (4099, 1024, 50257), (513, 9001, 8192),   # pairs
]


@pytest.mark.parametrize("t,n,k", SIZES)
def test_products_are_exact(mx4, t, n, k):
    a, b = exact.matrix(t, k, 1, "cuda"), exact.matrix(n, k, 2, "cuda")
    want = exact.product(a, b)
    p, q = mx4.quantize(a), mx4.quantize(b)
    assert torch.equal(p.dequantize(), a) and torch.equal(q.dequantize(), b)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(mx4.product(p, q, dtype=dtype), want.to(dtype)), dtype
        assert torch.equal(mx4.product(a.bfloat16(), q, dtype=dtype), want.to(dtype)), dtype   # (bfloat16 holds them too)
    assert mx4.errors() == 0


@pytest.mark.parametrize("t,n,k", [(5, 3000, 4100), (24, 20000, 4096), (100, 20000, 1500), (20000, 100, 2048), (300, 2001, 700)])
def test_dropout_of_exact_products(mx4, t, n, k):
    a, b = exact.matrix(t, k, 3, "cuda"), exact.matrix(n, k, 4, "cuda")
    y = torch.empty(t, n, device="cuda")
    drop = abi.DropoutArgsC(0.25, abi.RandomC(11, None))
    p, q = mx4.quantize(a), mx4.quantize(b)
    assert mx4._library().falcom_mx4_product(p._ref, q._ref, y.data_ptr(), abi.TYPE_F32, n, ctypes.byref(drop),
                                             torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(y.cpu(), ref.dropped(exact.product(a, b).float().cpu(), 0.25, 11).float())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 33), (129, 513), (300, 70), (256, 384)])
@pytest.mark.parametrize("random", [False, True])
@pytest.mark.parametrize("along", ["rows", "columns", "both"])
def test_rounding_after_dropout(mx4, rows, cols, dtype, random, along):
    x = wild(rows, cols, dtype, 1)
    xg = x.cuda()
    by_rows = mx4.Mx4Matrix.empty(rows, cols, "cuda") if along != "columns" else None
    by_cols = mx4.Mx4Matrix.empty(cols, rows, "cuda") if along != "rows" else None
    rnd, drop = abi.RandomC(77, None), abi.DropoutArgsC(0.3, abi.RandomC(5, None))
    assert mx4._library().falcom_mx4_quantize(
        xg.data_ptr(), mx4._TYPES[dtype], rows, cols, cols, ctypes.byref(rnd) if random else None, ctypes.byref(drop),
        by_rows._ref if by_rows else None, by_cols._ref if by_cols else None, torch.cuda.current_stream().cuda_stream) == 0
    d = ref.dropped(x, 0.3, 5).float()
    bits = ref.random_bits(ref.places(rows, cols), ref.ROUNDING, 77) if random else None
    for got, want in ((by_rows, (d, bits)), (by_cols, (d.t(), bits.t() if random else None))):
        if got is not None:
            codes, scales = ref.pack(*ref.codes(*want))
            assert torch.equal(got.codes.cpu(), codes) and torch.equal(got.scales.cpu(), scales)
