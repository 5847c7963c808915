"""The 4-bit operators on the GPU against their definition in 64 bits."""
import pytest
import torch

from tests import mx4_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def mx4():
    from compressor_b200 import mx4
    return mx4


def wild(rows, cols, dtype, seed=0):
    """Blocks of very different sizes, ties, zeros and signed zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-6, 6, (rows, -(-cols // 32)), generator=g).float()).repeat_interleave(32, 1)[:, :cols]
    flat = x.view(-1)
    flat[::5] = torch.round(flat[::5] * 8) / 8
    flat[3::17] = 0.0
    flat[4::29] = -0.0
    return x.to(dtype)


# (1, 1) to several tiles, panels and groups; sizes off every boundary
SHAPES = [(1, 1), (1, 32), (2, 33), (3, 255), (7, 256), (8, 257), (9, 31), (33, 64), (127, 130), (128, 128), (129, 513), (300, 70), (257, 1025)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("rounding", ["nearest", "random"])
def test_quantize_is_exact(mx4, rows, cols, dtype, rounding):
    x = wild(rows, cols, dtype)
    bits = ref.random_bits(ref.places(rows, cols), ref.ROUNDING, 77) if rounding == "random" else None
    q, t = mx4.quantize(x.cuda(), along="both", rounding=rounding, seed=77)
    for got, want in ((q, ref.codes(x, bits)), (t, ref.codes(x.t(), bits.t() if bits is not None else None))):
        codes, scales = ref.pack(*want)
        assert torch.equal(got.codes.cpu(), codes) and torch.equal(got.scales.cpu(), scales)
    one, other = (mx4.quantize(x.cuda(), along=a, rounding=rounding, seed=77) for a in ("rows", "columns"))
    assert torch.equal(one.codes, q.codes) and torch.equal(one.scales, q.scales)
    assert torch.equal(other.codes, t.codes) and torch.equal(other.scales, t.scales)
    assert torch.equal(q.dequantize().cpu().double(), ref.values(x, bits))
    assert torch.equal(t.dequantize(dtype).cpu(), ref.values(x.t(), bits.t() if bits is not None else None).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n,k", [(1, 1, 1), (1, 130, 64), (2, 128, 65), (16, 384, 512), (17, 100, 1000), (33, 300, 96),
                                   (64, 129, 257), (65, 128, 300), (128, 1, 2048), (129, 257, 513), (256, 256, 1024), (300, 1000, 2048), (5, 40, 8192)])
def test_product(mx4, t, n, k, dtype):
    a, b = mx4.quantize(wild(t, k, torch.float32, 1).cuda()), mx4.quantize(wild(n, k, torch.float32, 2).cuda())
    y = mx4.product(a, b, dtype=dtype)
    u, v = a.dequantize().cpu().double(), b.dequantize().cpu().double()
    assert y.dtype == dtype and y.shape == (t, n)
    finite = (u @ v.t()).abs() < torch.finfo(dtype).max / 2
    assert ((y.cpu().double() - u @ v.t()).abs() <= ref.sum_bound(u, v, dtype))[finite].all()
    assert torch.equal(y, mx4.product(a, b, dtype=dtype)) and mx4.errors() == 0


# enough tiles for every SM to take several, rows of `out` at all offsets from 16 bytes, sums of one and of many panels
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n,k", [(2048, 4096, 64), (1500, 5001, 300), (4099, 2051, 1025), (300, 20010, 256), (257, 19000, 2048),
                                   (129, 20001, 300), (20001, 129, 257), (10007, 300, 64), (5000, 2304, 100)])
def test_product_of_many_tiles(mx4, t, n, k, dtype):
    a, b = mx4.quantize(wild(t, k, torch.float32, 1).cuda()), mx4.quantize(wild(n, k, torch.float32, 2).cuda())
    room = torch.full((t * n + 64,), 7.0, dtype=dtype, device="cuda")
    y = mx4.product(a, b, out=room[13:13 + t * n].view(t, n))
    u, v = a.dequantize().double(), b.dequantize().double()
    want = u @ v.t()
    finite = want.abs() < torch.finfo(dtype).max / 2
    assert ((y.double() - want).abs() <= ref.sum_bound(u, v, dtype))[finite].all()
    assert (room[:13] == 7).all() and (room[13 + t * n:] == 7).all() and mx4.errors() == 0
    assert torch.equal(y, mx4.product(a, b, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("t,k,n", [(1, 32, 8), (77, 513, 10), (130, 96, 257)])
def test_linear_and_its_gradients(mx4, t, k, n, p, dtype):
    x, w, dy = wild(t, k, dtype, 3) / 8, wild(n, k, torch.float32, 4) / 64, wild(t, n, dtype, 5) / 64
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = mx4.linear(xg, wg, p=p, seed=9)
    dx, dw = torch.autograd.grad(y, (xg, wg), dy.cuda())
    d = ref.dropped(x, p, 9)
    bits = ref.random_bits(ref.places(t, n), ref.ROUNDING, 9)
    parts = {"y": (y, ref.values(d), ref.values(w)),
             "dx": (dx, ref.values(dy, bits), ref.values(w.t())),
             "dw": (dw, ref.values(dy.t(), bits.t()), ref.values(d.t()))}
    for name, (got, a, b) in parts.items():
        want, bound = a @ b.t(), ref.sum_bound(a, b, got.dtype)
        if name == "dx":   # dropout of the sum, times a factor rounded to float32 (two roundings)
            factor = (ref.dropped(torch.ones(t, k), p, 9))
            want, bound = want * factor, (bound + 2.0 ** -23 * want.abs()) * 2
        assert ((got.detach().cpu().double() - want).abs() <= bound).all(), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 31, 32, 33, 255, 256, 257, 5130, 70001])
@pytest.mark.parametrize("rounding", ["nearest", "random"])
@pytest.mark.parametrize("shift", [0, 1])
def test_encode_and_decode(mx4, n, dtype, rounding, shift):
    x, base, out = wild(1, n + shift, dtype, 6)[0], wild(1, n + shift, torch.float32, 7)[0], wild(1, n + shift, dtype, 8)[0]
    xg, bg, og = (t.cuda()[shift:] for t in (x, base, out))
    x, base, out = (t[shift:] for t in (x, base, out))
    bits = ref.random_bits(ref.places(1, n), ref.ROUNDING, 11, 5) if rounding == "random" else None
    counter = torch.tensor([5], device="cuda")
    sent = mx4.encode(xg, base=bg, rounding=rounding, seed=11, counter=counter)
    change = x.float() - base
    v = ref.values(change[None], bits)[0]
    assert torch.equal(sent.decode().cpu().double(), v)
    assert torch.equal(bg.cpu(), base + v.float())
    mx4.decode(sent, out=og, weight=0.3, accumulate=True)
    assert torch.equal(og.cpu(), (out.float() + torch.tensor(0.3) * v.float()).to(dtype))
    alone = mx4.encode(xg, rounding=rounding, seed=11, counter=counter)
    assert torch.equal(alone.decode().cpu().double(), ref.values(x[None], bits)[0])


# rounded inside the product (few rows and columns) or before it: the same bits either way
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n,k", [(1, 1, 1), (1, 50257, 1024), (3, 200, 31), (4, 1024, 4096), (5, 129, 300), (16, 384, 1024), (16, 130, 1025), (16, 200, 2049), (8, 20000, 4096),
                                   (17, 130, 64), (1, 300, 4097), (2, 70, 8191)])
def test_product_of_a_tensor(mx4, t, n, k, dtype):
    b = mx4.quantize(wild(n, k, torch.float32, 2).cuda())
    whole = wild(t, k + 3, dtype, 1).cuda()
    if t > 2:
        whole[1, k // 2] = float("nan")
    for x in (whole[:, 3:], whole[:, :k].contiguous(), whole[:, 1:k + 1]):
        for out in TYPES:
            y = mx4.product(x, b, dtype=out)
            assert torch.equal(y.nan_to_num(7.5), mx4.product(mx4.quantize(x), b, dtype=out).nan_to_num(7.5))
    assert y.isnan().any().item() == (t > 2) and mx4.errors() == 0
