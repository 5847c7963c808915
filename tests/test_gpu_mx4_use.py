"""GPU tests of what surrounds the 4-bit operators and dropout: values that
are not finite, strides, empty sizes, streams, graphs, autograd, refusals, and
a whole round on them."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from tests import mx4_reference as ref  # noqa: E402
from tests.test_gpu_mx4 import wild  # noqa: E402


@pytest.fixture(scope="module")
def mx4(product_lib):
    from compressor_b200 import mx4
    return mx4


@pytest.fixture(scope="module")
def dropout(product_lib):
    from compressor_b200.dropout import dropout
    return dropout


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rounding", ["nearest", "random"])
def test_infinities_and_nan_stay_in_their_blocks(mx4, dtype, rounding):
    x = wild(70, 300, dtype, 1)
    x[3, 40], x[9, 0], x[9, 299], x[64, 64] = float("nan"), float("inf"), float("-inf"), float("nan")
    bits = ref.random_bits(ref.places(70, 300), ref.ROUNDING, 1) if rounding == "random" else None
    q, t = mx4.quantize(x.cuda(), along="both", rounding=rounding, seed=1)
    for got, want in ((q, ref.codes(x, bits)), (t, ref.codes(x.t(), bits.t() if bits is not None else None))):
        codes, scales = ref.pack(*want)
        assert torch.equal(got.codes.cpu(), codes) and torch.equal(got.scales.cpu(), scales)
    v = q.dequantize().cpu().double()
    assert torch.equal(v.isnan(), ref.values(x, bits).isnan()) and v.isnan().sum() == 32 + 32 + 12 + 32
    w = wild(40, 300, torch.float32, 2)
    w[5, 299] = float("nan")
    y = mx4.product(q, mx4.quantize(w.cuda()), dtype=torch.float32).cpu()
    bad = torch.zeros(70, 40, dtype=torch.bool)
    bad[[3, 9, 64]] = True
    bad[:, 5] = True
    assert torch.equal(y.isnan(), bad)
    sent = mx4.encode(x.cuda().view(-1), rounding=rounding, seed=1)
    flat = x.view(1, -1)
    assert torch.equal(sent.decode().cpu().isnan(), ref.values(flat)[0].isnan())


def test_extremes_of_float32(mx4):
    """The largest and smallest numbers; blocks of zeros of both signs."""
    big, tiny = 3.4028234663852886e38, 2.0 ** -149
    x = torch.zeros(6, 64)
    x[0, :4] = torch.tensor([big, -big, big / 3, 1.0])
    x[1, :4] = torch.tensor([tiny, -tiny, 2.0 ** -126, 2.0 ** -128])
    x[2, :4] = torch.tensor([2.0 ** -127 * 6, 2.0 ** -128, 2.0 ** -129, -(2.0 ** -127)])
    x[3] = -0.0
    x[4, :3] = torch.tensor([6.0, 2.0 ** -126, -(2.0 ** -140)])
    for rounding in ("nearest", "random"):
        bits = ref.random_bits(ref.places(6, 64), ref.ROUNDING, 2) if rounding == "random" else None
        q, t = mx4.quantize(x.cuda(), along="both", rounding=rounding, seed=2)
        for got, want in ((q, ref.codes(x, bits)), (t, ref.codes(x.t(), bits.t() if bits is not None else None))):
            codes, scales = ref.pack(*want)
            assert torch.equal(got.codes.cpu(), codes) and torch.equal(got.scales.cpu(), scales)
        # (the largest number's neighbour 4 * 2^126 is above float32's range: read back in that type it is infinity)
        assert torch.equal(q.dequantize().cpu(), ref.values(x, bits).float())
        flat = ref.values(x.view(1, -1), ref.random_bits(ref.places(1, 384), ref.ROUNDING, 2) if bits is not None else None)[0]
        assert torch.equal(mx4.encode(x.cuda(), rounding=rounding, seed=2).decode().cpu(), flat.float())


def test_views_of_larger_tensors(mx4, dropout):
    """Rows of a wider tensor at any offset, transposed and expanded ones:
    what lies beside them is neither read into the result nor written."""
    whole = wild(300, 500, torch.bfloat16, 3).cuda()
    for x in (whole[:, 7:407], whole[3:290, 1:], whole[::2, 130:], whole.t()[5:300], whole[:1, 3:90], whole[:, 4:5],
              whole[2].expand(130, 500), whole.view(30, 10, 500)[:, :, 8:264], whole[5:5], whole[:, 5:5]):
        flat = x.reshape(-1, x.shape[-1]) if x.numel() else x.reshape(x.shape[0], x.shape[-1])
        q, t = mx4.quantize(x, along="both", rounding="random", seed=4)
        p, s = mx4.quantize(flat.contiguous(), along="both", rounding="random", seed=4)
        for a, b in ((q, p), (t, s)):
            assert a.shape == b.shape and torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        assert torch.equal(dropout(x, 0.4, seed=4), dropout(x.contiguous(), 0.4, seed=4))
    y = wild(4, 64, torch.float32, 1).cuda()
    w = mx4.quantize(wild(130, 64, torch.float32, 2).cuda())
    room = torch.full((6, 130), 5.0, device="cuda")
    mx4.product(y, w, out=room[1:5])
    assert torch.equal(room[1:5], mx4.product(y, w, dtype=torch.float32)) and (room[[0, 5]] == 5).all()
    assert mx4.product(y.view(2, 2, 64), w).shape == (2, 2, 130)


def test_empty_and_single_sizes(mx4, dropout):
    e = torch.empty
    for t, k, n in [(0, 5, 3), (4, 0, 3), (4, 5, 0), (0, 0, 0), (1, 1, 1)]:
        x, w = e(t, k, device="cuda").normal_().requires_grad_(), e(n, k, device="cuda").normal_().requires_grad_()
        y = mx4.linear(x, w, p=0.5, seed=1)
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert y.shape == (t, n) and dx.shape == (t, k) and dw.shape == (n, k)
        if k == 0:
            assert (y == 0).all()
        if t == 0:
            assert (dw == 0).all()
        if n == 0:
            assert (dx == 0).all()
        q = mx4.quantize(w.detach())
        assert q.shape == (n, k) and q.dequantize().shape == (n, k)
        assert torch.equal(mx4.product(x.detach(), q, dtype=torch.float32), torch.zeros(t, n, device="cuda")) or k
        d = dropout(x, 0.5, seed=1, residual=x)
        assert d.shape == x.shape
    v = mx4.encode(e(0, device="cuda"))
    assert v.n == 0 and v.decode().shape == (0,)
    s = torch.tensor(3.0, device="cuda")
    assert dropout(s, 0.5, seed=1).shape == () and float(dropout(s, 0.5, seed=1)) in (0.0, 6.0)
    assert dropout(s, 0.0) is s
    with pytest.raises(ValueError, match="dimensions"):
        mx4.quantize(s)


def test_linear_needs_only_what_is_asked_for(mx4):
    x, w = wild(40, 96, torch.bfloat16, 1).cuda(), wild(24, 96, torch.bfloat16, 2).cuda()
    dy = wild(40, 24, torch.bfloat16, 3).cuda()
    both = mx4.linear(x.clone().requires_grad_(), w.clone().requires_grad_(), p=0.25, seed=3)
    plain = mx4.linear(x, w, p=0.25, seed=3)
    assert torch.equal(plain, both) and not plain.requires_grad
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    full = torch.autograd.grad(mx4.linear(xg, wg, p=0.25, seed=3), (xg, wg), dy)
    assert torch.equal(torch.autograd.grad(mx4.linear(xg, w, p=0.25, seed=3), xg, dy)[0], full[0])
    assert torch.equal(torch.autograd.grad(mx4.linear(x, wg, p=0.25, seed=3), wg, dy)[0], full[1])
    y = mx4.linear(xg, wg, p=0.25, seed=3)
    y.backward(dy)
    assert torch.equal(xg.grad, full[0]) and torch.equal(wg.grad, full[1])
    # an expanded gradient, as of a sum
    a = torch.autograd.grad(mx4.linear(xg, wg, seed=3).sum(), (xg, wg))
    b = torch.autograd.grad(mx4.linear(xg, wg, seed=3), (xg, wg), torch.ones_like(dy))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    with pytest.raises(RuntimeError):   # no gradient of the gradient
        g = torch.autograd.grad(mx4.linear(xg, wg, seed=3), xg, dy, create_graph=True)[0]
        g.sum().backward()
    # three dimensions, and the composition from its parts
    x3 = x.view(4, 10, 96)
    assert torch.equal(mx4.linear(x3, w, p=0.25, seed=3), plain.view(4, 10, 24))
    assert torch.equal(mx4.linear(x, w), mx4.product(x, mx4.quantize(w), dtype=torch.bfloat16))


def test_gradient_against_differences(mx4):
    """Values that 4 bits hold make the layer linear: its gradients are then
    the slopes of its sum."""
    g = torch.Generator().manual_seed(0)
    pick = lambda *s: ref.VALUES[torch.randint(0, 8, s, generator=g)].float() * (torch.randint(0, 2, s, generator=g) * 2 - 1)  # noqa: E731
    x, w, dy = pick(6, 32), pick(5, 32), pick(6, 5)
    for m in (x, w, dy):
        m[0, 0] = 6.0
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    dx, dw = torch.autograd.grad(mx4.linear(xg, wg, seed=1), (xg, wg), dy.cuda())
    f = lambda x, w: float((mx4.linear(x.cuda(), w.cuda(), seed=1).cpu().double() * dy).sum())  # noqa: E731
    # rows of dy and of w^T are blocks of their own there: compare with the parts that stay exact
    want_dx = ref.values(dy, ref.random_bits(ref.places(6, 5), ref.ROUNDING, 1)) @ ref.values(w.t()).t()
    assert torch.equal(dx.cpu().double(), want_dx)
    for i, k in [(1, 3), (4, 30)]:
        up, down = x.clone(), x.clone()
        up[i, k], down[i, k] = 4.0, 2.0
        assert (f(up, w) - f(down, w)) / 2 == float((dy.double() @ w.double())[i, k])
    assert torch.equal(dw.cpu().double(), ref.values(dy.t(), ref.random_bits(ref.places(6, 5), ref.ROUNDING, 1).t()) @ ref.values(x.t()).t())


def test_dropout_derivatives_and_masks(dropout):
    x = wild(33, 65, torch.float32, 1).cuda().requires_grad_()
    y = dropout(x, 0.3, seed=7)
    kept = y != 0
    g, = torch.autograd.grad(y.pow(2).sum(), x, create_graph=True)
    factor = 65536 / (65536 - ref.threshold(0.3))
    assert torch.equal(g != 0, kept & (x != 0))
    gg, = torch.autograd.grad(g.sum(), x)
    assert torch.allclose(gg, 2 * factor ** 2 * kept_mask(33, 65, 0.3, 7).cuda(), rtol=1e-6)
    # what is dropped is 0, whatever it was, and so is its gradient
    bad = torch.full((8, 64), float("nan"), device="cuda", requires_grad=True)
    y = dropout(bad, 0.5, seed=1)
    mask = kept_mask(8, 64, 0.5, 1).cuda()
    assert torch.equal(y.isnan(), mask.bool()) and (y[~mask.bool()] == 0).all()
    g, = torch.autograd.grad(y, bad, torch.full_like(y, float("inf")))
    assert torch.equal(g.isinf(), mask.bool()) and (g[~mask.bool()] == 0).all()
    # a share of p, other masks for other seeds (10^6 draws: five standard deviations)
    one = torch.ones(1000, 1000, device="cuda")
    a, b = dropout(one, 0.1, seed=1) == 0, dropout(one, 0.1, seed=2) == 0
    assert abs(a.float().mean().item() - 0.1) < 5 * (0.09 / 1e6) ** 0.5
    assert abs((a & b).float().mean().item() - 0.01) < 5 * (0.01 / 1e6) ** 0.5


def kept_mask(rows, cols, p, seed, counter=0):
    return (ref.random_bits(ref.places(rows, cols), ref.DROPOUT, seed, counter) >= ref.threshold(p)).float()


def test_dropout_in_place_and_refusals(mx4, dropout, product_lib):
    import ctypes
    from compressor_b200 import abi
    lib = mx4._library()
    x, r = wild(9, 64, torch.float32, 1).cuda(), wild(9, 64, torch.float32, 2).cuda()
    args = abi.DropoutArgsC(0.5, abi.RandomC(3, None))
    want = dropout(x, 0.5, seed=3, residual=r)
    s = torch.cuda.current_stream().cuda_stream
    a, b = x.clone(), r.clone()
    assert lib.falcom_dropout(a.data_ptr(), r.data_ptr(), a.data_ptr(), 0, 9, 64, ctypes.byref(args), s) == 0
    assert lib.falcom_dropout(x.data_ptr(), b.data_ptr(), b.data_ptr(), 0, 9, 64, ctypes.byref(args), s) == 0
    assert torch.equal(a, want) and torch.equal(b, want)
    # shifted by part of itself
    assert lib.falcom_dropout(a.data_ptr(), None, a.data_ptr() + 4, 0, 1, 64, ctypes.byref(args), s) == abi.ERROR_INVALID_PARAM
    q = mx4.quantize(x)
    with pytest.raises(RuntimeError):
        mx4.product(x, q, out=x.view(-1)[:81].view(9, 9))
    host = torch.zeros(9, 64)
    assert lib.falcom_dropout(host.data_ptr(), None, a.data_ptr(), 0, 9, 64, ctypes.byref(args), s) == abi.ERROR_INVALID_PARAM
    assert lib.falcom_mx4_encode(a.data_ptr() + 2, 0, 8, None, None, q.buffer.data_ptr(), q.buffer.data_ptr() + 1024, s) \
        == abi.ERROR_INVALID_PARAM
    for call in (lambda: mx4.product(x[:, :32], q), lambda: mx4.encode(x.t()), lambda: mx4.encode(x, base=x.bfloat16()),
                 lambda: mx4.decode(mx4.encode(x), out=x[:, :3]), lambda: mx4.linear(x, x[:, :5]),
                 lambda: dropout(x, 0.5, residual=r.bfloat16()), lambda: dropout(x, 0.5, counter=torch.zeros(1, device="cuda")),
                 lambda: mx4.product(x, q, dtype=torch.int8), lambda: mx4.decode(mx4.encode(x), weight=float("inf")) and None):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("t,k,n", [(9, 70, 33), (700, 130, 20001)])
def test_dropout_inside_rounding_and_product(mx4, p, t, k, n):
    """The C calls' own dropout: the same as before the rounding, or after the
    product, in the few-rows and the many-tiles form."""
    import ctypes
    from compressor_b200 import abi
    lib, r, s = mx4._library(), ctypes.byref, torch.cuda.current_stream().cuda_stream
    drop = abi.DropoutArgsC(p, abi.RandomC(5, None))
    x = wild(t, k, torch.float32, 1)
    rows, cols = mx4.Mx4Matrix.empty(t, k, "cuda"), mx4.Mx4Matrix.empty(k, t, "cuda")
    assert lib.falcom_mx4_quantize(x.cuda().data_ptr(), 0, t, k, k, None, r(drop), rows._ref, cols._ref, s) == 0
    d = ref.dropped(x, p, 5).float().cuda()
    want = mx4.quantize(d, along="both")
    assert torch.equal(rows.buffer, want[0].buffer) and torch.equal(cols.buffer, want[1].buffer)
    b = mx4.quantize(wild(n, k, torch.float32, 2).cuda())
    y = torch.empty(t, n, device="cuda")
    assert lib.falcom_mx4_product(rows._ref, b._ref, y.data_ptr(), 0, n, r(drop), s) == 0
    plain = mx4.product(rows, b, dtype=torch.float32).cpu()
    assert torch.equal(y.cpu(), ref.dropped(plain, p, 5).float())


def test_two_streams_give_the_same_bits(mx4, dropout):
    """Calls in flight at the same time share nothing."""
    x, w = wild(2050, 1030, torch.bfloat16, 1).cuda(), wild(4100, 1030, torch.float32, 2).cuda()

    def work():
        q, t = mx4.quantize(x, along="both", rounding="random", seed=1)
        b = mx4.quantize(w)
        return [t.codes, t.scales, mx4.product(q, b), mx4.product(x[:3], b), dropout(x, 0.2, seed=5), mx4.encode(x, rounding="random").buffer[:100]]

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    assert mx4.errors() == 0


def test_captured_steps_follow_the_counter(mx4, dropout):
    """Forward and backward in one graph: each replay has the counter's bits,
    and those of the eager call with that counter."""
    x, w = wild(70, 130, torch.bfloat16, 1).cuda().requires_grad_(), wild(48, 130, torch.float32, 2).cuda().requires_grad_()
    dy = wild(70, 48, torch.bfloat16, 3).cuda()
    counter = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        h = dropout(x, 0.25, seed=2, counter=counter, residual=x)
        y = mx4.linear(h, w, p=0.25, seed=3, counter=counter)
        counter.add_(1)                      # before the gradients are asked for
        return (y, *torch.autograd.grad(y, (x, w), dy))

    eager = []
    for c in range(3):
        counter.fill_(c)
        eager.append([t.detach().clone() for t in step()])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    counter.zero_()
    for c in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert int(counter) == c + 1
        assert all(torch.equal(a, b) for a, b in zip(out, eager[c])), c
    assert not torch.equal(eager[0][1], eager[1][1])


def test_positions_past_32_bits(mx4, dropout):
    """A vector of more than 2^33 elements: the words of the pairs above 2^32."""
    n = (1 << 33) + 1000
    x = torch.zeros(n, dtype=torch.float16, device="cuda")
    tail = wild(1, 1000 + 64, torch.float16, 4)[0]
    x[-1064:] = tail.cuda()
    at = torch.arange(n - 1064, n)
    sent = mx4.encode(x, rounding="random", seed=6)
    got = torch.empty(n, dtype=torch.float16, device="cuda")
    mx4.decode(sent, out=got)
    bits = ref.random_bits(at, ref.ROUNDING, 6)[None]
    assert torch.equal(got[-1064:].cpu(), ref.values(tail[None], bits)[0].half())   # (n - 1064 is a multiple of 32)
    assert not got[:-1064].any()
    del got
    y = dropout(x.view(1, -1), 0.5, seed=6)
    keep = ref.random_bits(at, ref.DROPOUT, 6) >= ref.threshold(0.5)
    assert torch.equal(y[0, -1064:].cpu(), torch.where(keep, tail * 2, torch.zeros_like(tail)))
    # rows that lie more than 2^32 bytes apart
    del y
    far = x.view(-1)[:3 * (1 << 31)].view(3, 1 << 31)[:, (1 << 31) - 300:]
    far.copy_(wild(3, 300, torch.float16, 5).cuda())
    q, p = mx4.quantize(far), mx4.quantize(far.contiguous())
    assert torch.equal(q.buffer, p.buffer)


def test_a_round_down_and_up(mx4, dropout, product_lib):
    """Server and client as they work together: the server steps and sends its
    model in 4 bits, the client brings its copy forward, trains a layer in 4
    bits with dropout, clips and steps, and its update goes through the codec
    into the server's aggregate."""
    import numpy as np
    from compressor_b200 import federated as fed
    from compressor_b200.abi import Codec
    from compressor_b200.optim import AdamW, GradNorm
    shapes = [("fc1.weight", (192, 96)), ("fc2.weight", (33, 192))]
    names = [n for n, _ in shapes]
    layout = fed.AggregateLayout.of(names, [s for _, s in shapes], align=64)
    spans = {n: (o, o + int(np.prod(s)), s) for (n, s), o in zip(shapes, layout.offsets)}
    gen = torch.Generator("cuda").manual_seed(0)
    weights = torch.randn(layout.total, device="cuda", generator=gen) * 0.05
    mine = weights.clone()
    aggregate = torch.zeros_like(weights)
    server = fed.ServerAdamW(layout, weights, aggregate, lr=1e-2, max_norm=1.0)
    down = fed.Downlink(weights, rounding="random", seed=8)
    enc, dec = Codec(product_lib, client="c0", param_count_threshold=16), Codec(product_lib, client="server", param_count_threshold=16)
    x = torch.randn(50, 96, device="cuda", generator=gen, dtype=torch.bfloat16)
    for t in range(3):
        before, old = weights.clone(), mine.clone()
        sent = down.send()
        fed.broadcast(sent, None)
        assert fed.Downlink.receive(sent, mine) is mine
        assert torch.equal(mine, down.held) and torch.equal(weights, before)
        # within a rounding of the server: two 4-bit neighbours are at most 2 scales apart, a scale is under a third of
        # the largest difference (and the sums are rounded to float32: half a step of values below 1)
        assert (mine - weights).abs().max() <= (2 / 3) * (weights - old).abs().max() + 2.0 ** -25
        start = mine.clone()
        ps = {n: mine[a:b].view(s).clone().requires_grad_() for n, (a, b, s) in spans.items()}
        h = mx4.linear(x, ps["fc1.weight"], seed=10 * t)
        h = dropout(torch.relu(h), 0.1, seed=10 * t + 1)
        y = mx4.linear(h, ps["fc2.weight"], p=0.1, seed=10 * t + 2)
        loss = (y.float() ** 2).mean()
        loss.backward()
        grads = [p.grad for p in ps.values()]
        assert all(g.isfinite().all() and g.abs().max() > 0 for g in grads)
        opt = AdamW([p for p in ps.values()], grads, lr=1e-3)
        opt.step(clip=GradNorm(grads)(max_norm=1.0))
        update = {n: (p.detach() - start[spans[n][0]:spans[n][1]].view(p.shape)).cpu().numpy() for n, p in ps.items()}
        ret, layers, errs = enc.compress_batch(names, [update[n] for n in names])
        assert ret == 0, errs
        fed.set_client_weight(dec.lib, dec.h, aggregate.data_ptr(), layout.c_offsets(), len(names), 1.0)
        fed.set_aggregate_store(dec.lib, dec.h, True)
        assert dec.decompress_batch(names, layers, client="c0")[0] == 0
        server.step()
        assert not torch.equal(weights, before)
    torch.cuda.synchronize()
    assert server.errors() == 0 and mx4.errors() == 0
    # nothing is lost on the way: with rounding to the nearest a few more sends bring the copy close
    near = fed.Downlink(weights, held=down.held)
    gaps = []
    for _ in range(4):
        fed.Downlink.receive(near.send(), mine)
        gaps.append(float((mine - weights).abs().max()))
    assert gaps[-1] < gaps[0] / 20   # each leaves a third at most of a block's largest difference, and 3^3 = 27
    for o in (server, enc, dec):
        o.close()
