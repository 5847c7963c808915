"""GPU tests of the optimiser operators (falcom_norm_*, falcom_adamw_*, and
compressor_b200.optim on top of them) against plain 64-bit formulas; the
checks and their tolerances are in tests/optim_cases.py."""
import ctypes
import math

import numpy as np
import pytest

from compressor_b200 import abi
from tests import optim_cases as oc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class Gpu:
    class Mem:
        def __init__(self, raw):
            self.t = torch.from_numpy(raw).cuda()
            self.ptr = self.t.data_ptr()

    def __init__(self, path):
        self.lib = ctypes.CDLL(path)
        abi.bind_optim(self.lib)

    @property
    def stream(self):
        return torch.cuda.current_stream().cuda_stream

    def upload(self, raw):
        return Gpu.Mem(raw)

    def download(self, h):
        torch.cuda.synchronize()
        return h.t.cpu().numpy()

    def sync(self):
        torch.cuda.synchronize()


@pytest.fixture(scope="module")
def gpu(product_lib):
    return Gpu(product_lib)


@pytest.fixture(scope="module")
def optim(product_lib):
    from compressor_b200 import optim
    return optim


# ------------------------------------------------------------- C entry points
@pytest.mark.parametrize("name", list(oc.NORM_CASES))
def test_norm(gpu, name):
    ns, kinds, shifts = oc.NORM_CASES[name]
    rng = np.random.default_rng(1)
    xs = [rng.standard_normal(n) * 10.0 ** rng.integers(-4, 2) for n in ns]
    oc.check_norm(gpu, xs, kinds, shifts, scale=-0.5, max_norm=0.75)


@pytest.mark.parametrize("value", [0.0, 1e-30, 1e30, -3e38, math.inf, -math.inf, math.nan])
def test_norm_extremes(gpu, value):
    """Squares past float32's range, an exact zero, infinities and NaN in one element."""
    x = np.zeros(5000)
    x[4321] = value
    oc.check_norm(gpu, [x, x[:7]], ["f32", "f32"], [0, 1], max_norm=1.0)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pk", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("gk", ["f32", "bf16", "f16"])
def test_adamw_types(gpu, bits, pk, gk):
    oc.run_adamw(gpu, oc.case_tensors(gpu, "odd", bits, pk, gk), bits, steps=3, start=5)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("name", ["one", "units", "shifted"])
def test_adamw_shapes(gpu, bits, name):
    oc.run_adamw(gpu, oc.case_tensors(gpu, name, bits, "f32", "f32", start=False), bits, steps=4, clip=0.25,
                 grad_scale=-1.0)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("hyper", [dict(beta1=0.0), dict(beta2=0.0), dict(lr=0.0), dict(eps=1e-3),
                                   dict(seed=0), dict(seed=(1 << 64) - 1), dict(beta1=0.95, beta2=0.9999)])
def test_adamw_hyperparameters(gpu, bits, hyper):
    oc.run_adamw(gpu, oc.case_tensors(gpu, "odd", bits, "f32", "f32"), bits, steps=2, start=3, **hyper)


@pytest.mark.parametrize("start", [0, 1, 999, 10**6, 2**32 - 2, 2**40])
def test_adamw_step_numbers(gpu, start):
    for bits in (32, 8):
        oc.run_adamw(gpu, oc.case_tensors(gpu, "shifted", bits, "f32", "bf16"), bits, steps=3, start=start)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_mixed_types(gpu, bits):
    rng = np.random.default_rng(2)
    kinds = [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")]
    ts = [oc.Tensor(gpu, rng, 300 + 1000 * i, pk, gk, bits, 0.1) for i, (pk, gk) in enumerate(kinds)]
    oc.run_adamw(gpu, ts, bits, steps=3, lr_device=3e-3)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_no_tensors(gpu, bits):
    oc.run_adamw(gpu, [], bits, steps=2)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, 1e25])
def test_adamw_non_finite_gradient(gpu, bits, value):
    """One bad gradient: 32-bit states go bad at that element alone, 8-bit
    ones in its block alone; every other block steps as ever."""
    rng = np.random.default_rng(4)
    g = rng.standard_normal(1000) * 1e-3
    g[300] = value
    x = oc.Tensor(gpu, np.random.default_rng(4), 1000, "f32", "f32", bits, 0.1, g=g)
    clean = oc.Tensor(gpu, np.random.default_rng(4), 1000, "f32", "f32", bits, 0.1, g=np.where(np.arange(1000) == 300, 0, g))
    counter = [oc.Placed(gpu, np.zeros(1, np.int64)) for _ in range(2)]
    for t, c in zip((x, clean), counter):
        plan = gpu.lib.falcom_adamw_create(oc.c_array(abi.AdamWTensorC, [t.c()]), 1, bits, c.ptr)
        assert gpu.lib.falcom_adamw_step(plan, ctypes.byref(oc.make_args()), gpu.stream) == 0
        gpu.sync()
        gpu.lib.falcom_adamw_destroy(plan)
        t.refresh()
    others = np.arange(1000) != 300
    assert (x.p[others] == clean.p[others]).all()
    outside = others if bits == 32 else (np.arange(1000) // 256 != 1)
    assert (x.m[outside] == clean.m[outside]).all() and (x.v[outside] == clean.v[outside]).all()
    if bits == 32:
        assert not math.isfinite(x.v[300])
    else:
        scales = x.dvs.get()
        assert np.isnan(scales[1]) and np.isfinite(scales[[0, 2, 3]]).all()
        assert not x.dv.get()[256:512].any()


def test_adamw8_zero_and_tiny_blocks(gpu):
    """No gradient on a fresh state leaves zeros (codes, scales) and a plain
    decay; gradients below 2^-100 round the first moment's block to zero."""
    rng = np.random.default_rng(5)
    g = np.zeros(1000)
    g[600:700] = 1e-33
    oc.run_adamw(gpu, [oc.Tensor(gpu, rng, 1000, "f32", "f32", 8, 0.1, g=g, start=False)], 8, steps=2)


@pytest.mark.parametrize("bits", [32, 8])
def test_clip_skips_step(gpu, bits):
    """A NaN coefficient leaves parameters, states and the counter alone."""
    rng = np.random.default_rng(6)
    x = oc.Tensor(gpu, rng, 5000, "f32", "f32", bits, 0.1)
    before = [d.get() for d in (x.dp, x.dm, x.dv)]
    counter = oc.Placed(gpu, np.array([41], np.int64))
    clip = oc.Placed(gpu, np.array([np.inf, np.nan], np.float32))
    plan = gpu.lib.falcom_adamw_create(oc.c_array(abi.AdamWTensorC, [x.c()]), 1, bits, counter.ptr)
    assert gpu.lib.falcom_adamw_step(plan, ctypes.byref(oc.make_args(clip=clip.ptr)), gpu.stream) == 0
    assert counter.get()[0] == 41
    assert all((a == d.get()).all() for a, d in zip(before, (x.dp, x.dm, x.dv)))
    assert gpu.lib.falcom_adamw_step(plan, ctypes.byref(oc.make_args()), gpu.stream) == 0
    assert counter.get()[0] == 42
    gpu.lib.falcom_adamw_destroy(plan)


# ------------------------------------------------------------------- classes
SHAPES = [(64, 33), (64,), (3, 5, 7), (1,), (0,), (300, 1001)]


def _params(optim, bits, seed=0, dtype=torch.float32, shapes=SHAPES, **kw):
    gen = torch.Generator("cuda").manual_seed(seed)
    ps = [torch.randn(s, device="cuda", generator=gen).mul_(0.05).to(dtype) for s in shapes]
    gs = [torch.randn(s, device="cuda", generator=gen).mul_(1e-2).to(dtype) for s in shapes]
    return ps, gs, optim.AdamW(ps, gs, state_bits=bits, **kw)


def _same(a, b):
    """Equal bits."""
    ints = {1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}
    return all(torch.equal(x.contiguous().view(ints[x.element_size()]), y.contiguous().view(ints[y.element_size()]))
               for x, y in zip(a, b))


@pytest.mark.parametrize("bits", [32, 8])
def test_class_follows_torch_float64(optim, bits):
    """Ten clipped steps on changing gradients against torch's AdamW in
    float64.  With 32 bits the parameters agree within the rounding of ten
    updates; with 8 bits only the moments' rounding separates them, which
    moves an update by about the codes' spacing (12 %)."""
    ps, gs, opt = _params(optim, bits, lr=1e-2, weight_decay=0.1)
    norm = optim.GradNorm(gs)
    ref = [p.double().clone().requires_grad_() for p in ps]
    tor = torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.1)
    start = [p.clone() for p in ps]
    for i in range(10):
        gen = torch.Generator("cuda").manual_seed(100 + i)
        for g in gs:
            g.copy_(torch.randn(g.shape, device="cuda", generator=gen) * (0.1 + i))
        total = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
        for r, g in zip(ref, gs):
            r.grad = g.double() * min(1.0, 1.0 / total)
        tor.step()
        opt.step(clip=norm(max_norm=1.0))
    assert int(opt.state["step"]) == 10
    for p, r, s, mom, w in zip(ps, ref, start, opt.moments(), opt.params):
        if not p.numel():
            continue
        moved = (r.detach() - s.double()).norm()
        off = (p.double() - r.detach()).norm()
        # an update is at most a few lr; each of the ten rounds p to half a step of |p| < 1
        if bits == 32:
            assert off <= 10 * 2.0 ** -24 * (p.numel() ** 0.5) + 1e-5 * moved, off
        else:
            assert off <= 0.13 * moved, off / moved
        st = tor.state[r]
        lim = 1e-5 if bits == 32 else 0.13
        assert (mom[0].double() - st["exp_avg"]).norm() <= lim * st["exp_avg"].norm()
        assert (mom[1].double() - st["exp_avg_sq"]).norm() <= 2 * lim * st["exp_avg_sq"].norm()


@pytest.mark.parametrize("bits", [32, 8])
def test_repeatable_and_state_round_trip(optim, bits):
    """The same start gives the same bits, on one or many tensors' layout; a
    loaded state continues where the saved one stood."""
    a, ga, oa = _params(optim, bits, seed=3, dtype=torch.bfloat16)
    b, gb, ob_ = _params(optim, bits, seed=3, dtype=torch.bfloat16)
    for _ in range(3):
        oa.step(grad_scale=0.5)
        ob_.step(grad_scale=0.5)
    assert _same(a, b) and _same(oa.state.values(), ob_.state.values())
    saved = {k: v.clone() for k, v in oa.state.items()}
    c = [p.clone() for p in a]
    oc_ = optim.AdamW(c, ga, state_bits=bits)
    oc_.load_state(saved)
    for o in (oa, oc_):
        o.step(grad_scale=2.0)
    assert _same(a, c) and _same(oa.state.values(), oc_.state.values())
    other = optim.AdamW(c, ga, state_bits=40 - bits)
    with pytest.raises(ValueError):
        other.load_state(saved)
    with pytest.raises(ValueError):
        oc_.load_state({**saved, "step": saved["step"].int()})


def test_adamw8_seed_and_step_change_the_rounding(optim):
    outs = []
    for seed in (0, 1, 1 << 40):
        _, _, o = _params(optim, 8, seed=5)
        o.seed = seed
        o.step()
        outs.append(o.state["m"].view(torch.uint8).clone())
    assert not torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], outs[2])


def test_adamw8_second_moment_follows_on_average(optim):
    """sqrt(v) under a steady gradient reaches its 32-bit value on average,
    and falls again when the gradient does: 1000 steps of beta2 = 0.99, then
    300 on a tenth.  Rounding to the nearest code would stop both."""
    n = 256 * 64
    p = torch.zeros(n, device="cuda")
    g = torch.full((n,), 0.0, device="cuda")
    size = torch.exp(torch.linspace(-5, 0, 256, device="cuda")).repeat(64)
    g.copy_(size)
    opt = optim.AdamW([p], [g], state_bits=8, betas=(0.9, 0.99), weight_decay=0.0)
    for part, steps in ((1.0, 1000), (0.1, 300)):
        g.copy_(size * part)
        want = part ** 2 if part == 1.0 else 0.99 ** 300 + (1 - 0.99 ** 300) * part ** 2
        for _ in range(steps):
            opt.step()
        root = opt.moments()[0][1].sqrt() / size
        # one value's deviation stays under 30 %; the mean over 64 blocks x 256 within 3 %
        assert abs(float(root.mean()) / want ** 0.5 - 1) < 0.03, (part, float(root.mean()))


@pytest.mark.parametrize("bits", [32, 8])
def test_other_stream_device_and_memory_formats(optim, bits):
    """A step on a side stream, permuted but dense parameters, and views off
    their alignment give what plain contiguous copies give."""
    gen = torch.Generator("cuda").manual_seed(9)
    base = torch.randn(4, 6, 5, 3, device="cuda", generator=gen).contiguous(memory_format=torch.channels_last)
    flat = torch.randn(2000, device="cuda", generator=gen)
    params = [base, flat[1:1001]]
    grads = [torch.randn(4, 6, 5, 3, device="cuda", generator=gen).contiguous(memory_format=torch.channels_last),
             torch.randn(2000, device="cuda", generator=gen)[3:1003]]
    copies = [base.permute(0, 2, 3, 1).clone().contiguous(), flat[1:1001].clone()]
    cgrads = [grads[0].permute(0, 2, 3, 1).clone().contiguous(), grads[1].clone()]
    keep = flat.clone()
    oa = optim.AdamW(params, grads, state_bits=bits)
    ob_ = optim.AdamW(copies, cgrads, state_bits=bits)
    side = torch.cuda.Stream()
    na, nb = optim.GradNorm(grads), optim.GradNorm(cgrads)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            oa.step(clip=na(max_norm=0.1))
    for _ in range(3):
        ob_.step(clip=nb(max_norm=0.1))
    torch.cuda.synchronize()
    assert _same([params[0].permute(0, 2, 3, 1), params[1]], copies)
    assert _same([flat[:1], flat[1001:]], [keep[:1], keep[1001:]])
    assert _same(oa.state.values(), ob_.state.values())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays(optim, bits):
    """Norm, clip and step in one graph: replays count the steps and read the
    gradients and the learning rate of their time."""
    ps, gs, opt = _params(optim, bits, seed=11)
    qs, hs, ref = _params(optim, bits, seed=11)
    norm, rnorm = optim.GradNorm(gs), optim.GradNorm(hs)
    lr = torch.full((1,), 2.0 ** -7, device="cuda")   # powers of two: the same number in both types
    opt.step(lr=lr, clip=norm(max_norm=0.5))          # warm-up outside the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        clip = norm(max_norm=0.5)
        opt.step(lr=lr, clip=clip)
    ref.step(lr=2.0 ** -7, clip=rnorm(max_norm=0.5))
    for i in range(4):
        for g, h in zip(gs, hs):
            g.mul_(1.5)
            h.mul_(1.5)
        lr.fill_(2.0 ** (-5 - i))
        graph.replay()
        ref.step(lr=float(lr), clip=rnorm(max_norm=0.5))
    torch.cuda.synchronize()
    assert int(opt.state["step"]) == 5 and int(ref.state["step"]) == 5
    assert _same(ps, qs) and _same(opt.state.values(), ref.state.values())


def test_two_captured_norms_replay_side_by_side(optim):
    """Two graphs of one plan on two streams at once have scratch of their own."""
    gs = [torch.randn(3_000_000, device="cuda") for _ in range(2)]
    norm = optim.GradNorm(gs)
    want = norm(max_norm=1.0).clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(norm(max_norm=1.0))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(50):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    eager = []
    for s in streams:
        with torch.cuda.stream(s):
            eager += [norm(max_norm=1.0) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(_same([o], [want]) for o in outs + eager)


@pytest.mark.parametrize("bits", [32, 8])
def test_autograd_sees_the_change(optim, bits):
    """A graph that saved a parameter refuses to run backward after a step."""
    w = torch.randn(8, 8, device="cuda", requires_grad=True)
    w.grad = torch.zeros_like(w)
    opt = optim.AdamW([w], [w.grad], state_bits=bits)
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    y = (x @ w).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_training_loop(optim, bits):
    """Gradients written in place by backward, clipped, stepped on: the
    parameters move exactly as a second loop that computes them anew."""
    def loop():
        torch.manual_seed(0)
        net = torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.GELU(), torch.nn.Linear(65, 7)).cuda()
        params = list(net.parameters())
        for p in params:
            p.grad = torch.zeros_like(p)
        opt = optim.AdamW(params, [p.grad for p in params], lr=1e-2, state_bits=bits)
        norm = optim.GradNorm([p.grad for p in params])
        x, y = torch.randn(16, 33, device="cuda"), torch.randn(16, 7, device="cuda")
        for _ in range(5):
            for p in params:
                p.grad.zero_()
            torch.nn.functional.mse_loss(net(x), y).backward()
            opt.step(clip=norm(max_norm=0.1))
        return [p.detach().clone() for p in params]
    a, b = loop(), loop()
    assert _same(a, b)
    assert all(torch.isfinite(p).all() for p in a)


def test_class_refusals(optim):
    x = torch.zeros(16, 16, device="cuda")
    y = torch.zeros(16, 16, device="cuda")
    bad = [([x.cpu()], [y]), ([x], [y.cpu()]), ([x.double()], [y]), ([x], [y.int()]), ([x], []), ([x], [y[:8]]),
           ([x[:, ::2]], [y[:, ::2]]), ([x], [y.t()]), ([x[:1].expand(16, 16)], [y])]
    for ps, gs in bad:
        with pytest.raises((ValueError, TypeError)):
            optim.AdamW(ps, gs)
    with pytest.raises(TypeError):
        optim.AdamW([1.0], [y])
    for kw in (dict(lr=-1), dict(lr=math.nan), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=0.0),
               dict(weight_decay=-1.0), dict(weight_decay=[0.1, 0.1]), dict(state_bits=16), dict(seed=-1),
               dict(seed=1 << 64)):
        with pytest.raises(ValueError):
            optim.AdamW([x], [y], **kw)
    with pytest.raises(RuntimeError):
        optim.AdamW([x, x], [y, y])                    # one memory written twice
    with pytest.raises(RuntimeError):
        optim.AdamW([x], [x])
    opt = optim.AdamW([x], [y])
    for kw in (dict(lr=-1.0), dict(lr=math.inf), dict(grad_scale=math.nan), dict(clip=torch.ones(2)),
               dict(clip=torch.ones(1, device="cuda")), dict(clip=torch.ones(2, device="cuda").double()),
               dict(lr=torch.ones(1)), dict(lr=torch.ones(2, device="cuda"))):
        with pytest.raises(ValueError):
            opt.step(**kw)
    assert int(opt.state["step"]) == 0
    norm = optim.GradNorm([y])
    for kw in (dict(max_norm=0), dict(max_norm=math.nan), dict(grad_scale=math.inf)):
        with pytest.raises(ValueError):
            norm(**kw)
    with pytest.raises(ValueError):
        optim.GradNorm([y[:, ::2]])
    opt.close()
    norm.close()
    with pytest.raises(RuntimeError):
        opt.step()
    with pytest.raises(RuntimeError):
        norm()
