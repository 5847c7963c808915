"""More GPU tests of the optimiser operators: the 8-bit states bit for bit
against the formulas in separately rounded float32, every offset from the
16-byte alignment, tensors past 2^32 elements, and uses that captures and
collectors make of the plans."""
import gc
import math

import numpy as np
import pytest

from tests import optim_cases as oc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F = np.float32


@pytest.fixture(scope="module")
def optim(product_lib):
    from compressor_b200 import optim
    return optim


def _codes(x, chance, least):
    """Codes and scales of magnitudes x [blocks, 256] in float32, each operation rounded once."""
    top = x.max(1)
    live = top >= F(2.0 ** -100)
    with np.errstate(divide="ignore"):
        up = np.where(live, F(448) / top, F(0))
    y = (x * up[:, None]) * F(2.0 ** -120)
    code = np.minimum((y.view(np.uint32) + chance) >> 20, 126)
    code = np.maximum(code, ((x > 0) & live[:, None]) * least)
    return code.astype(np.uint8), np.where(live, top * F(1 / 448.0), F(0))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("spread", [1.0, 12.0])
def test_adamw8_bits(optim, dtype, spread):
    """Codes and scales equal the formulas' in float32 (products and sums
    rounded one by one, IEEE root and quotient); `spread`: e-folds between a
    block's largest and smallest gradients."""
    kind = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    n = 2048 * 40
    rng = np.random.default_rng(1)
    size = np.exp(-rng.random(n) * spread) * (0.0 if dtype == "f16" else 1.0) + (dtype == "f16")
    g32 = (rng.standard_normal(n) * size * np.repeat(np.exp(rng.standard_normal(n // 256)), 256)).astype(F)
    g32[::97] = 0
    g = torch.from_numpy(g32).cuda().to(kind)
    p = torch.zeros(n, device="cuda", dtype=kind)
    beta1, beta2, seed, scale = 0.9, 0.999, 12345678901234567890, -0.3
    opt = optim.AdamW([p], [g], state_bits=8, betas=(beta1, beta2), seed=seed)
    gs = g.float().cpu().numpy() * F(scale)
    m = np.zeros((n // 256, 256), F)
    root = np.zeros_like(m)
    for t in range(1, 6):
        opt.step(grad_scale=scale)
        m = m * F(beta1) + (gs * F(1 - beta1)).reshape(-1, 256)
        v = (root * root) * F(beta2) + ((gs * gs) * F(1 - beta2)).reshape(-1, 256)
        root = np.sqrt(v)
        w = oc.words(seed, t, np.arange(n, dtype=np.uint64)).astype(np.uint32).reshape(-1, 256)
        mc, ms = _codes(np.abs(m), w >> np.uint32(12), 0)
        vc, vs = _codes(root, w & np.uint32(0xFFFFF), 1)
        got = {k: x.cpu() for k, x in opt.state.items()}
        hm = got["m"].view(torch.uint8).numpy().reshape(-1, 256)
        assert (got["m_scale"].numpy() == ms).all() and (got["v_scale"].numpy() == vs).all(), t
        assert ((hm & 0x7F) == mc).all() and (got["v"].view(torch.uint8).numpy().reshape(-1, 256) == vc).all(), t
        assert ((hm >> 7) == (m < 0))[mc > 0].all()
        m = (oc.e4m3(mc).astype(F) * ms[:, None]) * np.where(m < 0, F(-1), F(1))
        root = oc.e4m3(vc).astype(F) * vs[:, None]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_any_offset_gives_the_same_bits(optim, bits, kind):
    """Parameters and gradients 0 to 7 elements off their alignment, each on its own."""
    n = 3 * 2048 + 700
    gen = torch.Generator("cuda").manual_seed(4)
    src = torch.randn(n, device="cuda", generator=gen).to(kind)
    grad = torch.randn(n, device="cuda", generator=gen).to(kind)
    first = None
    for ps, gs in [(0, 0)] + [(k, 0) for k in range(1, 8)] + [(0, k) for k in range(1, 8)] + [(3, 5), (4, 4)]:
        pb, gb = (torch.full((n + 16,), 7.0, device="cuda", dtype=kind) for _ in range(2))
        p, g = pb[ps:ps + n], gb[gs:gs + n]
        p.copy_(src)
        g.copy_(grad)
        opt = optim.AdamW([p], [g], state_bits=bits)
        norm = optim.GradNorm([g])
        for _ in range(2):
            opt.step(clip=norm(max_norm=1.0))
        out = [p.clone()] + [t.clone() for t in opt.state.values()]
        first = first or out
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(first, out)), (ps, gs)
        assert (pb[:ps] == 7).all() and (pb[ps + n:] == 7).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_more_than_2_32_elements(optim, bits):
    """One tensor of over 2^32 elements behind a short one: whole blocks on
    both sides of position 2^32, the ends, and the norm over all of it."""
    n = (1 << 32) + 5001
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of free device memory")
    head_p, head_g = torch.ones(600, device="cuda").bfloat16(), torch.ones(600, device="cuda").bfloat16()
    g = torch.empty(n, device="cuda", dtype=torch.bfloat16).normal_()
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    opt = optim.AdamW([head_p, p], [head_g, g], state_bits=bits, lr=1e-2, weight_decay=0.0, seed=9)
    norm = optim.GradNorm([head_g, g])()
    opt.step()
    total = 600.0 + sum(float(part.double().square().sum()) for part in g.split(1 << 28))
    assert abs(float(norm[0]) - math.sqrt(total)) <= 2.0 ** -23 * math.sqrt(total)
    assert opt.offsets[1] == 768
    edge = (1 << 32) - 768                        # the tensor's element at position 2^32
    for at in (0, 256 * 4321, edge - 2048 - 256, edge - 256, edge, edge + 256, edge + 2048, (n // 256 - 1) * 256):
        w = slice(at, at + 256)
        gw = g[w].double().cpu().numpy()
        # a first step: m = 0.1 g, v = 0.001 g^2, an update of lr * sign(g) but for eps
        want = -1e-2 * np.sign(gw) * (np.abs(gw) / (np.abs(gw) + 1e-8))
        assert (np.abs(p[w].double().cpu().numpy() - want) <= 1e-2 * (2.0 ** -8 + 2.0 ** -18)).all(), at
        o = opt.offsets[1] + at
        if bits == 32:
            assert (np.abs(opt.state["m"][o:o + 256].double().cpu().numpy() - 0.1 * gw) <= 4 * oc.U * 0.1 * np.abs(gw)).all()
            assert (np.abs(opt.state["v"][o:o + 256].double().cpu().numpy() - 0.001 * gw * gw) <= 6 * oc.U * 0.001 * gw * gw).all()
            continue
        chance = oc.words(9, 1, np.arange(o, o + 256, dtype=np.uint64)).astype(np.int64)
        for key, x, c, least in (("m", 0.1 * np.abs(gw), chance >> 12, 0), ("v", math.sqrt(0.001) * np.abs(gw), chance & 0xFFFFF, 1)):
            code = opt.state[key][o:o + 256].view(torch.uint8).cpu().numpy().astype(np.int64) & 0x7F
            live = x > 0
            oc.check_block(x[live] / x.max() * 448, code[live], c[live] / 2.0 ** 20, np.full(live.sum(), least),
                           np.full(live.sum(), 16 * oc.U))
    assert opt.errors() == 0


def test_many_captured_norms(optim):
    """More captured calls than the plan has scratch prepared for, replayed out of order."""
    gs = [torch.randn(100_001, device="cuda")]
    norm = optim.GradNorm(gs)
    graphs = []
    for k in range(12):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = norm(max_norm=1.0, grad_scale=1.0 + k)
        graphs.append((g, out))
    want = [norm(max_norm=1.0, grad_scale=1.0 + k) for k in range(12)]
    for _ in range(3):
        for g, _ in reversed(graphs):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for (_, o), w in zip(graphs, want))


def test_plan_dropped_during_a_capture(optim):
    """A collector that frees another plan inside a capture does not end it."""
    old = optim.GradNorm([torch.randn(1000, device="cuda")])
    p, g = torch.randn(5000, device="cuda"), torch.randn(5000, device="cuda")
    opt = optim.AdamW([p], [g])
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
        del old
        gc.collect()
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert int(opt.state["step"]) == 3


def test_plans_hold_no_copies(optim):
    """Gradients rewritten between steps are the ones read; a tensor used twice as a gradient counts twice."""
    g = torch.ones(1000, device="cuda")
    norm = optim.GradNorm([g, g, g[:10]])
    assert abs(float(norm()[0]) - math.sqrt(2010)) < 1e-4
    g.fill_(2.0)
    assert abs(float(norm()[0]) - 2 * math.sqrt(2010)) < 1e-4


def test_refuses_what_does_not_hold_its_values(optim):
    x = torch.randn(8, 8, device="cuda")
    with pytest.raises(ValueError):
        optim.GradNorm([x.to_sparse()])
    neg = torch.randn(8, device="cuda", dtype=torch.complex64).conj().imag
    with pytest.raises(ValueError):
        optim.GradNorm([neg])
    assert optim.GradNorm([])().tolist() == [0.0, 1.0]
    empty = optim.AdamW([], [])
    empty.step()
    assert int(empty.state["step"]) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_two_plans_at_once(optim, bits):
    """Two optimisers with their norms on two streams at once leave what they leave one after the other."""
    def make():
        gen = torch.Generator("cuda").manual_seed(8)
        sets = []
        for n in (700_001, 1_300_000):
            p = torch.randn(n, device="cuda", generator=gen)
            g = torch.randn(n, device="cuda", generator=gen)
            sets.append((p, optim.AdamW([p], [g], state_bits=bits), optim.GradNorm([g])))
        return sets

    apart, together = make(), make()
    for _, opt, norm in apart:
        for _ in range(30):
            opt.step(clip=norm(max_norm=0.5))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(30):
        for s, (_, opt, norm) in zip(streams, together):
            with torch.cuda.stream(s):
                opt.step(clip=norm(max_norm=0.5))
    torch.cuda.synchronize()
    for (p, o, _), (q, r, _) in zip(apart, together):
        assert torch.equal(p, q) and all(torch.equal(o.state[k].view(torch.uint8), r.state[k].view(torch.uint8)) for k in o.state)
