"""GPU tests of what surrounds the optimiser operators' steps: error reports,
plans and the graphs and tensors that they are used with."""
import gc
import time

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def optim(product_lib):
    from compressor_b200 import optim
    return optim


def test_errors_waits_for_steps_on_other_streams(optim):
    p, g = torch.randn(70_000, device="cuda"), torch.randn(70_000, device="cuda")
    opt = optim.AdamW([p], [g], state_bits=8)
    opt.step()                                      # a kernel's first launch loads it, which may wait
    torch.cuda._sleep(1000)
    side = torch.cuda.Stream()                      # does not wait for the default stream, nor it for this one
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)              # about a tenth of a second
        opt.step()
    assert not side.query()
    assert opt.errors() == 0
    assert side.query() and int(opt.state["step"]) == 2


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["drop", "close"])
def test_graphs_outlive_their_objects(optim, bits, how):
    """Captured calls replay as ever after the objects are gone and their
    memory would have been used anew; with the last graph the rest goes."""
    def make():
        gen = torch.Generator("cuda").manual_seed(3)
        p = [torch.randn(n, device="cuda", generator=gen) for n in (70_001, 300)]
        g = [torch.randn(n, device="cuda", generator=gen) for n in (70_001, 300)]
        return p, optim.AdamW(p, g, state_bits=bits), optim.GradNorm(g)

    p, opt, norm = make()
    q, ref, rnorm = make()
    for o, n in ((opt, norm), (ref, rnorm)):
        o.step(clip=n(max_norm=0.5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step(clip=norm(max_norm=0.5))          # a stream that has seen eager steps is captured too
    ref.step(clip=rnorm(max_norm=0.5))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step(clip=norm(max_norm=0.5))
    lib, handles = opt.lib, (norm._h, opt._h)
    assert lib.falcom_norm_graphs(handles[0]) == 1 and lib.falcom_adamw_graphs(handles[1]) == 1
    if how == "close":
        opt.close()
        norm.close()
    del opt, norm
    gc.collect()
    torch.cuda.empty_cache()
    junk = [torch.full((k,), 7, dtype=torch.uint8, device="cuda") for k in (512, 3000, 70_144, 300_000, 1 << 20) for _ in range(8)]
    for _ in range(3):
        graph.replay()
        ref.step(clip=rnorm(max_norm=0.5))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(p, q)) and all(bool((j == 7).all()) for j in junk)
    assert len(optim._kept) == 2
    del graph
    gc.collect()
    torch.cuda.synchronize()
    for _ in range(100):                           # a graph's end reaches the count on a thread of the driver's
        if lib.falcom_norm_graphs(handles[0]) + lib.falcom_adamw_graphs(handles[1]) == 0:
            break
        time.sleep(0.05)
    rnorm.close()
    assert not optim._kept


@pytest.mark.parametrize("bits", [32, 8])
def test_replaced_gradients_stop_the_step(optim, bits):
    """A training loop that drops its gradients fails loudly and changes nothing."""
    net = torch.nn.Linear(33, 65).cuda()
    for p in net.parameters():
        p.grad = torch.zeros_like(p)
    opt = optim.AdamW(list(net.parameters()), [p.grad for p in net.parameters()], state_bits=bits)
    x = torch.randn(16, 33, device="cuda")
    net.zero_grad(set_to_none=False)
    net(x).square().sum().backward()
    opt.step()
    before = [p.detach().clone() for p in net.parameters()]
    net.zero_grad()
    net(x).square().sum().backward()
    with pytest.raises(RuntimeError, match="set_to_none=False"):
        opt.step()
    assert all(torch.equal(a, b) for a, b in zip(before, net.parameters())) and int(opt.state["step"]) == 1


def test_replaced_memory_is_held(optim):
    """What a plan's addresses lead to is not given to others while it exists."""
    p, g = torch.zeros(100_000, device="cuda"), torch.ones(100_000, device="cuda")
    opt, norm = optim.AdamW([p], [g], weight_decay=0.0), optim.GradNorm([g])
    places = {p.data_ptr(), g.data_ptr()}
    p.data, g.data = torch.zeros(7, device="cuda"), torch.zeros(7, device="cuda")
    others = [torch.empty(100_000, device="cuda") for _ in range(16)]
    assert not places & {t.data_ptr() for t in others}
    norm()
    opt.step()


def test_norms_at_other_offsets_differ_in_the_last_place(optim):
    """The sum's order follows the arrays' offsets from 16 bytes: the same
    offsets give the same bits wherever the arrays lie, others at most
    neighbouring results."""
    src = torch.randn(1_000_003, device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    first = None
    for k in (0, 0, 1, 1, 2, 3, 3):
        buf = torch.empty(src.numel() + 8, device="cuda")
        g = buf[k:k + src.numel()].copy_(src)
        got = optim.GradNorm([g])(max_norm=1.0)
        again = optim.GradNorm([g.clone() if k == 0 else g])(max_norm=1.0)
        assert torch.equal(got, again)
        first = got if first is None else first
        # 64-bit sums in another order, each result rounded to float32 once
        assert bool(((got - first).abs() <= 2.0 ** -23 * first).all())
