"""GPU tests of what the 4-bit operators and dropout promise beside their
values: operands of any strides, every byte of what is sent, and the rounds of
the way down."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from tests.test_gpu_mx4 import wild  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dropout_takes_residuals_of_any_strides(dtype):
    from compressor_b200.dropout import dropout
    x, whole = wild(65, 96, dtype, 1).cuda(), wild(130, 200, dtype, 2).cuda()
    for r in (whole[:65, 3:99], whole[::2, 104:], whole.t()[7:72, 5:101], whole[4, :96].expand(65, 96), whole[:65, 9:10].expand(65, 96)):
        assert not r.is_contiguous()
        for a in (x, whole.t()[60:125, 20:116]):
            want = dropout(a.contiguous(), 0.3, seed=4, residual=r.contiguous())
            assert torch.equal(dropout(a, 0.3, seed=4, residual=r), want)
            leaf = r.clone().requires_grad_()   # (the clone keeps the strides of views that have any)
            y = dropout(a, 0.3, seed=4, residual=leaf)
            assert torch.equal(y, want)
            g, = torch.autograd.grad(y, leaf, whole.t()[:65, :96])
            assert torch.equal(g, whole.t()[:65, :96])


@pytest.mark.parametrize("n", [1, 31, 33, 256, 1000, 5130, 70001])
@pytest.mark.parametrize("shift", [0, 1])
def test_every_byte_of_a_vector_is_written(n, shift):
    """Memory that held something else: the bytes between codes and scales,
    which are nobody's, are 0, and two encodes give the same buffer."""
    from compressor_b200 import mx4
    x = wild(1, n + shift, torch.float32, 3).cuda()[0, shift:]
    buffers = []
    for fill in (0xA5, 0x3C):
        room = [torch.full((mx4.Mx4Vector.size_of(n),), fill, dtype=torch.uint8, device="cuda") for _ in range(4)]
        del room
        buffers.append(mx4.encode(x).buffer)
    codes, scales = (n + 1) // 2, buffers[0].numel() - -(-n // 32)
    assert torch.equal(buffers[0], buffers[1]) and not buffers[0][codes:scales].any()


@pytest.mark.parametrize("rounding", ["nearest", "random"])
def test_rounds_of_the_way_down(rounding):
    """Each vector has its round's number, in a replayed graph too, and a client
    that is given another one is told before its weights change."""
    from compressor_b200 import federated as fed
    weights = wild(1, 5000, torch.bfloat16, 1).cuda()[0]
    held = torch.zeros(5000, device="cuda")
    down, mine = fed.Downlink(weights, held=held, rounding=rounding, seed=3), held.clone()
    for t in range(2):
        sent = down.send()
        assert int(sent.round) == t
        fed.Downlink.receive(sent, mine, round=t)
    before = mine.clone()
    with pytest.raises(ValueError, match="round 1, .* round 2"):
        fed.Downlink.receive(sent, mine, round=2)
    assert torch.equal(mine, before) and torch.equal(mine, down.held)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        sent = down.send()
    for t in range(2, 5):
        weights.add_(1)
        graph.replay()
        assert int(sent.round) == t and int(down.round) == t + 1
        fed.Downlink.receive(sent, mine, round=t)
        assert torch.equal(mine, down.held)
