"""GPU tests of what surrounds the optimiser operators' steps: error reports,
plans and the graphs and tensors that they are used with."""
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
