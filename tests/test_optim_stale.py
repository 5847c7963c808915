"""Parameters and gradients that are no longer where an AdamW plan found them
are noticed (on the CPU: the check itself; tests/test_gpu_optim_use.py has the
class)."""
import pytest

torch = pytest.importorskip("torch")


def _model():
    net = torch.nn.Sequential(torch.nn.Linear(5, 3), torch.nn.Linear(3, 2))
    for p in net.parameters():
        p.grad = torch.zeros_like(p)
    return net, list(net.parameters())


def test_kept_gradients_pass():
    from compressor_b200 import optim
    net, params = _model()
    ties = optim._ties(params, [p.grad for p in params])
    assert len(ties) == 4
    for _ in range(2):
        optim._check_ties(ties)
        net.zero_grad(set_to_none=False)
        net(torch.randn(4, 5)).sum().backward()
    for p in params:
        p.grad.zero_()
    optim._check_ties(ties)


@pytest.mark.parametrize("how", ["zero_grad", "zero_grad and backward", "assigned", "gradient's data", "parameter's data",
                                 "double and float"])
def test_replaced_memory_is_refused(how):
    from compressor_b200 import optim
    net, params = _model()
    grads = [p.grad for p in params]
    ties = optim._ties(params, [g.detach() for g in grads])     # another object, the same memory
    if how.startswith("zero_grad"):
        net.zero_grad()
        if "backward" in how:
            net(torch.randn(4, 5)).sum().backward()
    elif how == "assigned":
        params[2].grad = torch.zeros_like(params[2])
    elif how == "gradient's data":
        grads[1].data = torch.zeros_like(params[1])
    elif how == "parameter's data":
        params[3].data = params[3].data.clone()
    else:
        net.double().float()
    with pytest.raises(RuntimeError, match="zero_grad\\(set_to_none=False\\)|has moved"):
        optim._check_ties(ties)


def test_gradients_of_ones_own_are_not_tied():
    from compressor_b200 import optim
    net, params = _model()
    plain = [torch.zeros(3), torch.zeros(0)]
    assert optim._ties(params + plain, [torch.zeros_like(p) for p in params + plain]) == []
    empty = torch.zeros(0, requires_grad=True)
    empty.grad = torch.zeros(0)
    assert optim._ties([empty], [empty.grad]) == []


def test_slices_of_a_leaf_are_not_asked_for_gradients(recwarn):
    """torch warns where .grad of a tensor is read that autograd never fills."""
    from compressor_b200 import optim
    flat = torch.zeros(10, requires_grad=True)
    flat.grad = torch.zeros(10)
    assert optim._ties([flat[:4], flat[4:]], [flat.grad[:4], flat.grad[4:]]) == []
    assert not recwarn.list
    kept = flat * 2
    kept.retain_grad()
    kept.sum().backward()
    assert len(optim._ties([kept], [kept.grad])) == 1 and not recwarn.list
