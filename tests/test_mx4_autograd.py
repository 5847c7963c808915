"""Which calls of linear and dropout go through autograd, on the CPU with a
stand-in for the launches: those that a gradient is wanted of, and those whose
tensors carry a tangent of forward mode, which is refused and never lost."""
import pytest

torch = pytest.importorskip("torch")
import torch.autograd.forward_ad as forward_ad  # noqa: E402

from compressor_b200 import dropout, mx4  # noqa: E402


@pytest.fixture
def calls(monkeypatch):
    """The calls of either operator with the launches counted instead of made."""
    made = []

    def run(x, residual, p, seed, counter):
        made.append("dropout")
        return torch.zeros_like(x)

    def forward(x, w, p, seed, counter, need_x, need_w):
        made.append((need_x, need_w))
        return x.new_zeros(*x.shape[:-1], w.shape[0]), None, torch.zeros(0)

    monkeypatch.setattr(mx4, "_check", lambda t, what: None)
    monkeypatch.setattr(dropout, "_run", run)
    monkeypatch.setattr(mx4, "_linear_forward", forward)
    return made


CALLS = {
    "linear x": (lambda t: mx4.linear(t, torch.ones(3, 4), p=0.5, seed=1)),
    "linear weight": (lambda t: mx4.linear(torch.ones(2, 4), t, seed=1)),
    "dropout x": (lambda t: dropout.dropout(t, 0.5, seed=1)),
    "dropout x beside a residual": (lambda t: dropout.dropout(t, 0.5, seed=1, residual=torch.ones(2, 4))),
    "dropout residual": (lambda t: dropout.dropout(torch.ones(2, 4), 0.5, seed=1, residual=t)),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_tangents_are_refused(calls, name, mode):
    with mode(), forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(2, 4), torch.ones(2, 4))
        with pytest.raises(NotImplementedError):
            CALLS[name](dual)


@pytest.mark.parametrize("name", CALLS)
def test_other_calls(calls, name):
    with forward_ad.dual_level():   # no tangent on what the call is given
        assert not CALLS[name](torch.ones(2, 4)).requires_grad
    assert CALLS[name](torch.ones(2, 4, requires_grad=True)).requires_grad
    with torch.no_grad():
        assert not CALLS[name](torch.ones(2, 4, requires_grad=True)).requires_grad
    assert len(calls) == 3


def test_a_residual_sum_without_dropout_keeps_tangents(calls):
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(2, 4), torch.full((2, 4), 3.0))
        assert dropout.dropout(dual, 0.0) is dual
        y = dropout.dropout(dual, 0.0, residual=dual)
        assert torch.equal(forward_ad.unpack_dual(y).tangent, torch.full((2, 4), 6.0)) and not calls
