"""Dropout on the GPU against its definition."""
import pytest
import torch

from tests import mx4_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 8), (5, 33), (2, 1024), (65, 1000), (7, 257)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_is_exact(rows, cols, dtype, p, residual):
    from compressor_b200.dropout import dropout
    g = torch.Generator().manual_seed(rows * cols)
    x, r, dy = (torch.randn(rows, cols, generator=g).to(dtype) for _ in range(3))
    xg, rg = x.cuda().requires_grad_(), r.cuda().requires_grad_()
    y = dropout(xg, p, seed=3, residual=rg if residual else None)
    want = ref.dropped(x, p, 3).float()
    if residual:
        want = want + r.float()
    assert torch.equal(y.detach().cpu(), want.to(dtype))
    grads = torch.autograd.grad(y, (xg, rg) if residual else (xg,), dy.cuda())
    assert torch.equal(grads[0].cpu(), ref.dropped(dy, p, 3).to(dtype))
    if residual:
        assert torch.equal(grads[1].cpu(), dy)
