"""Matrices of 4-bit values whose products float32 holds exactly, in any order
of summation: what a product has to give is then known to the last bit."""
import torch

from tests import mx4_reference as ref


def matrix(rows, cols, seed, device="cpu"):
    """float32 values that 4 bits hold: scales of 1/2, 1 and 2, elements of all
    codes, in each block one of 6 times the scale."""
    g = torch.Generator(device).manual_seed(seed)
    blocks = -(-cols // 32)
    code = torch.randint(0, 8, (rows, blocks, 32), generator=g, device=device)
    code[:, :, 0] = 7
    sign = 1.0 - 2.0 * torch.randint(0, 2, code.shape, generator=g, device=device)
    scale = torch.exp2(torch.randint(-1, 2, (rows, blocks, 1), generator=g, device=device).float())
    return (ref.VALUES.to(device)[code].float() * sign * scale).view(rows, -1)[:, :cols].contiguous()


def product(a, b):
    """a @ b.t() in float64.  Products are multiples of 1/16 (1/2 x 1/2 x 1/2 x
    1/2); below 2^20 in sum every partial sum has at most 24 bits."""
    a, b = a.double(), b.double()
    assert float((a.abs() @ b.abs().t()).max()) < 2 ** 20
    return a @ b.t()
