"""The 4-bit format, its rounding, its random bits and dropout in 64 bits, on
the CPU and apart from the library's code: what its tests compare with."""
import torch

BLOCK = 32
VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
ROUNDING, DROPOUT = 0x9E3779B9, 0x7F4A7C15
FULL = 0xFFFFFFFF


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & FULL
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & FULL
    return x ^ (x >> 16)


def random_bits(positions, purpose, seed, counter=0):
    """The 16 bits of each position (an int64 tensor)."""
    a = (seed & FULL) ^ purpose
    for part in (seed >> 32, counter & FULL, (counter >> 32) & FULL):
        a = mix(a) ^ part
    a = mix(a)
    b = mix(a ^ 0x85EBCA77)
    pair = positions >> 1
    x = (pair & FULL) ^ a ^ mix(pair >> 32)
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & FULL
    x = x ^ b
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & FULL
    x = x ^ (x >> 16)
    return torch.where(positions % 2 == 1, x >> 16, x & 0xFFFF)


def places(rows, cols):
    wide = -(-cols // BLOCK) * BLOCK
    return torch.arange(rows)[:, None] * wide + torch.arange(cols)


def scales(x):
    """Exponents of the blocks of the rows of a float64 matrix, and which are
    finite: the smallest e >= -127 with max <= 6 * 2^e."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    top = b.abs().amax(2)
    fine = b.isfinite().all(2)
    top = torch.where(fine, top, torch.zeros_like(top))
    e = torch.full(top.shape, -127, dtype=torch.int64)
    for k in range(-126, 128):
        e = torch.where(top > 6 * 2.0 ** (k - 1), k, e)
    return e, fine


def codes(x, bits=None):
    """(codes 0..15, exponents, finite blocks) of the rows of a matrix of
    float32 values; `bits`: 16 random bits for each element."""
    x = x.double()
    rows, cols = x.shape
    e, fine = scales(x)
    unit = torch.exp2(e.double()).repeat_interleave(BLOCK, 1)[:, :cols]
    ok = fine.repeat_interleave(BLOCK, 1)[:, :cols]
    y = torch.where(ok, x.abs(), torch.zeros_like(x)) / unit
    low = (y[..., None] >= VALUES[1:]).sum(-1).clamp(max=6)
    part = (y - VALUES[low]) / (VALUES[low + 1] - VALUES[low])
    if bits is None:
        up = (part > 0.5) | ((part == 0.5) & (low % 2 == 1))
    else:
        up = part >= 1 - (bits.double() + 0.5) / 65536
    code = low + up.long() + 8 * x.signbit().long()
    return torch.where(ok, code, torch.zeros_like(code)), e, fine


def values(x, bits=None):
    """What x reads back as, in float64."""
    rows, cols = x.shape
    code, e, fine = codes(x, bits)
    unit = torch.where(fine, torch.exp2(e.double()), torch.full(e.shape, float("nan"), dtype=torch.float64))
    v = VALUES[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    return v * unit.repeat_interleave(BLOCK, 1)[:, :cols]


def pack(code, e, fine):
    """Codes and scales of a matrix as they lie in memory."""
    rows, cols = code.shape
    panels, rows8, groups = -(-cols // 256), -(-rows // 8) * 8, -(-rows // 128)
    packed = torch.zeros(panels * rows8 * 128, dtype=torch.uint8)
    out = torch.zeros(panels * groups * 1024, dtype=torch.uint8)
    code = torch.nn.functional.pad(code, (0, -cols % BLOCK))
    pairs = (code[:, ::2] | code[:, 1::2] << 4).to(torch.uint8)
    r = torch.arange(rows)[:, None]
    k = torch.arange(e.shape[1])[None, :]
    at = (k // 8 * rows8 + r) * 128 + ((k % 8) ^ (r % 8)) * 16
    packed[(at[..., None] + torch.arange(16)).reshape(-1)] = pairs.reshape(-1)
    at = ((k // 8 * groups + r // 128) * 2 + k // 4 % 2) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + k % 4
    out[at.reshape(-1)] = torch.where(fine, e + 127, 255).to(torch.uint8).reshape(-1)
    return packed, out


def threshold(p):
    return int(p * 65536 + 0.5)


def dropped(x, p, seed, counter=0):
    """x after dropout, as float32 values (in float64)."""
    rows, cols = x.shape
    keep = random_bits(places(rows, cols), DROPOUT, seed, counter) >= threshold(p)
    factor = torch.tensor(65536 / (65536 - threshold(p)), dtype=torch.float32)
    return torch.where(keep, (x.float() * factor).double(), torch.zeros(x.shape, dtype=torch.float64))


def sum_bound(a, b, dtype):
    """How far out = a @ b.t() may be off: float32 sums of k products, in any
    order and cut off instead of rounded at worst (2^-23 of the magnitudes
    added up for each of k additions), and one rounding to dtype."""
    k = a.shape[1]
    size = a.abs() @ b.abs().t()
    return (k * 2.0 ** -23 * size) * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).eps / 2 * (a @ b.t()).abs() \
        + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
