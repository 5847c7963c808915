"""Cases of the 4-bit operators and of dropout: what brings a model to its
clients in 4 bits, and what a client then answers and trains with.

Microscaled 4-bit floating point (MX): 32 consecutive elements share a scale
that is a power of two, the smallest under which no magnitude is above 6; an
element is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign.  Values are rounded
to the nearest (ties to the even code), or up or down at random in proportion
to the distance.  A block with an infinity or NaN reads back as NaN.

Random bits: element (r, c) of a matrix of C columns has 16 bits of a hash of
(seed, counter, position), the position being r * (C rounded up to 32) + c;
two neighbouring elements share a 32-bit word, the even one has its low half.

  downlink  a server encodes new weights as the 4-bit difference from what its
            clients hold and brings its copy of that forward; a client adds
            what it receives to its weights
  product   activations, rounded to 4 bits on the way, times 4-bit weights
  linear    a training step of a layer: both factors of each of its three
            products in 4 bits along the summed dimension, the incoming
            gradient rounded at random, dropout before the first
  dropout   with a residual sum, forward and backward, the mask made again
"""
import math
import random

import torch

own = False

BLOCK, SEED = 32, 20250917
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
LARGEST = {"flops": 6 * 4099 * 1024 * 50257, "bytes": 7e9}


# --- cases ---------------------------------------------------------------

def listed():
    return [
        # a linear head goes out to clients: the latency of two small calls
        {"name": "downlink head", "op": "downlink", "n": 5130, "type": "f32", "rounding": "random", "weight": 1.0, "shift": 0},
        # a convolutional network, off its alignment, into a mean over clients
        {"name": "downlink resnet50", "op": "downlink", "n": 23_528_522, "type": "f32", "rounding": "nearest", "weight": 0.25, "shift": 1},
        # a language model
        {"name": "downlink gpt2-medium", "op": "downlink", "n": 354_823_168, "type": "f32", "rounding": "random", "weight": 1.0, "shift": 0},
        # the logits of one token, after each of which the next waits
        {"name": "product token logits", "op": "product", "t": 1, "k": 1024, "n": 50257, "type": "bf16", "out": "f32"},
        # a few sequences' tokens through the narrowing half of a feed-forward block
        {"name": "product few rows", "op": "product", "t": 5, "k": 4096, "n": 1024, "type": "f16", "out": "f16"},
        # a prompt of odd length through the widening half
        {"name": "product prompt", "op": "product", "t": 1001, "k": 1024, "n": 4096, "type": "bf16", "out": "bf16"},
        # a client scores its texts: all logits of 8192 tokens
        {"name": "product all logits", "op": "product", "t": 8192, "k": 1024, "n": 50257, "type": "bf16", "out": "bf16"},
        # a classifier's head on odd sizes: the latency of a training step
        {"name": "linear head", "op": "linear", "t": 77, "k": 513, "n": 10, "type": "f32", "weights": "f32", "p": 0.1},
        # a local step of a feed-forward block on 16 texts of 1024 tokens
        {"name": "linear feed-forward", "op": "linear", "t": 16384, "k": 1024, "n": 4096, "type": "bf16", "weights": "bf16", "p": 0.1},
        # the output layer on a ragged batch, 32-bit weights under 16-bit activations
        {"name": "linear vocabulary", "op": "linear", "t": 4099, "k": 1024, "n": 50257, "type": "bf16", "weights": "f32", "p": 0.0},
        # one token's row
        {"name": "dropout row", "op": "dropout", "t": 1, "k": 1024, "type": "f32", "p": 0.1, "residual": False},
        # a block's output on its residual stream
        {"name": "dropout residual", "op": "dropout", "t": 16384, "k": 4096, "type": "bf16", "p": 0.1, "residual": True},
    ]


def draw(rng):
    def size(low, high):
        return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))

    op = rng.choice(["downlink", "product", "linear", "dropout"])
    kind = rng.choice(list(TYPES))
    if op == "downlink":
        return {"op": op, "n": size(1, 300_000_000), "type": kind, "rounding": rng.choice(["nearest", "random"]),
                "weight": rng.choice([1.0, 0.25, 0.1]), "shift": rng.choice([0, 0, 1, 2, 3])}
    t, k = size(1, 16384), size(1, 8192)
    if op == "dropout":
        return {"op": op, "t": t, "k": k, "type": kind, "p": rng.choice([0.0, 0.1, 0.3, 0.5]), "residual": rng.random() < 0.5}
    n = size(1, 50257)
    t = max(1, min(t, LARGEST["flops"] // (6 * n * k), 400_000_000 // max(n, k)))
    if op == "product":
        return {"op": op, "t": t, "k": k, "n": n, "type": kind, "out": rng.choice(list(TYPES))}
    return {"op": op, "t": t, "k": k, "n": n, "type": kind, "weights": rng.choice([kind, "f32"]), "p": rng.choice([0.0, 0.1, 0.5])}


def work(case):
    c, s = case, SIZE[case["type"]]
    if c["op"] == "downlink":
        return {"bytes": c["n"] * (s + 8 + 8) + 2 * (c["n"] / 2 + c["n"] / BLOCK), "flops": 8 * c["n"]}
    t, k = c["t"], c["k"]
    if c["op"] == "dropout":   # forward: x, the residual, y; backward: dy, dx
        return {"bytes": t * k * s * (4 + c["residual"]), "flops": (4 + c["residual"]) * t * k}
    n = c["n"]
    if c["op"] == "product":
        return {"bytes": t * k * s + n * (k / 2 + k / BLOCK) + t * n * SIZE[c["out"]], "flops": 2 * t * k * n}
    return {"bytes": 2 * (t * k * s + n * k * SIZE[c["weights"]] + t * n * s), "flops": 6 * t * k * n}


# --- inputs --------------------------------------------------------------

def prepare(case, seed):
    c, kind = case, TYPES[case["type"]]
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    s = {"case": c, "seed": SEED + seed}
    if c["op"] == "downlink":
        n, total = c["n"], c["n"] + c["shift"]
        held = normal(total) * 0.02
        # updates of very different sizes from block to block, one block in eight without any
        blocks = -(-total // 256)
        sizes = 1e-3 * torch.exp(normal(blocks)) * (torch.rand(blocks, device=dev, generator=gen) > 0.125)
        s["x"] = (held + normal(total) * sizes.repeat_interleave(256)[:total]).to(kind)[c["shift"]:]
        s["base"] = held[c["shift"]:]
        s["weights"] = held.clone()[c["shift"]:]
        assert s["x"].numel() == n
        return s
    t, k = c["t"], c["k"]
    # activations with a few large features
    s["x"] = (normal(t, k) * (1 + 7 * (torch.rand(k, device=dev, generator=gen) > 0.98))).to(kind)
    if c["op"] == "dropout":
        s["residual"] = normal(t, k).to(kind) if c["residual"] else None
        s["dy"] = (normal(t, k) * 1e-2).to(kind)
        if own:
            s["x"].requires_grad_()
        return s
    n = c["n"]
    w = normal(n, k) * 0.02
    if c["op"] == "product":
        if own:
            from compressor_b200 import mx4
            s["w"] = mx4.quantize(w)
        else:
            s["w"] = values(w)
        return s
    s["w"] = w.to(TYPES[c["weights"]])
    # gradients of tokens that differ in size
    s["dy"] = (normal(t, n) * (1e-2 * torch.exp(normal(t, 1)))).to(kind)
    if own:
        s["x"].requires_grad_()
        s["w"].requires_grad_()
    return s


# --- one pass ------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        from compressor_b200 import dropout, mx4
        if c["op"] == "downlink":
            sent = mx4.encode(s["x"], base=s["base"], rounding=c["rounding"], seed=s["seed"])
            mx4.decode(sent, out=s["weights"], weight=c["weight"], accumulate=True)
            return {"base": s["base"], "weights": s["weights"]}
        if c["op"] == "product":
            return mx4.product(s["x"], s["w"], dtype=TYPES[c["out"]])
        if c["op"] == "linear":
            y = mx4.linear(s["x"], s["w"], p=c["p"], seed=s["seed"])
            dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw}
        y = dropout.dropout(s["x"], c["p"], seed=s["seed"], residual=s["residual"])
        return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    if c["op"] == "downlink":
        change = s["x"].float() - s["base"]
        v = values(change[None], words(s["seed"], ROUNDING, 1, c["n"], change.device) if c["rounding"] == "random" else None)[0]
        s["base"] += v
        s["weights"] += v * c["weight"]
        return {"base": s["base"], "weights": s["weights"]}
    if c["op"] == "product":
        return (values(s["x"].float()) @ s["w"].t()).to(TYPES[c["out"]])
    if c["op"] == "linear":
        return plain_linear(s["x"], s["w"], s["dy"], c["p"], s["seed"])
    keep = kept(c["p"], s["seed"], *s["x"].shape, s["x"].device)
    y = drop(s["x"].float(), keep, c["p"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(s["x"].dtype), "dx": drop(s["dy"].float(), keep, c["p"]).to(s["x"].dtype)}


ROUNDING, DROPOUT = 0x9E3779B9, 0x7F4A7C15   # what the random bits are for


def _avalanche(x):
    """A 32-bit avalanche of shifts and odd products, on whole numbers."""
    x = ((x ^ (x >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def words(seed, purpose, rows, cols, device):
    """16 random bits for each element, as whole numbers (counter 0; positions under 2^33)."""
    first = _avalanche(_avalanche(_avalanche(_avalanche((seed & 0xFFFFFFFF) ^ purpose) ^ (seed >> 32))))
    second = _avalanche(first ^ 0x85EBCA77)
    wrap = (lambda v: v - (1 << 32) if v >> 31 else v)
    wide = -(-cols // BLOCK) * (BLOCK // 2)
    x = torch.arange(rows * wide, dtype=torch.int32, device=device) ^ wrap(first)
    x = (x ^ ((x >> 16) & 0xFFFF)) * -2048144789 ^ wrap(second)
    x = (x ^ ((x >> 13) & 0x7FFFF)) * -1028477387
    x = x ^ ((x >> 16) & 0xFFFF)
    return torch.stack([x & 0xFFFF, (x >> 16) & 0xFFFF], -1).view(rows, 2 * wide)[:, :cols]


def values(x, bits=None):
    """What the float32 matrix x reads back as after it is rounded to 4 bits along its rows."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    blocks = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, BLOCK)
    top = blocks.abs().amax(2, keepdim=True)
    fine = top.isfinite()
    part, power = torch.frexp(torch.where(fine, top, torch.zeros_like(top)))
    power = (power - 3 + (part > 0.75).int()).clamp(min=-127)
    unit = torch.exp2(power.double())
    y = blocks.double().abs() / unit
    steps = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    low = torch.bucketize(y, steps, right=True).sub_(1).clamp_(0, 6)
    below = steps[low]
    part = (y - below) / (steps[low + 1] - below)
    del y
    if bits is None:   # the even code of two that are as near
        up = (part > 0.5) | ((part == 0.5) & (low % 2 == 1))
    else:
        up = part >= 1 - (torch.nn.functional.pad(bits, (0, pad)).view_as(part).double() + 0.5) / 65536
    del part, below
    v = (steps[low + up] * unit).float() * blocks.sign()
    return torch.where(fine, v, torch.full_like(v, float("nan"))).view(rows, -1)[:, :cols]


def _threshold(p):
    return math.floor(p * 65536 + 0.5)


def kept(p, seed, rows, cols, device):
    return words(seed, DROPOUT, rows, cols, device) >= _threshold(p) if p > 0 else None


def drop(x, keep, p):
    return x if keep is None else torch.where(keep, x * (65536 / (65536 - _threshold(p))), torch.zeros_like(x))


def plain_linear(x, w, dy, p, seed):
    keep = kept(p, seed, *x.shape, x.device)
    a, weights, g = drop(x.float(), keep, p), w.float(), dy.float()
    bits = words(seed, ROUNDING, *g.shape, g.device)
    y = values(a) @ values(weights).t()
    dx = values(g, bits) @ values(weights.t()).t()
    dw = values(g.t(), bits.t()) @ values(a.t()).t()
    return {"y": y.to(x.dtype), "dx": drop(dx, keep, p).to(x.dtype), "dw": dw.to(w.dtype)}


# --- the definition in 64 bits -------------------------------------------

def _chances(seed, purpose, rows, cols, device):
    """The random bits of each element over 2^16, in 64-bit whole numbers."""
    full = 0xFFFFFFFF
    key = _avalanche((seed & full) ^ purpose)
    for part in (seed >> 32, 0, 0):
        key = _avalanche(key ^ part)
    at = torch.arange(rows, device=device)[:, None] * (-(-cols // BLOCK) * BLOCK) + torch.arange(cols, device=device)
    x = (at >> 1) ^ key
    x = (((x ^ (x >> 16)) * 0x85EBCA6B) & full) ^ _avalanche(key ^ 0x85EBCA77)
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & full
    x ^= x >> 16
    return ((x >> (16 * (at & 1))) & 0xFFFF).double() / 65536


def _rounded(x, chance=None):
    """Nearest or random 4-bit values of the rows of a float64 matrix, a range of columns at a time."""
    out = torch.empty_like(x)
    for begin in range(0, x.shape[1], BLOCK * 65536):
        part = x[:, begin:begin + BLOCK * 65536]
        room = -part.shape[1] % BLOCK
        b = torch.nn.functional.pad(part, (0, room)).unflatten(1, (-1, BLOCK))
        top = b.abs().amax(2, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2((top / 6).clamp(min=2.0 ** -127))))
        scale = torch.where(top > 6 * scale, 2 * scale, torch.where((top <= 3 * scale) & (scale > 2.0 ** -127), scale / 2, scale))
        size = (b / scale).abs()
        gap = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0)).double()
        if chance is None:
            near = torch.round(size / gap) * gap   # halves to the even multiple, whose code is even too
        else:
            u = torch.nn.functional.pad(chance[:, begin:begin + BLOCK * 65536], (0, room)).unflatten(1, (-1, BLOCK))
            near = torch.floor(size / gap + u + 2.0 ** -17) * gap
        out[:, begin:begin + BLOCK * 65536] = (torch.copysign(near, b) * scale).flatten(1)[:, :part.shape[1]]
    return out


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    c, at, dev = case, s["seed"], s["x"].device
    x = s["x"].double()
    if c["op"] == "downlink":
        change = (s["x"].float() - s["base"]).double()[None]
        v = _rounded(change, _chances(at, ROUNDING, 1, c["n"], dev) if c["rounding"] == "random" else None)[0]
        return {"base": s["base"].double() + v, "weights": s["weights"].double() + c["weight"] * v}
    if c["op"] == "product":
        return _rounded(x) @ s["w"].double().t()
    keep = _chances(at, DROPOUT, *x.shape, dev) * 65536 >= round(c["p"] * 65536)
    factor = keep / (1 - round(c["p"] * 65536) / 65536)
    dy = s["dy"].double()
    if c["op"] == "dropout":
        return {"y": x * factor + (0 if s["residual"] is None else s["residual"].double()), "dx": dy * factor}
    dropped = (s["x"].float() * factor.float()).double()   # 32 bits go to the rounding
    w, u = s["w"].double(), _chances(at, ROUNDING, *dy.shape, dev)
    y = _rounded(dropped) @ _rounded(w).t()
    dx = (_rounded(dy, u) @ _rounded(w.t().contiguous()).t()) * factor
    dw = _rounded(dy.t().contiguous(), u.t().contiguous()) @ _rounded(dropped.t().contiguous()).t()
    return {"y": y, "dx": dx, "dw": dw}
