"""Cases of the optimiser operators: the gradient norm with its clipping
coefficient, and AdamW steps over many tensors with 32-bit and 8-bit states.

A server that has summed its clients' updates, and a client that trains
between two rounds, both take such a step next to the codec.  Tensors lie one
after another in flat buffers, each from a multiple of 256 elements on, those
with weight decay first; `shift` moves parameters and gradients off their
16-byte alignment by that many elements.

8-bit states: per 256 elements of a tensor, the first moment and the root of
the second are held as float8 e4m3 codes times a float32 scale (largest
magnitude / 448), rounded up or down at random in proportion to the distance,
with random bits that are a hash of seed, step number and position.
"""
import math
import random

import torch

own = False

BLOCK = 256
BETA1, BETA2, EPS, LR, DECAY, SEED = 0.9, 0.999, 1e-8, 1e-3, 0.01, 20240611
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# --- cases ---------------------------------------------------------------

def listed():
    return [
        # a linear head that a client fine-tunes alone: the latency of one small call
        {"name": "norm head", "op": "norm", "model": "head", "grad": "f32", "shift": 0},
        # the summed update of a convolutional network, off its alignment
        {"name": "norm resnet50", "op": "norm", "model": "resnet50", "grad": "f32", "shift": 1},
        # the local gradient of a language model in half the bytes
        {"name": "norm gpt2-medium bf16", "op": "norm", "model": "gpt2-medium", "grad": "bf16", "shift": 0},
        # the same head's step
        {"name": "adamw32 head", "op": "adamw32", "model": "head", "param": "f32", "grad": "f32", "shift": 0, "clip": False, "start": 1000},
        # a server's first step on a convolutional network, clipped
        {"name": "adamw32 resnet50 first", "op": "adamw32", "model": "resnet50", "param": "f32", "grad": "f32", "shift": 0, "clip": True, "start": 0},
        # a client's local step on the embeddings and one block of a language model, all in 16 bits
        {"name": "adamw32 slice bf16", "op": "adamw32", "model": "gpt2-medium-slice", "param": "bf16", "grad": "bf16", "shift": 0, "clip": False, "start": 1000},
        # adapters: hundreds of small odd tensors, 32-bit weights with fp16 gradients under a loss scale
        {"name": "adamw32 adapters", "op": "adamw32", "count": 384, "total": 6_000_011, "mix": 5, "param": "f32", "grad": "f16", "shift": 3, "clip": True, "start": 40},
        # a server's step on a language model
        {"name": "adamw32 gpt2-medium", "op": "adamw32", "model": "gpt2-medium", "param": "f32", "grad": "f32", "shift": 0, "clip": True, "start": 1000},
        # the head with 8-bit states
        {"name": "adamw8 head", "op": "adamw8", "model": "head", "param": "f32", "grad": "f32", "shift": 0, "clip": False, "start": 1000},
        # a network's first step, its update off its alignment
        {"name": "adamw8 resnet18 first", "op": "adamw8", "model": "resnet18", "param": "f32", "grad": "f32", "shift": 1, "clip": True, "start": 0},
        # a client that saves memory: everything in 16 and 8 bits
        {"name": "adamw8 slice bf16", "op": "adamw8", "model": "gpt2-medium-slice", "param": "bf16", "grad": "bf16", "shift": 0, "clip": False, "start": 1000},
        # a server that keeps the states of a language model in 8 bits
        {"name": "adamw8 gpt2-medium", "op": "adamw8", "model": "gpt2-medium", "param": "f32", "grad": "f32", "shift": 0, "clip": True, "start": 1000},
    ]


def draw(rng):
    op = rng.choice(["norm", "adamw32", "adamw8"])
    total = int(math.exp(rng.uniform(0.0, math.log(3e8))))
    count = min(total, int(math.exp(rng.uniform(0.0, math.log(600.0)))))
    case = {"op": op, "count": count, "total": total, "mix": rng.randrange(1 << 30), "grad": rng.choice(list(TYPES)), "shift": rng.choice([0, 0, 0, 1, 2, 5])}
    if op != "norm":
        case.update(param=rng.choice(list(TYPES)), clip=rng.random() < 0.5, start=rng.choice([0, 7, 1000, 200_000]))
    return case


def _residual_net(blocks, bottleneck):
    out, width, expansion, last = [(64, 3, 3, 3), (64,), (64,)], 64, 4 if bottleneck else 1, 64
    for stage, n in enumerate(blocks):
        width = 64 << stage
        for i in range(n):
            wide = width * expansion
            convs = [(width, last, 1, 1), (width, width, 3, 3), (wide, width, 1, 1)] if bottleneck else [(width, last, 3, 3), (width, width, 3, 3)]
            if last != wide or (i == 0 and stage > 0):
                convs.append((wide, last, 1, 1))
            for c in convs:
                out += [c, (c[0],), (c[0],)]
            last = wide
    return out + [(10, last), (10,)]


def _language_model(layers):
    d, vocab, positions = 1024, 50257, 1024
    block = [(d,), (d,), (d, 3 * d), (3 * d,), (d, d), (d,), (d,), (d,), (d, 4 * d), (4 * d,), (4 * d, d), (d,)]
    return [(vocab, d), (positions, d)] + block * layers + [(d,), (d,)]


def sizes(case):
    """Element counts of the tensors with weight decay, and of those without."""
    if "model" in case:
        shapes = {"head": lambda: [(10, 512), (10,)], "resnet18": lambda: _residual_net((2, 2, 2, 2), False), "resnet50": lambda: _residual_net((3, 4, 6, 3), True), "gpt2-medium": lambda: _language_model(24), "gpt2-medium-slice": lambda: _language_model(1)}[case["model"]]()
        return [math.prod(s) for s in shapes if len(s) > 1], [math.prod(s) for s in shapes if len(s) == 1]
    rng = random.Random(case["mix"])
    weights = [math.exp(rng.gauss(0.0, 2.0)) for _ in range(case["count"])]
    ns = [max(1, int(case["total"] * w / sum(weights))) for w in weights]
    first = (len(ns) + 1) // 2
    return ns[:first], ns[first:]


def work(case):
    n = sum(map(sum, sizes(case)))
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "norm":
        return {"bytes": n * size[case["grad"]] + 8, "flops": 2 * n}
    state = 16 * n if case["op"] == "adamw32" else 4 * n + 16 * -(-n // BLOCK)
    return {"bytes": n * (2 * size[case["param"]] + size[case["grad"]]) + state + 16, "flops": (14 + 2 * case["clip"]) * n}


# --- inputs --------------------------------------------------------------

def prepare(case, seed):
    decayed, others = sizes(case)
    ns = decayed + others
    offsets, total = [], 0
    for n in ns:
        offsets.append(total)
        total += -(-n // BLOCK) * BLOCK
    split = offsets[len(decayed)] if others else total
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    blocks = total // BLOCK

    def normal(n):
        return torch.randn(n, device=dev, generator=gen)

    def padded(flat):
        for n, o in zip(ns, offsets):
            if n % BLOCK:
                flat[o + n:o + -(-n // BLOCK) * BLOCK] = 0
        return flat

    def shifted(flat, kind):
        buf = torch.zeros(total + case["shift"], dtype=TYPES[kind], device=dev)
        buf[case["shift"]:] = padded(flat)
        return buf[case["shift"]:]

    # gradients of very different sizes from block to block, one block in eight without any
    size = 1e-3 * torch.exp(normal(blocks)) * (torch.rand(blocks, device=dev, generator=gen) > 0.125)
    scale = 1024.0 if case["grad"] == "f16" else 1.0
    g = shifted((normal(total).view(blocks, BLOCK) * (scale * size[:, None])).view(-1), case["grad"])
    s = {"case": case, "g": g, "scale": -1.0 / scale, "split": split, "max_norm": 1.0}
    if case["op"] != "norm":
        s["p"] = shifted(normal(total) * 0.02, case["param"])
        s["step"] = torch.full((1,), case["start"], dtype=torch.int64, device=dev)
        live = float(case["start"] > 0)
        if case["op"] == "adamw32":
            size = (size + 1e-5) * live
            s["m"] = padded((normal(total).view(blocks, BLOCK) * (0.3 * size[:, None])).view(-1))
            s["v"] = padded(((normal(total).view(blocks, BLOCK) * size[:, None]) ** 2 + 1e-3 * size[:, None] ** 2).view(-1))
        else:
            s["m"] = padded((normal(total) * (100.0 * live)).clamp(-448, 448)).to(torch.float8_e4m3fn)
            s["v"] = padded((normal(total).abs() * (150.0 * live) + live).clamp(max=448)).to(torch.float8_e4m3fn)
            s["m_scale"] = (size + 1e-5) * (0.003 * live)
            s["v_scale"] = (size + 1e-5) * (0.007 * live)
    if own:
        from compressor_b200.optim import AdamW, GradNorm
        views = [slice(o, o + n) for n, o in zip(ns, offsets)]
        grads = [s["g"][w] for w in views]
        if case["op"] == "norm" or case["clip"]:
            s["norm"] = GradNorm(grads)
        if case["op"] != "norm":
            s["opt"] = AdamW([s["p"][w] for w in views], grads, lr=LR, betas=(BETA1, BETA2), eps=EPS,
                             weight_decay=[DECAY] * len(decayed) + [0.0] * len(others),
                             state_bits=32 if case["op"] == "adamw32" else 8, seed=SEED)
            s["opt"].load_state({k: s.pop(k) for k in ("m", "v", "m_scale", "v_scale", "step") if k in s})
    return s


# --- one pass ------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        clip = s["norm"](max_norm=s["max_norm"], grad_scale=s["scale"]) if "norm" in s else None
        if c["op"] == "norm":
            return clip
        opt = s["opt"]
        opt.step(grad_scale=s["scale"], clip=clip)
        return {"p": s["p"], **opt.state, "clip": clip}
    clip = plain_norm(s["g"], s["max_norm"], s["scale"]) if c["op"] == "norm" or c["clip"] else None
    if c["op"] == "norm":
        return clip
    (plain_adamw32 if c["op"] == "adamw32" else plain_adamw8)(s, clip)
    return {**{k: s[k] for k in ("p", "m", "v", "m_scale", "v_scale", "step") if k in s}, "clip": clip}


def plain_norm(g, max_norm, scale):
    """[norm of scale * g, the factor that brings it down to max_norm]."""
    norm = g.double().square().sum().sqrt() * abs(scale)
    factor = torch.where(norm > max_norm, max_norm / norm, torch.ones_like(norm))
    factor = torch.where(norm.isfinite(), factor, torch.full_like(norm, float("nan")))
    return torch.stack([norm, factor]).float()


def _update(s, m, root):
    """The parameters' step, from the first moment and the root of the second after it."""
    t = s["step"].double()
    size = (LR / (1 - BETA1 ** t)).float()
    bias = (1 / (1 - BETA2 ** t).sqrt()).float()
    p = s["p"].float()
    p[:s["split"]] *= 1 - LR * DECAY
    s["p"].copy_(p - size * (m / (root * bias + EPS)))


def _scaled(s, clip):
    return s["g"].float() * (s["scale"] if clip is None else clip[1] * s["scale"])


def plain_adamw32(s, clip):
    s["step"] += 1
    g = _scaled(s, clip)
    m = s["m"] * BETA1 + g * (1 - BETA1)
    v = s["v"] * BETA2 + (g * g) * (1 - BETA2)
    _update(s, m, v.sqrt())
    s["m"].copy_(m)
    s["v"].copy_(v)


def _mix(x):
    """A 32-bit avalanche of shifts and odd products, on int32 values."""
    x = (x ^ ((x >> 16) & 0xFFFF)) * -2048144789
    x = (x ^ ((x >> 13) & 0x7FFFF)) * -1028477387
    return x ^ ((x >> 16) & 0xFFFF)


def _dither(step, n):
    """One random 32-bit word for each position."""
    key = _mix(torch.full_like(step, (SEED & 0xFFFFFFFF) ^ 0x9E3779B9).to(torch.int32))
    key = _mix(key ^ (SEED >> 32))
    key = _mix(_mix(key ^ step.to(torch.int32)))  # positions under 2^32: their high word is 0
    return _mix(key ^ torch.arange(n, dtype=torch.int32, device=step.device))


def _encode(x, dither, least):
    """e4m3 values (held as float8) and scales of non-negative x [blocks, 256]: in units of 2^-9 or of the value's
    last bit, the float32 bits shifted down to e4m3's are rounded up where the dither carries."""
    top = x.amax(1)
    live = top >= 2.0 ** -100
    up = torch.where(live, torch.div(torch.full_like(top, 448.0), top), torch.zeros_like(top))
    y = (x * up[:, None]) * 2.0 ** -120
    code = ((y.view(torch.int32) + dither) >> 20).clamp(max=126)
    code = torch.maximum(code, ((x > 0) & live[:, None]).to(torch.int32) * least)
    return code, torch.where(live, top * (1 / 448.0), torch.zeros_like(top))


def plain_adamw8(s, clip):
    s["step"] += 1
    g = _scaled(s, clip).view(-1, BLOCK)
    m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]) * BETA1 + g * (1 - BETA1)
    v = s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]
    v = (v * v) * BETA2 + (g * g) * (1 - BETA2)
    root = v.sqrt()
    _update(s, m.view(-1), root.view(-1))
    word = _dither(s["step"], m.numel()).view(-1, BLOCK)
    code, scale = _encode(m.abs(), (word >> 12) & 0xFFFFF, 0)
    code = code | ((m < 0).to(torch.int32) * 128)
    s["m"].copy_(code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1))
    s["m_scale"].copy_(scale)
    code, scale = _encode(root, word & 0xFFFFF, 1)
    s["v"].copy_(code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1))
    s["v_scale"].copy_(scale)


# --- the definition in 64 bits -------------------------------------------

def _e4m3(x, chance, least):
    """Values that e4m3 holds next below or above x (0 <= x <= 448), above where the chance in [0, 1) is large enough."""
    gap = torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0 ** -6))) - 3)
    value = (torch.floor(x / gap + chance) * gap).clamp(max=448.0)
    return torch.where(x > 0, value.clamp(min=least), value)


def _words(step, n, device):
    """The random words, in 64-bit whole numbers."""
    full = 0xFFFFFFFF

    def avalanche(x):
        x = ((x ^ (x >> 16)) * 0x85EBCA6B) & full
        x = ((x ^ (x >> 13)) * 0xC2B2AE35) & full
        return x ^ (x >> 16)

    key = avalanche((SEED & full) ^ 0x9E3779B9)
    for part in (SEED >> 32, step & full, 0):
        key = avalanche(key ^ part)
    return avalanche(torch.arange(n, dtype=torch.int64, device=device) ^ key)


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    g = s["g"].double() * s["scale"]
    norm = torch.linalg.vector_norm(g)
    factor = s["max_norm"] / norm if norm > s["max_norm"] else torch.ones_like(norm)
    out = torch.stack([norm, factor])
    if case["op"] == "norm":
        return out
    if case["clip"]:
        g *= factor
    step = case["start"] + 1
    m, v = s["m"].double(), s["v"].double()
    if case["op"] == "adamw8":
        m = m * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    del g
    p = s["p"].double()
    p[:s["split"]] -= LR * DECAY * p[:s["split"]]
    p -= LR * (m / (1 - BETA1 ** step)) / ((v / (1 - BETA2 ** step)).sqrt() + EPS)
    done = {"p": p, "m": m, "v": v, "step": s["step"] + 1, "clip": out if case["clip"] else None}
    if case["op"] == "adamw8":
        word = _words(step, m.numel(), m.device)
        for key, x, chance, least in (("m", m, word >> 12, 0.0), ("v", v.sqrt(), word & 0xFFFFF, 2.0 ** -9)):
            top = x.view(-1, BLOCK).abs().amax(1)
            unit = (top / 448).repeat_interleave(BLOCK)
            held = torch.where(unit > 0, x.abs() / unit, torch.zeros_like(x))
            done[key] = _e4m3(held, chance.double() / 2.0 ** 20, least) * x.sign()
            done[key + "_scale"] = top / 448
    return done
