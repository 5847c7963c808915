"""Checks of the optimiser entry points (falcom_norm_*, falcom_adamw_*)
through the C ABI against plain 64-bit formulas, on any memory the library
under test can address: the GPU tests and the kernel-emulation tests run the
same checks.

A backend has upload(array) -> handle (with .ptr), download(handle) -> array
and lib.  Every array is placed between guard bytes that must not change.

Tolerances count roundings.  u = 2^-24 is half a float32 step relative to a
value; a float32 expression of k operations on exact inputs is within about k
u of its terms' magnitudes.  Constants (betas, the factor, decay, size, bias)
carry one rounding each.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from compressor_b200 import abi

U = 2.0 ** -24
BLOCK = abi.ADAMW_BLOCK
GUARD = 64


# ------------------------------------------------------------ element types
def round_to(x, kind):
    """float64 / float32 values as the storage of `kind`, rounded to nearest even."""
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return x
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32)
    r = ((b + np.uint32(0x7FFF) + ((b >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def widen(s, kind):
    """Storage of `kind` as float32."""
    if kind == "bf16":
        return (s.astype(np.uint32) << np.uint32(16)).view(np.float32)
    return s.astype(np.float32)


CODE = {"f32": abi.TYPE_F32, "bf16": abi.TYPE_BF16, "f16": abi.TYPE_F16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}   # half the smallest step


def e4m3(code):
    """Values of e4m3 codes, from the format's definition."""
    code = np.asarray(code, np.int64)
    e, f = (code >> 3) & 15, code & 7
    v = np.where(e > 0, (1 + f / 8.0) * 2.0 ** (e - 7.0), f / 8.0 * 2.0 ** -6)
    return np.where(code & 0x80, -v, v)


def e4m3_floor(y, chance):
    """Code of y in [0, 448] rounded up where its place between two
    neighbouring values plus `chance` reaches one."""
    y = np.asarray(y, np.float64)
    e = np.maximum(np.floor(np.log2(np.maximum(y, 2.0 ** -30))), -6)
    gap = 2.0 ** (e - 3)
    k = np.floor(y / gap + chance)           # 8..16 steps of a normal value, 0..8 of a subnormal one
    return np.minimum((e + 6) * 8 + k, 126).astype(np.int64)


def mix(x):
    x = np.asarray(x, np.uint64) & np.uint64(0xFFFFFFFF)
    m32 = np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x85EBCA6B)) & m32
    x = ((x ^ (x >> np.uint64(13))) * np.uint64(0xC2B2AE35)) & m32
    return x ^ (x >> np.uint64(16))


def words(seed, step, pos):
    """The dither of 64-bit positions."""
    pos = np.asarray(pos, np.uint64)
    key = mix(np.uint64((seed & 0xFFFFFFFF) ^ 0x9E3779B9))
    key = mix(key ^ np.uint64(seed >> 32))
    key = mix(key ^ np.uint64(step & 0xFFFFFFFF))
    key = mix(key ^ (pos >> np.uint64(32)))
    return mix(key ^ (pos & np.uint64(0xFFFFFFFF)))


# ----------------------------------------------------------------- placing
class Placed:
    """`arr` in backend memory, `shift` bytes past a 256-byte boundary, guards around it."""

    def __init__(self, backend, arr, shift=0):
        self.b, self.arr, self.dtype, self.n = backend, arr, arr.dtype, arr.size
        self.lead = 256 + shift
        raw = np.full(self.lead + arr.nbytes + GUARD, 0x5A, np.uint8)
        raw[self.lead:self.lead + arr.nbytes] = arr.reshape(-1).view(np.uint8)
        self.h = backend.upload(raw)
        self.ptr = self.h.ptr + self.lead

    def get(self):
        raw = self.b.download(self.h)
        end = self.lead + self.n * self.dtype.itemsize
        assert (raw[:self.lead] == 0x5A).all() and (raw[end:] == 0x5A).all(), "bytes around the array changed"
        return raw[self.lead:end].copy().view(self.dtype)


def c_array(kind, values):
    values = list(values)
    return (kind * max(1, len(values)))(*values)


# -------------------------------------------------------------------- norm
def check_norm(backend, arrays, kinds, shifts, scale=1.0, max_norm=math.inf, runs=2):
    """Norm and coefficient against 64-bit sums; the same bits on every run."""
    lib = backend.lib
    placed = [Placed(backend, round_to(a, k), SIZE[k] * s) for a, k, s in zip(arrays, kinds, shifts)]
    plan = lib.falcom_norm_create(c_array(ctypes.c_void_p, [p.ptr for p in placed]),
                                  c_array(ctypes.c_size_t, [p.n for p in placed]),
                                  c_array(ctypes.c_int, [CODE[k] for k in kinds]), len(placed))
    assert plan
    work = Placed(backend, np.zeros(lib.falcom_norm_work_bytes(plan), np.uint8))
    got = []
    for _ in range(runs):
        out = Placed(backend, np.full(2, 7, np.float32))
        assert lib.falcom_norm_run(plan, scale, max_norm, out.ptr, work.ptr, backend.stream) == 0
        got.append(out.get())
    assert all((g.view(np.uint32) == got[0].view(np.uint32)).all() for g in got)
    assert not work.get()[:4].any()           # ready for the next call
    lib.falcom_norm_destroy(plan)
    xs = [widen(round_to(a, k), k).astype(np.float64) for a, k in zip(arrays, kinds)]
    with np.errstate(invalid="ignore"):
        want = math.sqrt(float(sum((x * x).sum() for x in xs))) * abs(scale)
    norm, coef = float(got[0][0]), float(got[0][1])
    if not math.isfinite(want):
        assert math.isnan(coef) and (math.isnan(norm) if math.isnan(want) else norm == want)
        return got[0]
    # 64-bit sums in another order, then one rounding to float32 (or above float32's range)
    if want < 3.4e38:
        assert abs(norm - want) <= want * (U + 1e-12) + 2.0 ** -150, (norm, want)
    else:
        assert norm == math.inf
    c = max_norm / want if want > max_norm else 1.0
    assert abs(coef - c) <= c * (U + 1e-12) + 2.0 ** -150, (coef, c)
    return got[0]


# ------------------------------------------------------------------- AdamW
class Tensor:
    """One tensor of a case: float64 copies of what the device holds, and the placed arrays."""

    def __init__(self, backend, rng, n, pk, gk, bits, decay, shift=0, state_shift=0, g=None, start=True):
        self.n, self.pk, self.gk, self.bits, self.decay = n, pk, gk, bits, decay
        self.blocks = -(-n // BLOCK)
        p = rng.standard_normal(n) * 0.05
        size = np.repeat(np.exp(rng.standard_normal(self.blocks) * 2) * 1e-3, BLOCK)[:n]
        g = rng.standard_normal(n) * size if g is None else g
        ps, gs = round_to(p, pk), round_to(g, gk)
        self.p, self.g = widen(ps, pk).astype(np.float64), widen(gs, gk).astype(np.float64)
        self.dp = Placed(backend, ps, SIZE[pk] * shift)
        self.dg = Placed(backend, gs, SIZE[gk] * shift)
        on = float(start)
        if bits == 32:
            m = (rng.standard_normal(n) * size * 0.3 * on).astype(np.float32)
            v = ((size * rng.standard_normal(n)) ** 2 * on).astype(np.float32)
            self.dm, self.dv = Placed(backend, m, 4 * state_shift), Placed(backend, v, 4 * state_shift)
            self.dms = self.dvs = None
        else:
            m = rng.integers(0, 127, n).astype(np.uint8) | (rng.integers(0, 2, n) << 7).astype(np.uint8)
            v = rng.integers(1, 127, n).astype(np.uint8)
            m, v = m * np.uint8(on), v * np.uint8(on)
            ms = (np.exp(rng.standard_normal(self.blocks)) * 1e-5 * on).astype(np.float32)
            vs = (np.exp(rng.standard_normal(self.blocks)) * 1e-5 * on).astype(np.float32)
            self.dm, self.dv = Placed(backend, m, state_shift), Placed(backend, v, state_shift)
            self.dms, self.dvs = Placed(backend, ms), Placed(backend, vs)
        self.refresh()

    def refresh(self):
        """Float64 state from the device."""
        self.p = widen(self.dp.get(), self.pk).astype(np.float64)
        if self.bits == 32:
            self.m, self.v = self.dm.get().astype(np.float64), self.dv.get().astype(np.float64)
        else:
            rep = lambda s: np.repeat(s.get().astype(np.float64), BLOCK)[:self.n]  # noqa: E731
            self.m = e4m3(self.dm.get()) * rep(self.dms)
            self.v = (e4m3(self.dv.get()) * rep(self.dvs)) ** 2

    def c(self):
        t = abi.AdamWTensorC()
        t.param, t.grad, t.m, t.v = self.dp.ptr, self.dg.ptr, self.dm.ptr, self.dv.ptr
        if self.bits == 8:
            t.m_scale, t.v_scale = self.dms.ptr, self.dvs.ptr
        t.n, t.param_type, t.grad_type, t.weight_decay = self.n, CODE[self.pk], CODE[self.gk], self.decay
        return t


HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, seed=0x1234567890ABCDEF)


def make_args(**kw):
    a = abi.AdamWArgsC()
    for k, v in {**HYPER, **kw}.items():
        setattr(a, k, v)
    return a


def check_block(y, mag_code, chance, least, slack):
    """Codes of y (64-bit, in units of the block's scale) for a dither known
    exactly: between the codes of y a few roundings lower and higher."""
    lo = np.maximum(e4m3_floor(y * (1 - slack) - 2.0 ** -29, chance), 0)
    hi = e4m3_floor(np.minimum(y * (1 + slack) + 2.0 ** -29, 448), chance)
    lo, hi = np.maximum(lo, least), np.maximum(hi, least)
    bad = (mag_code < lo) | (mag_code > hi)
    assert not bad.any(), (np.flatnonzero(bad)[:5], y[bad][:5], mag_code[bad][:5], lo[bad][:5], hi[bad][:5])


def check_step(tensors, t, hyper, factor=1.0):
    """The tensors on the device after step t against 64-bit formulas from
    their float64 state before it (then refreshed)."""
    f = float(np.float32(hyper["grad_scale"])) * factor
    b1, b2, lr, eps = hyper["beta1"], hyper["beta2"], hyper["lr"], hyper["eps"]
    pos = 0
    for k, x in enumerate(tensors):
        old_p, old_m, old_v = x.p, x.m, x.v
        g = x.g * f
        m = b1 * old_m + (1 - b1) * g
        v = b2 * old_v + (1 - b2) * g * g
        root = np.sqrt(v)
        denom = root / math.sqrt(1 - b2 ** t) + eps
        size = lr / (1 - b1 ** t)
        p = old_p * (1 - lr * x.decay) - size * m / denom
        # m: each product has a rounded constant and a rounding of its own, the
        # gradient two more (factor, scaling), the old 8-bit moment one, then the sum
        terms_m = np.abs(b1 * old_m) + np.abs((1 - b1) * g)
        em = 7 * U * terms_m + 2.0 ** -148
        # v: g' squared doubles its two roundings, plus square, constant, product, sum (8-bit: root squared)
        ev = 10 * U * v + 2.0 ** -147
        # root: half of v's relative error and its own; near 0 the absolute error's root
        er = np.where(v > 2.0 ** -120, 6 * U * root, np.sqrt(ev))
        # root * bias + eps: bias, product, eps, sum; quotient, size, product
        ed = er / math.sqrt(1 - b2 ** t) + 4 * U * denom
        eu = size * (em / denom + np.abs(m) / denom * (ed / denom + 4 * U))
        ep = 4 * U * np.abs(old_p) + eu + 2 * U * np.abs(p) + 2.0 ** -148
        ep = ep + HALF_STEP[x.pk] * (np.abs(p) + ep) + TINY[x.pk]
        before = x.n
        x.refresh()
        assert x.n == before
        bad = ~(np.abs(x.p - p) <= ep)
        assert not bad.any(), (k, "p", np.flatnonzero(bad)[:5], x.p[bad][:5], p[bad][:5], ep[bad][:5])
        if x.bits == 32:
            assert (np.abs(x.m - m) <= em).all(), (k, "m")
            assert (np.abs(x.v - v) <= ev).all(), (k, "v")
        else:
            w = words(hyper["seed"], t, np.arange(pos, pos + x.n, dtype=np.uint64)).astype(np.int64)
            for name, val, err, codes, scales, chance in (
                    ("m", m, em, x.dm.get(), x.dms.get(), w >> 12),
                    ("v", root, er, x.dv.get(), x.dvs.get(), w & 0xFFFFF)):
                pad = np.zeros(x.blocks * BLOCK)
                pad[:x.n] = np.abs(val)
                top = pad.reshape(-1, BLOCK).max(1)
                perr = np.zeros(x.blocks * BLOCK)
                perr[:x.n] = err
                terr = perr.reshape(-1, BLOCK).max(1)
                live = top >= 2.0 ** -99
                dead = top < 2.0 ** -101
                assert (live | dead).all()
                assert (np.abs(scales - top / 448) <= terr / 448 + 3 * U * top / 448)[live].all(), (k, name)
                assert (scales[dead] == 0).all()
                c = codes.astype(np.int64)
                each = np.repeat(live, BLOCK)[:x.n]
                assert (c[~each] & 0x7F == 0).all()
                if name == "m":
                    sure = each & (np.abs(val) > err) & (c & 0x7F > 0)
                    assert ((c[sure] >> 7) == (val[sure] < 0)).all()
                else:
                    assert (c < 128).all()
                    assert (c[each & (old_v > 0)] > 0).all()
                tops = np.repeat(np.maximum(top, 1e-300), BLOCK)[:x.n]
                y = np.abs(val) / tops * 448
                # the value's error, its block maximum's, and three roundings of scaling
                with np.errstate(divide="ignore", invalid="ignore"):
                    rel = np.where(val != 0, err / np.abs(np.where(val == 0, 1, val)), 0)
                slack = np.minimum(rel + np.repeat(terr / np.maximum(top, 1e-300), BLOCK)[:x.n] + 4 * U, 1.0)
                least = ((name == "v") & (np.abs(val) > 0) & each).astype(np.int64)
                exact0 = (val == 0)
                assert (c[exact0] & 0x7F == 0).all() or name == "m"
                s = each & ~exact0
                check_block(y[s], c[s] & 0x7F, chance[s] / 2.0 ** 20, least[s], slack[s])
        pos += x.blocks * BLOCK


def run_adamw(backend, tensors, bits, steps=3, start=0, clip=None, lr_device=None, **kw):
    """`steps` steps of one plan, each checked; returns the counter."""
    lib = backend.lib
    hyper = {**HYPER, **kw}
    counter = Placed(backend, np.array([start], np.int64))
    table = c_array(abi.AdamWTensorC, [x.c() for x in tensors])
    plan = lib.falcom_adamw_create(table, len(tensors), bits, counter.ptr)
    assert plan
    args = make_args(**kw)
    factor = 1.0
    if clip is not None:
        dclip = Placed(backend, np.array([1.0, clip], np.float32))
        args.clip = dclip.ptr
        factor = float(np.float32(clip))
    if lr_device is not None:
        dlr = Placed(backend, np.array([lr_device], np.float32))
        args.lr_device = dlr.ptr
        hyper["lr"] = float(np.float32(lr_device))
    for i in range(steps):
        assert lib.falcom_adamw_step(plan, ctypes.byref(args), backend.stream) == 0
        backend.sync()
        assert int(counter.get()[0]) == start + i + 1
        check_step(tensors, start + i + 1, hyper, factor)
    lib.falcom_adamw_destroy(plan)
    for x in tensors:
        assert (widen(x.dg.get(), x.gk).astype(np.float64) == x.g).all()   # gradients are only read


# ---------------------------------------------------------- shared case lists
NORM_CASES = {
    "one": ([1], ["f32"], [0]),
    "none": ([], [], []),
    "empty tensors": ([0, 5, 0], ["f32", "bf16", "f16"], [0, 0, 0]),
    "odd": ([255, 256, 257, 2047, 2049, 4097, 3], ["f32"] * 7, [0, 1, 2, 3, 0, 0, 1]),
    "16 bits": ([1, 7, 8, 9, 2048, 5000, 4096], ["bf16", "f16"] * 3 + ["bf16"], [0, 1, 5, 0, 0, 3, 0]),
    "many": ([1 + (i * 37) % 600 for i in range(90)], ["f32", "bf16", "f16"] * 30, [i % 5 for i in range(90)]),
    "more units than warps": ([2048 * 150 + 17, 2048 * 40], ["f32", "bf16"], [0, 0]),
}

ADAMW_CASES = {
    "one": ([1], [0], [0]),
    "odd": ([255, 256, 257, 1023, 1025, 3, 0, 2051], [0, 0, 1, 0, 2, 0, 0, 3], [0, 0, 0, 1, 0, 0, 0, 2]),
    "units": ([1024 * 90 + 300, 512], [0, 0], [0, 0]),
    "shifted": ([5000, 700], [1, 3], [1, 0]),
}


def case_tensors(backend, name, bits, pk, gk, seed=0, start=True):
    ns, shifts, state_shifts = ADAMW_CASES[name]
    rng = np.random.default_rng(seed)
    return [Tensor(backend, rng, n, pk, gk, bits, 0.1 * (i % 3), s, q, start=start)
            for i, (n, s, q) in enumerate(zip(ns, shifts, state_shifts))]
