"""8-bit AdamW states bit for bit: one step from states set directly, with
the largest first moment and the largest root of the second chosen apart from
each other in every block, against the formulas in float32, each operation
rounded once (include/falcom_b200.h).  Backends as in optim_cases.py.

With beta1 = 1/2 and beta2 = 1/4 and no gradient both moments' values halve
exactly (the root of a rounded square is the value again, as long as the
square is a normal number), and a largest code of 256, a power of two, makes
a block's maximum any float32 that is wanted.
"""
from __future__ import annotations

import ctypes

import numpy as np

from compressor_b200 import abi
from tests import optim_cases as oc

F = np.float32
BLOCK = oc.BLOCK
CODE_256 = 0x78
BELOW_2_14 = float(np.nextafter(F(2.0 ** 14), F(0)))
# maxima after the step; squares of the roots stay normal numbers
M_TOPS = [2.0 ** -90, 1e-8, 1e-6, 1.0, BELOW_2_14, 2.0 ** 14, 3e4, 2.0 ** 40, 2.0 ** 90]
V_TOPS = [2.0 ** -50, 1e-8, 1e-6, 1.0, BELOW_2_14, 2.0 ** 14, 3e4, 2.0 ** 40]


def codes_of(x, chance, least):
    """Codes and scales of magnitudes x [blocks, 256]: |x| * (448 / max), the
    quotient rounded once and so the product, which is held to multiples of
    2^-29 where it lies below 2^-6 (float32's own subnormals, 2^120 down)."""
    top = x.max(1)
    live = (top >= F(2.0 ** -100)) & (top < F(2.0 ** 100))
    with np.errstate(divide="ignore", invalid="ignore"):
        up = np.where(live, F(448) / top, F(0))
    y = (x.astype(np.float64) * up[:, None].astype(np.float64) * 2.0 ** -120).astype(F)   # exact until here
    code = np.minimum((y.view(np.uint32) + chance) >> 20, 126)
    code = np.maximum(code, ((x > 0) & live[:, None]) * least)
    return code.astype(np.uint8), np.where(live, top * F(1 / 448.0), F(0))


# gradients of an element whose states are zero: roots so small that a
# 2^-100th of either is no float32 number
VANISHING = [2.0 ** -50, 2.0 ** -55, 2.0 ** -62]


def check_maxima(backend, pk, gk, shift=0, state_shift=0, gradient=0.0):
    """One step over every pair of maxima.  `gradient`: of one element, whose
    states are zero, in the blocks whose roots reach 1."""
    pairs = [(a, b) for a in M_TOPS for b in V_TOPS]
    blocks = len(pairs) + 1
    n = blocks * BLOCK - 100                       # the last block is short
    rng = np.random.default_rng(11)
    mc = rng.integers(0, CODE_256 + 1, (blocks, BLOCK)).astype(np.uint8)
    vc = rng.integers(0, CODE_256 + 1, (blocks, BLOCK)).astype(np.uint8)
    mc[:, 7], vc[:, 9] = CODE_256, CODE_256
    mc[:, 20:30], vc[:, 25:40] = 0, 0
    mc |= (rng.integers(0, 2, mc.shape) * 128 * (mc > 0)).astype(np.uint8)
    tops = np.array(pairs + [(3e4, 1e-6)])
    ms = (tops[:, 0] / 128).astype(F)              # 256 * scale / 2 is the maximum
    vs = (tops[:, 1] / 128).astype(F)
    g = np.zeros((blocks, BLOCK))
    g[:len(pairs), 28] = gradient * (tops[:len(pairs), 1] >= 1.0)
    gs = oc.round_to(g.reshape(-1)[:n], gk)
    ps = oc.round_to(np.zeros(n), pk)
    dp, dg = oc.Placed(backend, ps, oc.SIZE[pk] * shift), oc.Placed(backend, gs, oc.SIZE[gk] * shift)
    dm, dv = (oc.Placed(backend, c.reshape(-1)[:n].copy(), state_shift) for c in (mc, vc))
    dms, dvs = oc.Placed(backend, ms), oc.Placed(backend, vs)
    step = oc.Placed(backend, np.zeros(1, np.int64))
    t = abi.AdamWTensorC(param=dp.ptr, grad=dg.ptr, m=dm.ptr, v=dv.ptr, m_scale=dms.ptr, v_scale=dvs.ptr, n=n,
                         param_type=oc.CODE[pk], grad_type=oc.CODE[gk], weight_decay=0.0)
    plan = backend.lib.falcom_adamw_create(oc.c_array(abi.AdamWTensorC, [t]), 1, 8, step.ptr)
    assert plan
    seed = 0xFEDCBA9876543210
    args = oc.make_args(beta1=0.5, beta2=0.25, lr=1e-3, seed=seed)
    assert backend.lib.falcom_adamw_step(plan, ctypes.byref(args), backend.stream) == 0
    backend.sync()
    backend.lib.falcom_adamw_destroy(plan)

    g = np.zeros(blocks * BLOCK, F)
    g[:n] = oc.widen(gs, gk)
    g = g.reshape(blocks, BLOCK)
    keep = (np.arange(blocks * BLOCK) < n).reshape(blocks, BLOCK)
    sign = np.where(mc & 0x80, F(-1), F(1))
    m = (oc.e4m3(mc & 0x7F).astype(F) * sign * ms[:, None]) * F(0.5) + g * F(0.5)
    r = oc.e4m3(vc).astype(F) * vs[:, None]
    root = np.sqrt((r * r) * F(0.25) + (g * g) * F(0.75))
    m, root = np.where(keep, m, F(0)), np.where(keep, root, F(0))
    full = (keep.all(1)) & (g == 0).all(1)
    assert (np.abs(m).max(1)[full] == F(tops[full, 0])).all() and (root.max(1)[full] == F(tops[full, 1])).all()
    w = oc.words(seed, 1, np.arange(blocks * BLOCK, dtype=np.uint64)).astype(np.uint32).reshape(blocks, BLOCK)
    for what, got, scales, (code, scale), signed in (
            ("m", dm, dms, codes_of(np.abs(m), w >> np.uint32(12), 0), True),
            ("v", dv, dvs, codes_of(root, w & np.uint32(0xFFFFF), 1), False)):
        have = np.zeros(blocks * BLOCK, np.uint8)
        have[:n] = got.get()
        have = have.reshape(blocks, BLOCK)
        assert (scales.get() == scale).all(), what
        bad = ((have & 0x7F) != code) & keep
        if not signed:
            # a v' under 2^-100 may count as less than it is: with 2^-50 at
            # the top and codes down to 2^-17 of it, v' reaches 2^-134
            low = (root > 0) & (root < F(2.0 ** -50))
            bad &= ~(low & (have >= 1) & (have <= code))
        assert not bad.any(), (what, [(tuple(tops[b]), int(have[b, e]), int(code[b, e])) for b, e in np.argwhere(bad)[:6]],
                               int(bad.sum()))
        if signed:
            assert ((have >> 7) == (m < 0))[code > 0].all()
        else:
            assert (have < 128).all()
    assert np.isfinite(oc.widen(dp.get(), pk)).all()


# parameter and gradient types, elements off alignment, states' bytes off alignment
LAYOUTS = {
    "two runs of four": ("f32", "f32", 0, 0),
    "two runs of four, mixed": ("f32", "bf16", 0, 0),
    "runs of eight": ("bf16", "bf16", 0, 0),
    "shifted": ("f32", "f32", 1, 0),
    "shifted, 16 bits": ("bf16", "bf16", 3, 0),
    "ragged": ("f32", "f32", 0, 1),
    "ragged, 16 bits": ("bf16", "bf16", 1, 5),
}
