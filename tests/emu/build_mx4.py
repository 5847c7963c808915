"""Kernel-emulation library of the 4-bit entry points and of dropout (test
infrastructure only, see build.py): mc_mx4.c unchanged, mc_mx4.cu with
mc_mx4_device.h through prep.py's source transform, and a plain sum in place of
the tensor-core kernels (emu_mx4.h).
"""
from __future__ import annotations

import hashlib
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(os.path.dirname(HERE)))
from tests.emu import build as base  # noqa: E402
from tests.emu import prep  # noqa: E402

BUILD = os.path.join(HERE, "_build_mx4")
INPUTS = [os.path.join(base.CSRC, f) for f in ("mc_mx4.c", "mc_mx4.cu", "mc_mx4.h", "mc_mx4_device.h", "mc_call.h", "mc_util.c", "mc_internal.h")] + \
         [os.path.join(base.INCLUDE, "falcom_b200.h")] + \
         [os.path.join(HERE, f) for f in ("emu.h", "emu_optim.h", "emu_mx4.h", "fake_cudart.cpp", "prep.py", "build_mx4.py")]

# host bodies of the inline-PTX helpers
BODIES = {
    "mx_begin": "",
    "mx_mul2": " return make_float2(a.x * b.x, a.y * b.y); ",
    "mx_add2": " return make_float2(a.x + b.x, a.y + b.y); ",
    "mx_mul2_cut": " return make_float2(__fmul_rz(a.x, b.x), __fmul_rz(a.y, b.y)); ",
    "mx_codes8": " uint32_t r = 0; for (int i = 0; i < 8; i++) r |= emu_e2m1(y[i]) << (4 * i); return r; ",
    "mx_code_near": " return emu_e2m1(y); ",
    "larger2": """
    const unsigned infinity = sizeof(T) && std::is_same<T, __half2>::value ? 0x7C00 : 0x7F80;
    return emu_top_half(a, b, infinity) | emu_top_half(a >> 16, b >> 16, infinity) << 16;
""",
}
LAUNCH = """
    static_assert(EMU_TPB == 256, "");
    if (threads != EMU_TPB || cluster != 0) abort();
    (void)s;
    emu_run((int)grid, smem, [&] { kern(args...); });
    return cudaSuccess;
"""
PRODUCT = """
extern "C" int mc_launch_mx_product(const mx_product_launch *L, int type, int sms, void *stream) {
    (void)sms;
    (void)stream;
    const mx_key key = mx_key_of(L->drop.random);
    for (int64_t t = 0; t < L->a.rows; t++)
        for (int64_t n = 0; n < L->b.rows; n++) {
            double sum = 0;
            if (L->x) abort();
            for (int64_t k = 0; k < L->a.cols; k++) sum += emu_mx4_value(L->a, t, k) * emu_mx4_value(L->b, n, k);
            float v = (float)sum;
            if (L->drop.random.on) {
                const uint32_t w = mx_word_at(key, (uint64_t)(t * mx_wide(L->b.rows) + n) / 2);
                v = (n & 1 ? w >> 16 : w & 0xFFFFu) < L->drop.threshold ? 0.0f : v * L->drop.factor;
            }
            if (type == FALCOM_TYPE_F32) mx_from((float *)L->out + t * L->ld + n, v);
            else if (type == FALCOM_TYPE_BF16) mx_from((__nv_bfloat16 *)L->out + t * L->ld + n, v);
            else mx_from((__half *)L->out + t * L->ld + n, v);
        }
    return 0;
}
extern "C" __attribute__((visibility("default"))) uint32_t emu_mx4_gave_up = 0;   // CTAs, for a test to count up
extern "C" int mc_mx_errors(uint32_t *word) { *word = emu_mx4_gave_up; return 0; }
"""


def build() -> str:
    h = hashlib.sha256()
    for f in INPUTS:
        with open(f, "rb") as fh:
            h.update(fh.read())
    out = os.path.join(BUILD, f"libfalcom_mx4_emu_{h.hexdigest()[:16]}.so")
    if os.path.exists(out):
        return out
    os.makedirs(BUILD, exist_ok=True)
    with open(os.path.join(base.CSRC, "mc_mx4_device.h")) as f:
        head = f.read().replace("#pragma once", "")
    with open(os.path.join(base.CSRC, "mc_mx4.cu")) as f:
        src = f.read().replace('#include "mc_mx4_device.h"', head)
    src = re.sub(r"__launch_bounds__\(MX_TPB(?:, (?:[^()]|\([^()]*(?:\([^()]*\))?[^()]*\))*)?\)", "", src)
    src = re.sub(r"extern __shared__ __align__\(\d+\) uint8_t s_tile\[\];", "uint8_t *const s_tile = (uint8_t *)s_stage;", src)
    src = re.sub(r"cudaFuncSetAttribute\(.*?\);", "cudaSuccess;", src, flags=re.S)
    src = re.sub(r"mx_allow\(k_mx_quantize<[^>]*>, smem\)", "cudaSuccess", src)
    for word in ("__host__ ", "__noinline__ ", "__grid_constant__ ", "__constant__ "):
        src = src.replace(word, "")
    src = src.replace("__device__ uint32_t mx_p4", "static uint32_t mx_p4")
    s = prep.transform(src, helpers=False)
    for name, body in BODIES.items():
        s = prep._replace_body(s, name, body)
    at = s.index("static cudaError_t mx_launch(")
    s = prep._replace_block(s, s.index("{", at), LAUNCH)
    if "<<<" in s or re.search(r"\basm\b", s):
        raise ValueError("a launch or an inline instruction was not rewritten")
    s = s.replace('#include "emu.h"', '#include "emu.h"\n#include "emu_optim.h"\n#include "emu_mx4.h"\n#include <type_traits>', 1)
    kern = os.path.join(BUILD, "emu_mx4.cpp")
    with open(kern, "w") as f:
        f.write(s + PRODUCT)
    inc = ["-I" + HERE, "-I" + base.INCLUDE, "-I" + base.CSRC, "-I" + os.path.join(base.CUDA, "include")]
    common = ["-O1", "-g", "-fPIC", "-fvisibility=hidden", *base.SAN, *inc]
    cmds, objs = [], []
    for src in ("mc_mx4.c", "mc_util.c"):
        o = os.path.join(BUILD, src + ".o")
        cmds.append(["gcc", "-std=gnu11", *common, "-c", os.path.join(base.CSRC, src), "-o", o])
        objs.append(o)
    for path in (kern, os.path.join(HERE, "fake_cudart.cpp")):
        o = os.path.join(BUILD, os.path.basename(path) + ".o")
        cmds.append(["g++", "-std=c++17", "-ffp-contract=off", "-w", *common, "-c", path, "-o", o])
        objs.append(o)
    base._run_all(cmds)
    base._run_all([["g++", "-shared", *base.SAN, "-Wl,-Bsymbolic", "-Wl,--no-undefined", "-o", out + ".tmp", *objs,
                    "-ldl", "-lpthread", "-lm"]])
    os.replace(out + ".tmp", out)
    return out


if __name__ == "__main__":
    print(build())
