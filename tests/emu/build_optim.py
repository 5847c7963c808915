"""Kernel-emulation library of the optimiser entry points (test
infrastructure only, see build.py): mc_optim.c unchanged and mc_optim.cu
through prep.py's source transform, against emu.h and the fake runtime.
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

BUILD = os.path.join(HERE, "_build_optim")
INPUTS = [os.path.join(base.CSRC, f) for f in ("mc_optim.c", "mc_optim.cu", "mc_optim.h", "mc_call.h", "mc_util.c", "mc_internal.h")] + \
         [os.path.join(base.INCLUDE, "falcom_b200.h")] + \
         [os.path.join(HERE, f) for f in ("emu.h", "emu_optim.h", "fake_cudart.cpp", "prep.py", "build_optim.py")]

LD_STREAM = ' if (((uintptr_t)p) & (sizeof(*p) - 1)) abort(); return *p; '
# host bodies of the inline-PTX helpers
BODIES = {
    "prefetch": " (void)p; ",
    "pdl_wait": "",
    "pdl_release": "",
    "smem_u32": " return emu_smem_u32(p); ",
    "mbar_init": " emu_mbar_init(bar, count); ",
    # copies complete at issue
    "mbar_expect_tx": " (void)bytes; emu_mbar_arrive(bar); ",
    "mbar_arrive": " emu_mbar_arrive(bar); ",
    "bulk_g2s": """
    (void)bar;
    char *d = (char *)emu_smem_ptr(dst);
    if ((dst & 15) || (((uintptr_t)src) & 15) || (bytes & 15) || d < (char *)emu_cta->lo ||
        d + bytes > (char *)emu_cta->hi) abort();
    memcpy(d, src, bytes);
""",
    "copy_async4": " if ((char *)dst < (char *)emu_cta->lo || (char *)(dst + 1) > (char *)emu_cta->hi) abort(); *dst = *src; ",
    "arrive_after_copies": " emu_mbar_arrive(bar); ",
    "mbar_try_wait": " return emu_late_waits == 0 && emu_mbar_done(bar, parity); ",
    "mbar_wait_some": """
    if (emu_wait_is_late()) return false;
    for (int i = 0; i < 50000000; i++) {
        if (emu_mbar_done(bar, parity)) return true;
        std::this_thread::yield();
    }
    fprintf(stderr, "emu: a barrier never completed\\n");
    abort();
""",
    "add2": " return make_float2(a.x + b.x, a.y + b.y); ",
    "rsqrt_fast": " return 1.0f / sqrtf(x); ",
    "mul2": " return make_float2(a.x * b.x, a.y * b.y); ",
    "fma2": " return make_float2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); ",
    "sqrt_fast": " return sqrtf(x); ",
    "rcp_fast": " return 1.0f / x; ",
    "max_abs": " a = fabsf(a); return a != a || b != b || c != c ? NAN : fmaxf(a, fmaxf(fabsf(b), fabsf(c))); ",
    "warp_max": " for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o)); return v; ",
    "e4m3_quad": """
    a = make_float2(emu_e4m3(codes & 0xFF), emu_e4m3(codes >> 8 & 0xFF));
    b = make_float2(emu_e4m3(codes >> 16 & 0xFF), emu_e4m3(codes >> 24));
""",
}


def build() -> str:
    h = hashlib.sha256()
    for f in INPUTS:
        with open(f, "rb") as fh:
            h.update(fh.read())
    out = os.path.join(BUILD, f"libfalcom_optim_emu_{h.hexdigest()[:16]}.so")
    if os.path.exists(out):
        return out
    os.makedirs(BUILD, exist_ok=True)
    with open(os.path.join(base.CSRC, "mc_optim.cu")) as f:
        src = f.read()
    s = prep.transform(re.sub(r"extern __shared__ __align__\(\d+\) float s_stage\[\];", "", src).replace("__host__ ", "").replace("__noinline__ ", "").replace("__grid_constant__ ", ""), helpers=False)
    for vec in ("uint32_t", "uint2", "uint4"):   # the overloads one after another
        at = s.index(f"inline {vec} ld_stream(")
        s = prep._replace_block(s, s.index("{", at), LD_STREAM)
    for name, body in BODIES.items():
        s = prep._replace_body(s, name, body)
    if "emu_run(grid, smem" not in s or "<<<" in s or "asm volatile" in s:
        raise ValueError("a launch or an inline instruction was not rewritten")
    s = s.replace('#include "emu.h"', '#include "emu.h"\n#include "emu_optim.h"')
    kern = os.path.join(BUILD, "emu_optim.cpp")
    with open(kern, "w") as f:
        f.write(s)
    inc = ["-I" + HERE, "-I" + base.INCLUDE, "-I" + base.CSRC, "-I" + os.path.join(base.CUDA, "include")]
    common = ["-O1", "-g", "-fPIC", "-fvisibility=hidden", *base.SAN, *inc]
    cmds, objs = [], []
    for src in ("mc_optim.c", "mc_util.c"):
        o = os.path.join(BUILD, src + ".o")
        cmds.append(["gcc", "-std=gnu11", *common, "-c", os.path.join(base.CSRC, src), "-o", o])
        objs.append(o)
    for path in (kern, os.path.join(HERE, "fake_cudart.cpp")):
        o = os.path.join(BUILD, os.path.basename(path) + ".o")
        cmds.append(["g++", "-std=c++17", "-ffp-contract=off", *common, "-c", path, "-o", o])
        objs.append(o)
    base._run_all(cmds)
    base._run_all([["g++", "-shared", *base.SAN, "-Wl,-Bsymbolic", "-Wl,--no-undefined", "-o", out + ".tmp", *objs,
                    "-ldl", "-lpthread", "-lm"]])
    os.replace(out + ".tmp", out)
    return out


if __name__ == "__main__":
    print(build())
