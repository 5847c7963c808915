"""Kernel-emulation library of the optimiser entry points (test
infrastructure only, see build.py): mc_optim.c unchanged and mc_optim.cu
through prep.py's source transform, against emu.h and the fake runtime.
"""
from __future__ import annotations

import hashlib
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(os.path.dirname(HERE)))
from tests.emu import build as base  # noqa: E402
from tests.emu import prep  # noqa: E402

BUILD = os.path.join(HERE, "_build_optim")
INPUTS = [os.path.join(base.CSRC, f) for f in ("mc_optim.c", "mc_optim.cu", "mc_optim.h")] + \
         [os.path.join(base.INCLUDE, "falcom_b200.h")] + \
         [os.path.join(HERE, f) for f in ("emu.h", "emu_optim.h", "fake_cudart.cpp", "prep.py", "build_optim.py")]


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
    s = prep.transform(src.replace("__host__ ", ""), helpers=False)
    for name in ("pdl_wait", "pdl_release"):
        s = prep._replace_body(s, name, "")
    if "emu_run(grid, smem" not in s or "<<<" in s or "asm volatile" in s:
        raise ValueError("a launch or an inline instruction was not rewritten")
    s = s.replace('#include "emu.h"', '#include "emu.h"\n#include "emu_optim.h"')
    kern = os.path.join(BUILD, "emu_optim.cpp")
    with open(kern, "w") as f:
        f.write(s)
    inc = ["-I" + HERE, "-I" + base.INCLUDE, "-I" + base.CSRC, "-I" + os.path.join(base.CUDA, "include")]
    common = ["-O1", "-g", "-fPIC", "-fvisibility=hidden", *base.SAN, *inc]
    host = os.path.join(BUILD, "mc_optim.o")
    cmds, objs = [["gcc", "-std=gnu11", *common, "-c", os.path.join(base.CSRC, "mc_optim.c"), "-o", host]], [host]
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
