"""Kernel-emulation library of the 4-bit product (test infrastructure only):
mc_mx4_product.cu with mc_mx4_device.h through a source transform, on emu_product.h's
clusters, copies, tensor memory and matrix instructions.  Kernel code and the
choice of kernels stay as written; qualifiers go, __shared__ variables become
places in the emulated CTA's memory, and each wrapper of an instruction gets a
host body.
"""
from __future__ import annotations

import hashlib
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(os.path.dirname(HERE)))
from tests.emu import build as base  # noqa: E402
from tests.emu import build_mx4, prep  # noqa: E402

BUILD = os.path.join(HERE, "_build_mx4")
INPUTS = [os.path.join(base.CSRC, f) for f in ("mc_mx4_product.cu", "mc_mx4.h", "mc_mx4_device.h")] + \
         [os.path.join(base.INCLUDE, "falcom_b200.h")] + \
         [os.path.join(HERE, f) for f in ("emu_product.h", "build_mx4.py", "build_product.py", "prep.py")]

BODIES = {
    "mx_begin": "",
    "mx_codes8": build_mx4.BODIES["mx_codes8"],
    "mx_code_near": build_mx4.BODIES["mx_code_near"],
    "mx_mul2": build_mx4.BODIES["mx_mul2"],
    "mx_add2": build_mx4.BODIES["mx_add2"],
    "mx_mul2_cut": " abort(); ",
    "larger2": build_mx4.BODIES["larger2"],
    "smem_u32": " return (uint32_t)((const uint8_t *)p - emu_cta->mem); ",
    "mbar_init": " emu_bar_init(bar, count); ",
    "mbar_expect_tx": " emu_arrive(bar, -1, (int)bytes); ",
    "bulk_g2s": " emu_copy(dst, (const uint8_t *)src, bytes, bar, -1); ",
    "mbar_try_wait": " return emu_done(bar, parity, 0); ",
    "mbar_wait_long": """
    for (double t = 0; t < seconds; t += 0.25) {
        if (emu_done(bar, parity, 0.25)) return true;
        if (failed && *failed) return false;
    }
    return false;
""",
    "mbar_try_wait_cluster": " return emu_done(bar, parity, 0); ",
    "elect_one": " return (threadIdx.x & 31) == 0; ",
    "tmem_alloc": " emu_tmem_alloc(dst, COLUMNS); ",
    "tmem_free": " emu_tmem_free(at, COLUMNS); ",
    "tc_before_sync": "",
    "tc_after_sync": "",
    "tc_copy_scales": " emu_copy_scales(emu_cta, -1, tmem, desc); ",
    "tc_mma": " emu_mma(1, d, a, b, idesc, sa, sb, add); ",
    "tc_commit": " emu_arrive(bar, -1); ",
    "tc_wait_ld": "",
    "tc_ld16": " emu_tmem_load(at, r, 16); ",
    "cluster_sync": " emu_cluster->all.wait(); ",
    "ld_cluster": " return emu_load<float>(at, (int)rank); ",
    "mbar_arrive": " emu_arrive(bar, -1); ",
    "st_second": " emu_store<uint32_t>(at, v, 1); ",
    "tmem_alloc_pair": " emu_tmem_alloc(dst, 512); ",
    "tmem_free_pair": " emu_tmem_free(at, 512); ",
    "tc_copy_scales_pair": " for (int c = 0; c < 2; c++) emu_copy_scales(emu_cluster->cta[c].get(), c, tmem, desc); ",
    "tc_mma_pair": " emu_mma(2, d, a, b, idesc, sa, sb, add); ",
    "tc_commit_pair": " emu_arrive(bar, 0); emu_arrive(bar, 1); ",
    "mbar_arrive_first": " emu_arrive(bar, 0); ",
    "load_rows_pair": " emu_copy_box(dst, map, row, bar); ",
    "st_shared16": " emu_store(at, v); ",
    "ld_shared16": " return emu_load<uint4>(at); ",
    "bar_pair": " emu_cta->named[id]->wait(); ",
    "encoder": " return emu_encode_map; ",
}
# instructions that kernels use in place
INLINE = [
    (r'asm volatile\("fence\.[\w.:]+;" ::: "memory"\);', ";"),
    (r'asm volatile\("st\.shared\.b32 \[%0\], %1;" ::"r"\((.*)\), "r"\((.*)\) : "memory"\);', r"emu_store<uint32_t>(\1, \2);"),
    (r'asm volatile\("st\.shared\.b8 \[%0\], %1;" ::"r"\((.*)\), "r"\((.*)\) : "memory"\);', r"emu_store<uint8_t>(\1, (uint8_t)(\2));"),
    (r'asm volatile\("ld\.shared\.b32 %0, \[%1\];" : "=r"\((.*)\) : "r"\((.*)\) : "memory"\);', r"\1 = emu_load<uint32_t>(\2);"),
    (r'asm volatile\("ld\.shared\.b16 %0, \[%1\];" : "=h"\((.*)\) : "r"\((.*)\) : "memory"\);', r"\1 = emu_load<uint16_t>(\2);"),
    (r'asm volatile\("\{\\n\\t\.reg \.b16 x;\\n\\tld\.shared\.b16 x, \[%1\];\\n\\tcvt\.u32\.u16 %0, x;\\n\\t\}" : "=r"\((.*)\) : "r"\((.*)\) : "memory"\);',
     r"\1 = emu_load<uint16_t>(\2);"),
]
HEAD = """
inline unsigned emu_e2m1(float y) {   // nearest, ties to even codes; at most 6
    static const float value[8] = {0, 0.5f, 1, 1.5f, 2, 3, 4, 6};
    const float m = fabsf(y);
    unsigned c = 0;
    while (c < 7 && (m > (value[c] + value[c + 1]) / 2 || (m == (value[c] + value[c + 1]) / 2 && (c & 1)))) c++;
    return c | (std::signbit(y) ? 8u : 0u);
}
inline unsigned emu_top_half(unsigned a, unsigned b, unsigned infinity) {   // the larger magnitude; NaN above all
    a &= 0x7FFF;
    b &= 0x7FFF;
    return a > infinity || b > infinity ? 0x7FFF : a > b ? a : b;
}
"""
# a call of the kernels; the matrices as mc_mx4.c hands them on
CALL = """
#define EMU_API extern "C" __attribute__((visibility("default")))
EMU_API int emu_product(const mx_product_launch *given, double p, uint64_t seed, int type, int sms) {
    mx_product_launch L = *given;
    L.drop.threshold = (uint32_t)(p * 65536 + 0.5);
    L.drop.factor = (float)(65536.0 / (65536.0 - L.drop.threshold));
    const mx_key k = mx_key_with(mx_mix(mx_mix((uint32_t)seed ^ 0x7F4A7C15u) ^ (uint32_t)(seed >> 32)), 0);
    L.drop.random.a = k.a;
    L.drop.random.b = k.b;
    L.drop.random.on = p > 0;
    emu_global.clear();
    for (const mx_matrix *m : {&L.a, &L.b})
        if (m->codes) {
            const int64_t panels = (m->cols + 255) / 256, codes = panels * ((m->rows + 7) / 8 * 8) * 128, scales = panels * ((m->rows + 127) / 128) * 1024;
            emu_global.push_back({m->codes, m->codes + codes});
            emu_global.push_back({m->scales, m->scales + scales});
        }
    return mc_launch_mx_product(&L, type, sms, nullptr);
}
// From its copy number `from` on a CTA of that rank loses them, and a second is that short (rank -1: none, as it is).
EMU_API void emu_product_lose(int rank, int from, double second) {
    emu_lost_rank = rank;
    emu_lost_from = from;
    emu_second = rank < 0 ? 100.0 : second;
}
// How many CTAs gave up since the last call.
EMU_API int emu_product_errors() {
    static uint32_t seen;
    uint32_t word = 0;
    mc_mx_errors(&word);
    const int n = (int)(word - seen);
    seen = word;
    return n;
}
"""


def _shared(m: re.Match) -> str:
    """A __shared__ declaration as places of the emulated CTA."""
    out = []
    for d in m.group(2).split(", "):
        name, _, size = d.partition("[")
        slot = f"({m.group(1)} *)emu_slot({_shared.next})"
        out.append(f"{m.group(1)} *const {name} = {slot};" + (f" static_assert(sizeof({m.group(1)}) * ({size[:-1]}) <= 512, \"\");" if size else "")
                   if size else f"{m.group(1)} &{name} = *{slot};")
        _shared.next = (_shared.next + 1) % 12
    return " ".join(out)


def transform(head: str, src: str) -> str:
    s = src.replace('#include "mc_mx4_device.h"', head)
    s = s.replace("#include <cuda_runtime.h>", "").replace("#include <cuda_bf16.h>", "").replace("#include <cuda_fp16.h>", "")
    s = re.sub(r"__cluster_dims__\([^)]*\)", "", s)
    s = re.sub(r"__launch_bounds__\([^)]*\)", "", s)
    s = s.replace("extern __shared__ uint8_t s_raw[];", "uint8_t *const s_raw = emu_dynamic();")
    _shared.next = 0
    s = re.sub(r"__shared__ (?:__align__\(\d+\) )?((?:volatile )?\w+) ([^;]*);", _shared, s)
    s = s.replace("__device__ __constant__", "static").replace("__device__ __noinline__", "inline").replace("__device__ uint32_t g_", "static uint32_t g_")
    for word in ("__host__ ", "__grid_constant__ ", "__global__ "):
        s = s.replace(word, "")
    s = s.replace("__device__ __forceinline__", "inline").replace("__device__ ", "")
    s = re.sub(r"__align__\((\d+)\)", r"__attribute__((aligned(\1)))", s)
    for name, body in BODIES.items():
        s = prep._replace_body(s, name, body)
    at = s.index("static cudaError_t mx_launch(")
    s = prep._replace_block(s, s.index("{", at), " (void)s; emu_launch(grid, threads, smem, cluster > 0 ? cluster : 2, [&] { kern(args...); }); return cudaSuccess; ")
    s = prep._replace_block(s, s.index("{", s.index("static cudaError_t mx_allow(")), " (void)kern; return smem <= 227 * 1024 ? cudaSuccess : cudaErrorInvalidValue; ")
    for pattern, to in INLINE:
        s = re.sub(pattern, to, s)
    s = prep._replace_block(s, s.index("{", s.index('extern "C" int mc_mx_errors(')), " *word = g_mx_error; return 0; ")
    rest = re.search(r"\basm\b.*", s)
    if "<<<" in s or rest or "__shared__" in s:
        raise ValueError(f"an instruction was not rewritten: {rest and rest.group(0)}")
    return '#include "emu_product.h"\n#include <cuda_bf16.h>\n#include <cuda_fp16.h>\n' + HEAD + s + CALL


def build() -> str:
    h = hashlib.sha256()
    for f in INPUTS:
        with open(f, "rb") as fh:
            h.update(fh.read())
    out = os.path.join(BUILD, f"libfalcom_product_emu_{h.hexdigest()[:16]}.so")
    if os.path.exists(out):
        return out
    os.makedirs(BUILD, exist_ok=True)
    with open(os.path.join(base.CSRC, "mc_mx4_device.h")) as f:
        head = f.read().replace("#pragma once", "")
    with open(os.path.join(base.CSRC, "mc_mx4_product.cu")) as f:
        code = transform(head, f.read())
    kern = os.path.join(BUILD, "emu_product.cpp")
    with open(kern, "w") as f:
        f.write(code)
    inc = ["-I" + HERE, "-I" + base.INCLUDE, "-I" + base.CSRC, "-I" + os.path.join(base.CUDA, "include")]
    base._run_all([["g++", "-std=c++17", "-O2", "-g1", "-fPIC", "-fvisibility=hidden", "-ffp-contract=off", "-w", "-shared", *base.SAN,
                    "-Wl,-Bsymbolic", *inc, kern, "-o", out + ".tmp", "-lpthread", "-lm"]])
    os.replace(out + ".tmp", out)
    return out


if __name__ == "__main__":
    print(build())
