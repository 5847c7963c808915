// mc_mx4_device.h -- device code that the 4-bit kernels and dropout share:
// element types, random bits, the 4-bit rounding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "mc_mx4.h"

namespace {

__device__ __forceinline__ float mx_f32(float x) { return x; }
__device__ __forceinline__ float mx_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float mx_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void mx_from(float *p, float x) { *p = x; }
__device__ __forceinline__ void mx_from(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void mx_from(__half *p, float x) { *p = __float2half_rn(x); }

// ------------------------------------------------------------ random bits
// 32-bit avalanche (the finaliser of MurmurHash3, Appleby, public domain).
__host__ __device__ __forceinline__ uint32_t mx_mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x85EBCA6Bu;
    x ^= x >> 13;
    x *= 0xC2B2AE35u;
    return x ^ (x >> 16);
}

// The two key words of a purpose, seed and counter.  The second one enters
// between the two products, so that two keys do not give the same words in
// another order.
struct mx_key {
    uint32_t a, b;
};
__device__ __forceinline__ mx_key mx_key_of(const mx_random &r) {
    const uint64_t c = r.counter ? (uint64_t)*r.counter : 0;
    mx_key k;
    k.a = mx_mix(mx_mix(r.key ^ (uint32_t)c) ^ (uint32_t)(c >> 32));
    k.b = mx_mix(k.a ^ 0x85EBCA77u);
    return k;
}
// The key for positions with these high bits.
__device__ __forceinline__ mx_key mx_key_at(mx_key k, uint64_t pair) {
    if (pair >> 32) k.a ^= mx_mix((uint32_t)(pair >> 32));
    return k;
}
// The word of a pair of elements: 16 bits for each, the even one's below.
__device__ __forceinline__ uint32_t mx_word(mx_key k, uint32_t pair) {
    uint32_t x = pair ^ k.a;
    x = ((x ^ (x >> 16)) * 0x85EBCA6Bu) ^ k.b;
    x = (x ^ (x >> 13)) * 0xC2B2AE35u;
    return x ^ (x >> 16);
}
__device__ __forceinline__ int64_t mx_wide(int64_t cols) { return (cols + MX_BLOCK - 1) / MX_BLOCK * MX_BLOCK; }

// ---------------------------------------------------------- 4-bit rounding
// The scale of a block from its largest magnitude's bits: the smallest power
// of two (E8M0 code, at least 0 for 2^-127) of which no element is more than
// 6 times; 255 (NaN) where an element is infinite or NaN.  A significand up
// to 1.5 is 4 to 6 times 2^(exponent - 2), a larger one 3 to 4 times the next
// power.
__device__ __forceinline__ uint32_t mx_scale(uint32_t top) {
    if (top >= 0x7F800000u) return 255u;
    const int e = (int)((top + 0x3FFFFFu) >> 23) - 2;
    return (uint32_t)max(e, 0);
}
// 1 / scale, exactly; the codes of a block whose scale is NaN become 0.
__device__ __forceinline__ float mx_inverse(uint32_t scale) {
    return scale == 255u ? 0.0f : __uint_as_float((254u - scale) << 23);
}

// Codes of 8 elements (times 1 / scale), first one in the low bits; nearest,
// ties to the even code.
__device__ __forceinline__ uint32_t mx_codes8(const float *y) {
    uint32_t r;
    asm("{.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};}"
        : "=r"(r)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return r;
}

__device__ __forceinline__ uint32_t mx_code_near(float y) {
    uint32_t r;
    asm("{.reg .b8 a;\n\tcvt.rn.satfinite.e2m1x2.f32 a, 0f00000000, %1;\n\tmov.b32 %0, {a, a, a, a};}" : "=r"(r) : "f"(y));
    return r & 15u;
}

// One code, rounded up with the probability that its distance asks for.
// Times 2^-126 the codes 0 to 7 are the float32 bits 22 and up (0.5 a
// subnormal number): the bits below are the distance, and a carry from adding
// the random bits to them rounds up.  Digits below 2^-149 are cut off, which
// changes no carry: the random bits (16, and a half) end far above.
__device__ __forceinline__ uint32_t mx_code_random(float y, uint32_t bits16) {
    const uint32_t b = __float_as_uint(__fmul_rz(fabsf(y), 1.17549435e-38f));
    return ((b + (bits16 << 6) + 32u) >> 22) | (__float_as_uint(y) >> 31 << 3);
}

// The value of the code in bits 0 to 3, without its scale.
__device__ __forceinline__ float mx_value(uint32_t code) {
    // the reverse: magnitude bits to 22 and up, times 2^126
    const float m = __uint_as_float((code & 7u) << 22) * 8.50705917e37f;
    return __uint_as_float(__float_as_uint(m) | (code & 8u) << 28);
}
// The scale as a float32 (2^-127 is a subnormal number).
__device__ __forceinline__ float mx_scale_value(uint32_t scale) {
    return scale == 255u ? __uint_as_float(0x7FC00000u) : scale == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(scale << 23);
}

// ---------------------------------------------------------- matrix layout
__device__ __forceinline__ int64_t mx_rows8(int64_t rows) { return (rows + 7) & ~(int64_t)7; }
// Byte of the first element of block `k` (of its row) in the codes.
__device__ __forceinline__ int64_t mx_code_at(int64_t rows, int64_t r, int64_t k) {
    return (k / 8 * mx_rows8(rows) + r) * 128 + ((k & 7) ^ (r & 7)) * 16;
}
__device__ __forceinline__ int64_t mx_scale_at(int64_t rows, int64_t r, int64_t k) {
    const int64_t groups = (rows + MX_GROUP - 1) / MX_GROUP;
    return ((k / 8 * groups + r / MX_GROUP) * 2 + (k / 4 & 1)) * 512 + (r & 31) * 16 + (r / 32 & 3) * 4 + (k & 3);
}

}  // namespace
