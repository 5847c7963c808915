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

// Programmatic dependent launch: a kernel may start while its predecessor on
// the stream finishes; it waits for it (mx_begin) before it touches memory.
__device__ __forceinline__ void mx_begin() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// More dynamic shared memory than a kernel may have unasked.
template <typename K>
static cudaError_t mx_allow(K kern, size_t smem) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e;
}

// `cluster` > 0: of so many CTAs.
template <typename... P, typename... A>
static cudaError_t mx_launch(void (*kern)(P...), int64_t grid, int threads, size_t smem, int cluster, cudaStream_t s, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    const cudaError_t late = cudaGetLastError();
    return e != cudaSuccess ? e : late;
}

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

// The key of a purpose, seed and counter: two words, each with its own shift
// folded in, since (x ^ a) ^ ((x ^ a) >> n) = x ^ (x >> n) ^ (a ^ (a >> n)).
// The second enters between the two products, so that two keys do not give
// the same words in another order.
struct mx_key {
    uint32_t a, b;   // a ^ (a >> 16), b ^ (b >> 13)
};
__host__ __device__ __forceinline__ mx_key mx_key_with(uint32_t key, uint64_t counter) {
    const uint32_t a = mx_mix(mx_mix(key ^ (uint32_t)counter) ^ (uint32_t)(counter >> 32)), b = mx_mix(a ^ 0x85EBCA77u);
    mx_key k;
    k.a = a ^ (a >> 16);
    k.b = b ^ (b >> 13);
    return k;
}
__device__ __forceinline__ mx_key mx_key_of(const mx_random &r) {
    if (r.counter) return mx_key_with(r.key, (uint64_t)*r.counter);
    mx_key k;
    k.a = r.a;
    k.b = r.b;
    return k;
}
// The start of the words of positions from `pair` on, a multiple of 4: word j
// (0 to 3) is mx_word(key, start ^ j).
__device__ __forceinline__ uint32_t mx_start(mx_key k, uint64_t pair) {
    const uint32_t low = (uint32_t)pair, high = (uint32_t)(pair >> 32);
    uint32_t s = low ^ (low >> 16) ^ k.a;
    if (high) {
        const uint32_t m = mx_mix(high);
        s ^= m ^ (m >> 16);
    }
    return s;
}
// The word of a pair of elements: the even one's 16 bits below, the odd one's above.
__device__ __forceinline__ uint32_t mx_word(mx_key k, uint32_t start) {
    uint32_t x = start * 0x85EBCA6Bu;
    x = (x ^ (x >> 13) ^ k.b) * 0xC2B2AE35u;
    return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t mx_word_at(mx_key k, uint64_t pair) { return mx_word(k, mx_start(k, pair)); }
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

__device__ __forceinline__ float2 mx_mul2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 r, a, b;\n\t"
        "mov.b64 {%0, %1}, r;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mx_add2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 r, a, b;\n\t"
        "mov.b64 {%0, %1}, r;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mx_mul2_cut(float2 a, float2 b) {   // towards 0
    float2 r;
    asm("{.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rz.f32x2 r, a, b;\n\t"
        "mov.b64 {%0, %1}, r;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

// Rounding at random.  Times 2^-126 the magnitudes 0, 0.5, 1, ... 6 have the
// codes 0 to 7 in the float32's bits 22 and up (0.5 is a subnormal number); the
// bits below are the distance from the value below, and where adding the
// random bits to them carries, the code is rounded up.  Digits below 2^-149
// are cut off, which changes no carry: the random bits (16, and a half) end
// far above.
#define MX_CUT 1.17549435e-38f
// Powers of two that the compiler does not turn into shifts: these run on the
// pipe of multiplications, the other one bounds the rounding at random (4099 x
// 50257 bf16 both ways: 313 us against 295).
__device__ __constant__ uint32_t mx_p4 = 1u << 4, mx_p8 = 1u << 8, mx_p16 = 1u << 16;
// What is added for the lower and for the upper 16 bits of a word: 64 times
// them and 32.
__device__ __forceinline__ uint32_t mx_add_low(uint32_t word) { return ((word << 6) & 0x3FFFC0u) | 32u; }
__device__ __forceinline__ uint32_t mx_add_high(uint32_t word) { return ((word >> 10) & 0x3FFFC0u) | 32u; }
// The magnitude code of y * 2^-126.
__device__ __forceinline__ uint32_t mx_code_random(float cut, uint32_t add) { return (__float_as_uint(cut) + add) >> 22; }
// Magnitude codes of 8 elements: y their magnitudes times 1 / scale, two by
// two, and what is added to each.
__device__ __forceinline__ uint32_t mx_codes8_random(const float2 *y, const uint32_t *add) {
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 m = mx_mul2_cut(y[i], make_float2(MX_CUT, MX_CUT));
        p[i] = mx_code_random(m.x, add[2 * i]) + mx_code_random(m.y, add[2 * i + 1]) * mx_p4;
    }
    return (p[0] + p[1] * mx_p8) + (p[2] + p[3] * mx_p8) * mx_p16;
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

// ------------------------------------------------------------- elements
template <typename T>
struct __align__(16) mx_vec8 {
    T x[8];
};

template <typename T>
__device__ __forceinline__ mx_vec8<T> load8(const T *p) {
    mx_vec8<T> v;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(v) / 16); i++) ((uint4 *)&v)[i] = __ldg((const uint4 *)p + i);
    return v;
}

// What rounding needs of elements: the largest magnitude (of two at a time
// where they have 16 bits; NaN where one is), as bits, and float32 values.
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b, float) { return max(a, b & 0x7FFFFFFFu); }
template <typename T>
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
    T x, y;
    memcpy(&x, &a, 4);
    memcpy(&y, &b, 4);
    x = __hmax2_nan(x, __habs2(y));   // (the magnitude is a modifier of the operand)
    memcpy(&a, &x, 4);
    return a;
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b, __nv_bfloat16) { return larger2<__nv_bfloat162>(a, b); }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b, __half) { return larger2<__half2>(a, b); }
// The float32 bits of the largest, by the two halves of a 32-bit word for 16-bit types.
__device__ __forceinline__ uint32_t top_low(uint32_t m, __nv_bfloat16) { return m << 16; }
__device__ __forceinline__ uint32_t top_low(uint32_t m, __half) { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m))); }
template <typename T>
__device__ __forceinline__ uint32_t top_of(uint32_t m, T t) { return max(top_low(m & 0xFFFFu, t), top_low(m >> 16, t)); }
__device__ __forceinline__ uint32_t top_of(uint32_t m, float) { return m; }
// Float32 values of the two 16-bit elements of a word.
__device__ __forceinline__ float2 two_of(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ float2 two_of(uint32_t w, __half) {
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}
// Bit 7 of byte B of 8 words to bit 3 of the 8 nibbles of one, and of byte 3.
template <int B>
__device__ __forceinline__ uint32_t signs8(const uint32_t *w) {
    constexpr uint32_t PICK = (uint32_t)(B | (B + 4) << 4);
    const uint32_t e = __byte_perm(__byte_perm(w[0], w[2], PICK), __byte_perm(w[4], w[6], PICK), 0x5410);
    const uint32_t o = __byte_perm(__byte_perm(w[1], w[3], PICK), __byte_perm(w[5], w[7], PICK), 0x5410);
    return ((e >> 4) & 0x08080808u) | (o & 0x80808080u);
}
// The same of both halves of 4 words, in the order of the elements.
__device__ __forceinline__ uint32_t signs4x2(const uint32_t *w) {
    const uint32_t x = __byte_perm(w[0], w[1], 0x7351), y = __byte_perm(w[2], w[3], 0x7351);
    return ((__byte_perm(x, y, 0x5410) >> 4) & 0x08080808u) | (__byte_perm(x, y, 0x7632) & 0x80808080u);
}

// The codes of 8 elements.  y: values (at random: magnitudes) times 1 / scale, two by two.
template <bool RANDOM>
__device__ __forceinline__ uint32_t codes8(const float2 *y, uint32_t signs, const uint32_t *add) {
    if (RANDOM) return mx_codes8_random(y, add) | signs;
    return mx_codes8((const float *)y);
}

// A row's 8 elements (raw words) to codes.
template <typename T, bool RANDOM, bool DROP>
__device__ __forceinline__ uint32_t row_codes(const uint32_t *w, float inv, float factor, const uint32_t *words) {
    float2 y[4];
    uint32_t add[8], signs = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) y[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else y[i] = two_of(RANDOM ? w[i] & 0x7FFF7FFFu : w[i], T());
        if (sizeof(T) == 4 && RANDOM) y[i] = make_float2(fabsf(y[i].x), fabsf(y[i].y));
        if (DROP) y[i] = mx_mul2(y[i], make_float2(factor, factor));
        y[i] = mx_mul2(y[i], make_float2(inv, inv));
        if (RANDOM) {
            add[2 * i] = mx_add_low(words[i]);
            add[2 * i + 1] = mx_add_high(words[i]);
        }
    }
    if (RANDOM) {
        if constexpr (sizeof(T) == 4) signs = signs8<3>(w);
        else signs = signs4x2(w);
    }
    return codes8<RANDOM>(y, signs, add);
}

}  // namespace
