// emu_mx4.h -- what mc_mx4.cu, mc_mx4_device.h and mc_mx4.c use beyond emu.h,
// emu_optim.h and fake_cudart.cpp (test infrastructure only).  The product's
// kernels are tensor core instructions: a plain sum over the matrices as they
// lie in memory stands in for them, so that the layouts, the order of launches
// and the argument checks around it run on the host.
#pragma once

#include "mc_mx4.h"

template <class T>
inline T __ldg(const T *p) {
    if (((uintptr_t)p) & (sizeof(T) - 1)) abort();
    return *p;
}
inline unsigned __reduce_max_sync(unsigned m, unsigned v) {
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(m, v, o));
    return v;
}
// towards zero: the product of two float32 numbers is exact in 64 bits
inline float __fmul_rz(float a, float b) {
    const double p = (double)a * b;
    float r = (float)p;
    if (std::isfinite(r) && fabs((double)r) > fabs(p)) r = nextafterf(r, 0.0f);
    return r;
}
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

// [rows][panels] of a matrix's values, block by block, as the layout says
inline double emu_mx4_value(const mx_matrix &m, int64_t r, int64_t c) {
    static const double value[8] = {0, 0.5, 1, 1.5, 2, 3, 4, 6};
    const int64_t panel = c / 256, block = c % 256 / 32, rows8 = (m.rows + 7) / 8 * 8, groups = (m.rows + 127) / 128;
    const uint8_t byte = m.codes[(panel * rows8 + r) * 128 + (block ^ (r & 7)) * 16 + c % 32 / 2];
    const unsigned code = c & 1 ? byte >> 4 : byte & 15;
    const unsigned scale = m.scales[((panel * groups + r / 128) * 2 + block / 4) * 512 + r % 32 * 16 + r / 32 % 4 * 4 + block % 4];
    const double v = scale == 255 ? NAN : value[code & 7] * exp2((int)scale - 127.0);
    return code & 8 ? -v : v;
}
