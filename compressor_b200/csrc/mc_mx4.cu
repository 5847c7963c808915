// mc_mx4.cu -- 4-bit rounding (vectors with what their receivers hold,
// matrices along rows and columns), reading back, and dropout.  Every element
// is read once and written once.  On whole aligned rows vectors and dropout
// are bound by memory, the rounding of matrices by instructions.

#include "mc_mx4_device.h"

namespace {

#define MX_TPB 256

// ------------------------------------------------------------- vectors
// A warp has 8 blocks.  On 16-byte boundaries a lane has 8 elements, 4 lanes a
// block, as in a matrix's rows.  On others lane i has element i of each block,
// so that loads and stores are whole lines at any alignment, and a block's
// largest magnitude is one reduction.  The codes then change lanes: those of 8 elements of a block
// that make up a 32-bit word lie on 8 lanes, one for each block.

// Lane i of a group of 8 holds 8 nibbles, one for each of 8 words; returns
// word i of the group, nibble j from lane j.
__device__ __forceinline__ uint32_t transpose8(uint32_t v, int lane) {
    uint32_t o = __shfl_xor_sync(0xffffffffu, v, 4);
    v = lane & 4 ? (o >> 16) | (v & 0xFFFF0000u) : (v & 0x0000FFFFu) | (o << 16);
    o = __shfl_xor_sync(0xffffffffu, v, 2);
    v = lane & 2 ? ((o >> 8) & 0x00FF00FFu) | (v & 0xFF00FF00u) : (v & 0x00FF00FFu) | ((o << 8) & 0xFF00FF00u);
    o = __shfl_xor_sync(0xffffffffu, v, 1);
    return lane & 1 ? ((o >> 4) & 0x0F0F0F0Fu) | (v & 0xF0F0F0F0u) : (v & 0x0F0F0F0Fu) | ((o << 4) & 0xF0F0F0F0u);
}

__device__ __forceinline__ void store8(float *p, const float *v) {
    ((float4 *)p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    ((float4 *)p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float *v) {
    mx_vec8<T> r;
#pragma unroll
    for (int j = 0; j < 8; j++) mx_from(&r.x[j], v[j]);
    *(uint4 *)p = *(const uint4 *)&r;
}
// 8 elements, or as many as there are (0 for the others)
template <typename T>
__device__ __forceinline__ mx_vec8<T> load_up_to_8(const T *p, int n) {
    if (n >= 8) return load8(p);
    mx_vec8<T> v;
    memset(&v, 0, sizeof(v));
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j < n) v.x[j] = p[j];
    return v;
}
template <typename T>
__device__ __forceinline__ void store_up_to_8(T *p, const float *v, int n) {
    if (n >= 8) {
        store8(p, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j < n) mx_from(&p[j], v[j]);
}

// Bytes of the codes of n elements, filled up to a multiple of `unit` (1 or 16).
template <typename I>
__device__ __forceinline__ I code_bytes(I n, int unit) { return (n + 2 * unit - 1) / 2 & -unit; }

template <typename T, bool BASE, bool RANDOM>
__global__ void __launch_bounds__(MX_TPB) k_mx_encode8(const __grid_constant__ mx_encode_launch L) {
    mx_begin();
    mx_key key = {};
    if (RANDOM) key = mx_key_of(L.random);
    // whole warps: 4 lanes find a block's largest magnitude together
    const int64_t lanes = (L.n + 255) / 256 * 32, step = (int64_t)gridDim.x * MX_TPB;
    for (int64_t i = (int64_t)blockIdx.x * MX_TPB + threadIdx.x; i < lanes; i += step) {
        const int left = (int)max((int64_t)0, min(L.n - 8 * i, (int64_t)8));
        mx_vec8<float> v, held;
        memset(&held, 0, sizeof(held));
        if constexpr (sizeof(T) == 4) {
            v = load_up_to_8((const float *)L.x + 8 * i, left);
        } else {
            const mx_vec8<T> raw = load_up_to_8((const T *)L.x + 8 * i, left);
#pragma unroll
            for (int j = 0; j < 8; j++) v.x[j] = mx_f32(raw.x[j]);
        }
        if (BASE) {
            if (left == 8) {   // (not through the read-only cache: the values are written below)
                ((float4 *)held.x)[0] = ((const float4 *)(L.base + 8 * i))[0];
                ((float4 *)held.x)[1] = ((const float4 *)(L.base + 8 * i))[1];
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (j < left) held.x[j] = L.base[8 * i + j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) v.x[j] -= held.x[j];
        }
        uint32_t w[8], m = 0;
        memcpy(w, &v, sizeof(v));
#pragma unroll
        for (int j = 0; j < 8; j++) m = larger(m, w[j], 0.0f);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const uint32_t s = mx_scale(m);
        uint32_t words[4];
        if (RANDOM) {
            const uint32_t start = mx_start(key, (uint64_t)(4 * i));
#pragma unroll
            for (int j = 0; j < 4; j++) words[j] = mx_word(key, start ^ j);
        }
        uint32_t codes = row_codes<float, RANDOM, false>(w, mx_inverse(s), 1.0f, words);
        if (s == 255u) codes = 0;
        if (BASE) {
            const float unit = mx_scale_value(s);
#pragma unroll
            for (int j = 0; j < 8; j++) held.x[j] += mx_value(codes >> (4 * j)) * unit;
            store_up_to_8(L.base + 8 * i, held.x, left);
        }
        if (left == 8) ((uint32_t *)L.codes)[i] = codes;
        else   // (the codes behind the last element are 0, and so is what lies between them and the scales)
            for (int j = 0, end = min((int)(code_bytes(L.n, L.unit) - 4 * i), 4); j < end; j++) L.codes[4 * i + j] = (uint8_t)(codes >> (8 * j));
        if ((i & 3) == 0 && left > 0) L.scales[i / 4] = (uint8_t)s;
    }
}

template <typename T, bool ADD>
__global__ void __launch_bounds__(MX_TPB) k_mx_decode8(const __grid_constant__ mx_decode_launch L) {
    mx_begin();
    const int64_t lanes = (L.n + 7) / 8, step = (int64_t)gridDim.x * MX_TPB;
    T *out = (T *)L.out;
    for (int64_t i = (int64_t)blockIdx.x * MX_TPB + threadIdx.x; i < lanes; i += step) {
        const int left = (int)min(L.n - 8 * i, (int64_t)8);
        uint32_t codes = 0;
        if (left == 8) codes = __ldg((const uint32_t *)L.codes + i);
        else
            for (int j = 0; j < (left + 1) / 2; j++) codes |= (uint32_t)L.codes[4 * i + j] << (8 * j);
        const float unit = mx_scale_value(__ldg(L.scales + i / 4));
        mx_vec8<T> held;
        memset(&held, 0, sizeof(held));
        if (ADD) {
            if (left == 8) {
#pragma unroll
                for (int j = 0; j < (int)(sizeof(held) / 16); j++) ((uint4 *)&held)[j] = ((const uint4 *)(out + 8 * i))[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (j < left) held.x[j] = out[8 * i + j];
            }
        }
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[j] = L.weight * (mx_value(codes >> (4 * j)) * unit);
            if (ADD) v[j] = mx_f32(held.x[j]) + v[j];
        }
        store_up_to_8(out + 8 * i, v, left);
    }
}

template <typename T, bool BASE, bool RANDOM>
__global__ void __launch_bounds__(MX_TPB) k_mx_encode(const __grid_constant__ mx_encode_launch L) {
    mx_begin();
    const int lane = threadIdx.x & 31;
    const T *x = (const T *)L.x;
    mx_key key = {};
    if (RANDOM) key = mx_key_of(L.random);
    const int64_t chunks = (L.n + 255) / 256, step = (int64_t)gridDim.x * (MX_TPB / 32);
    for (int64_t c = (int64_t)blockIdx.x * (MX_TPB / 32) + (threadIdx.x >> 5); c < chunks; c += step) {
        const int64_t e0 = c * 256 + lane;
        const int left = (int)min(L.n - c * 256, (int64_t)256);
        float v[8], held[8];
        T raw[8];
#pragma unroll
        for (int b = 0; b < 8; b++) {
            const bool in = 32 * b + lane < left;
            memset(&raw[b], 0, sizeof(T));
            held[b] = 0.0f;
            if (in) raw[b] = x[e0 + 32 * b];
            if (BASE && in) held[b] = L.base[e0 + 32 * b];
        }
        uint32_t codes = 0, scales[2] = {0, 0};
#pragma unroll
        for (int b = 0; b < 8; b++) {
            v[b] = BASE ? mx_f32(raw[b]) - held[b] : mx_f32(raw[b]);
            const uint32_t s = mx_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(v[b]) & 0x7FFFFFFFu));
            scales[b >> 2] |= s << (8 * (b & 3));
            const float y = v[b] * mx_inverse(s);
            uint32_t code;
            if (RANDOM) {
                const uint32_t w = mx_word_at(key, (uint64_t)(c * 128 + 16 * b + (lane >> 1)));
                code = mx_code_random(__fmul_rz(fabsf(y), MX_CUT), lane & 1 ? mx_add_high(w) : mx_add_low(w)) | (__float_as_uint(y) >> 31 << 3);
            } else {
                code = mx_code_near(y);
            }
            if (s == 255u) code = 0;
            codes |= code << (4 * b);
            if (BASE && 32 * b + lane < left) L.base[e0 + 32 * b] = held[b] + mx_value(code) * mx_scale_value(s);
        }
        // lane 8 g + b: elements 8 g .. 8 g + 7 of block b
        codes = transpose8(codes, lane);
        const int word = (lane & 7) * 4 + (lane >> 3);   // of the chunk's 32
        const int bytes = code_bytes(left, L.unit);
        uint8_t *out = L.codes + c * 128 + 4 * word;
        if (4 * word + 4 <= bytes) *(uint32_t *)out = codes;
        else
            for (int i = 0; 4 * word + i < bytes; i++) out[i] = (uint8_t)(codes >> (8 * i));
        if (lane < (left + 31) / 32) L.scales[c * 8 + lane] = (uint8_t)((lane & 4 ? scales[1] : scales[0]) >> (8 * (lane & 3)));
    }
}

template <typename T, bool ADD>
__global__ void __launch_bounds__(MX_TPB) k_mx_decode(const __grid_constant__ mx_decode_launch L) {
    mx_begin();
    const int lane = threadIdx.x & 31;
    T *out = (T *)L.out;
    const int64_t chunks = (L.n + 255) / 256, step = (int64_t)gridDim.x * (MX_TPB / 32);
    for (int64_t c = (int64_t)blockIdx.x * (MX_TPB / 32) + (threadIdx.x >> 5); c < chunks; c += step) {
        const int left = (int)min(L.n - c * 256, (int64_t)256);
        const int bytes = (left + 1) / 2;
        const uint8_t *in = L.codes + c * 128 + 4 * lane;
        uint32_t word = 0, scale = 0;
        if (4 * lane + 4 <= bytes) word = *(const uint32_t *)in;
        else
            for (int i = 0; 4 * lane + i < bytes; i++) word |= (uint32_t)in[i] << (8 * i);
        if (lane < (left + 31) / 32) scale = L.scales[c * 8 + lane];
        T held[8];
        if (ADD) {
#pragma unroll
            for (int b = 0; b < 8; b++)
                if (32 * b + lane < left) held[b] = out[c * 256 + 32 * b + lane];
        }
#pragma unroll
        for (int b = 0; b < 8; b++) {
            const uint32_t code = __shfl_sync(0xffffffffu, word, 4 * b + (lane >> 3)) >> (4 * (lane & 7));
            const float v = L.weight * (mx_value(code) * mx_scale_value(__shfl_sync(0xffffffffu, scale, b)));
            if (32 * b + lane < left) {
                T r;
                mx_from(&r, ADD ? mx_f32(held[b]) + v : v);
                out[c * 256 + 32 * b + lane] = r;
            }
        }
    }
}

// ------------------------------------------------------------- matrices
// A CTA has 128 x 128 elements: 4 blocks of every row and of every column,
// whose scales are one 512-byte piece of either layout.  Rows are rounded as
// they come in (8 elements a thread, 4 threads a block); for the columns the
// tile goes through shared memory, where a thread has a block of each of two
// neighbouring columns, which share their random words.  To the nearest 16384 x
// 4096 bf16 take 36 us along rows, 50 both ways (the bytes at the copy rate: 26
// and 31): both ways 3.4 TB/s with the logic pipe 69 and the issue slots 72 %
// busy, more instructions than memory.  At random logic operations bound it, 84
// % busy with some 22 an element (both ways 87 us).  Dropout in front costs
// 16384 x 1024 both ways 2.5 us (12.6 and 15.1 in a graph).  Loads of 4 rows a
// thread ahead of their use and 4 to 5 CTAs an SM made 133 us of it 96; to have
// registers for so many CTAs 14 of the 36 instances keep up to 48 bytes a thread
// in local memory.
#define MX_TILE 128

// 8 elements from any address: the aligned 16-byte pieces that they lie in,
// and one more, which may lie outside of them by up to 16 bytes at either end.
template <typename T>
struct __align__(16) mx_pieces {
    uint32_t w[2 * sizeof(T) + 4];
};
template <typename T>
__device__ __forceinline__ mx_pieces<T> load_pieces(const T *p) {
    mx_pieces<T> v;
    const uint4 *q = (const uint4 *)((uintptr_t)p & ~(uintptr_t)15);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(v) / 16); i++) ((uint4 *)&v)[i] = __ldg(q + i);
    return v;
}
template <typename T>
__device__ __forceinline__ mx_vec8<T> from_pieces(mx_pieces<T> v, const T *p) {
    constexpr int N = 2 * sizeof(T);
    const uint32_t off = (uint32_t)(uintptr_t)p;
    const bool two = off & 8, one = off & 4;
#pragma unroll
    for (int i = 0; i < N + 2; i++) v.w[i] = two ? v.w[i + 2] : v.w[i];
#pragma unroll
    for (int i = 0; i < N + 1; i++) v.w[i] = one ? v.w[i + 1] : v.w[i];
    if (sizeof(T) == 2) {
        const uint32_t pick = off & 2 ? 0x5432u : 0x3210u;
#pragma unroll
        for (int i = 0; i < N; i++) v.w[i] = __byte_perm(v.w[i], v.w[i + 1], pick);
    }
    mx_vec8<T> r;
    memcpy(&r, v.w, sizeof(r));
    return r;
}

// Shared memory of a tile: its elements, and its random words (of which a
// column's rounding has the same as a row's).
template <typename T, bool COLS, bool RANDOM>
struct mx_tile {
    static constexpr int ELEMENTS = COLS ? MX_TILE * MX_TILE * (int)sizeof(T) : 0;
    static constexpr int BYTES = ELEMENTS + (COLS && RANDOM ? MX_TILE * MX_TILE * 2 : 0);
};

template <typename T, bool ROWS, bool COLS, bool RANDOM, bool DROP>
__global__ void __launch_bounds__(MX_TPB, COLS ? (sizeof(T) == 4 ? 3 : 4) : RANDOM ? 4 : 5) k_mx_quantize(const __grid_constant__ mx_quantize_launch L) {
    mx_begin();
    typedef mx_tile<T, COLS, RANDOM> S;
    constexpr int W = 8 * sizeof(T) / 4;   // words of 8 elements
    extern __shared__ __align__(16) uint8_t s_tile[];
    __shared__ __align__(16) uint8_t s_rows[512], s_cols[512];
    uint32_t *s_words = (uint32_t *)(s_tile + S::ELEMENTS);
    const int tid = threadIdx.x;
    const uint32_t band = blockIdx.x / L.tiles;
    const int64_t r0 = (int64_t)band * MX_TILE, c0 = (int64_t)(blockIdx.x - band * L.tiles) * MX_TILE;
    const int64_t wide = mx_wide(L.cols);
    mx_key key = {}, drop = {};
    if (RANDOM) key = mx_key_of(L.random);
    if (DROP) drop = mx_key_of(L.drop.random);
    const int tx = tid & 15, ty = tid >> 4;
    const int64_t c = c0 + 8 * tx;
    const T *row = (const T *)L.x + (r0 + ty) * L.ld;
    uint8_t *to = ROWS ? L.along_rows.codes + mx_code_at(L.rows, r0 + ty, c / MX_BLOCK) + (tx & 3) * 4 : NULL;
    uint64_t pair = (uint64_t)((r0 + ty) * wide + c) / 2;
    const int left = (int)min((int64_t)MX_TILE, L.rows - r0), left8 = (left + 7) & ~7;   // (below 0: a tile of padding)

    // One row's 8 elements; `i` counts 16 rows.
    auto one = [&](mx_vec8<T> v, int i, bool inside) {
        const int y = ty + 16 * i;
        __align__(16) uint32_t w[W], words[4];
        if (DROP) {
            const uint32_t start = mx_start(drop, pair);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint32_t u = mx_word(drop, start ^ (j / 2));
                if ((u & 0xFFFFu) < L.drop.threshold) memset(&v.x[j], 0, sizeof(T));
                if ((u >> 16) < L.drop.threshold) memset(&v.x[j + 1], 0, sizeof(T));
            }
        }
        memcpy(w, &v, sizeof(v));
        if (RANDOM) {
            const uint32_t start = mx_start(key, pair);
#pragma unroll
            for (int j = 0; j < 4; j++) words[j] = mx_word(key, start ^ j);
        }
        if (COLS) {
            uint4 *q = (uint4 *)(s_tile + (y * MX_TILE + 8 * tx) * sizeof(T));
#pragma unroll
            for (int j = 0; j < W / 4; j++) q[j] = *(const uint4 *)(w + 4 * j);
            if (RANDOM) *(uint4 *)(s_words + y * (MX_TILE / 2) + 4 * tx) = *(const uint4 *)words;
        }
        if (ROWS) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < W; j++) m = larger(m, w[j], T());
            if constexpr (sizeof(T) == 4) {
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            } else {
                m = larger(m, __shfl_xor_sync(0xffffffffu, m, 1), T());
                m = larger(m, __shfl_xor_sync(0xffffffffu, m, 2), T());
            }
            uint32_t top = top_of(m, T());
            // (the largest product is the largest element's)
            if (DROP) top = __float_as_uint(__uint_as_float(top) * L.drop.factor);
            const uint32_t s = mx_scale(top);
            uint32_t codes = row_codes<T, RANDOM, DROP>(w, mx_inverse(s), L.drop.factor, words);
            if (s == 255u) codes = 0;
            if (inside) *(uint32_t *)(to + i * 16 * 128) = codes;   // (16 rows on the pieces of a row lie alike)
            if ((tx & 3) == 0) s_rows[(y & 31) * 16 + (y >> 5) * 4 + (tx >> 2)] = (uint8_t)s;
        }
        pair += 8 * wide;
    };
    // Whole tiles: loads a batch ahead of their use.
    constexpr int BATCH = 8 / sizeof(T);
    if (left == MX_TILE && L.vectors && c0 + MX_TILE <= L.cols) {
        row += c;
#pragma unroll 1
        for (int i = 0; i < MX_TILE / 16; i += BATCH) {
            mx_vec8<T> v[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; j++, row += 16 * L.ld) v[j] = load8(row);
#pragma unroll
            for (int j = 0; j < BATCH; j++) one(v[j], i + j, true);
        }
    } else if (left == MX_TILE && c0 > 0 && c0 + MX_TILE + 16 <= L.cols) {   // rows on any boundary, and room beside
        row += c;
#pragma unroll 1
        for (int i = 0; i < MX_TILE / 16; i += BATCH) {
            mx_pieces<T> v[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; j++) v[j] = load_pieces(row + 16 * j * L.ld);
#pragma unroll
            for (int j = 0; j < BATCH; j++, row += 16 * L.ld) one(from_pieces(v[j], row), i + j, true);
        }
    } else {
        // part of a tile; 16 rows that are all padding need no rounding
#pragma unroll 1
        for (int i = 0; i < MX_TILE / 16; i += BATCH) {
            mx_vec8<T> v[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; j++, row += 16 * L.ld) {
                memset(&v[j], 0, sizeof(v[j]));
                if (ty + 16 * (i + j) < left && c < L.cols) {
                    if (L.vectors && c + 8 <= L.cols) {
                        v[j] = load8(row + c);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            if (c + k < L.cols) v[j].x[k] = row[c + k];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < BATCH; j++) {
                if (16 * (i + j) < left8) {
                    one(v[j], i + j, ty + 16 * (i + j) < left8);
                } else {
                    const int y = ty + 16 * (i + j);
                    if (COLS) memset(s_tile + (y * MX_TILE + 8 * tx) * sizeof(T), 0, 8 * sizeof(T));
                    if (COLS && RANDOM) *(uint4 *)(s_words + y * (MX_TILE / 2) + 4 * tx) = make_uint4(0, 0, 0, 0);
                    if (ROWS && (tx & 3) == 0) s_rows[(y & 31) * 16 + (y >> 5) * 4 + (tx >> 2)] = 0;
                }
            }
        }
    }
    __syncthreads();
    if (COLS) {
        const int p = tid & 63, b = tid >> 6;
        const int64_t cc = c0 + 2 * p;
        uint32_t s[2];
        const uint32_t *q = (const uint32_t *)(s_tile + (32 * b * MX_TILE + 2 * p) * sizeof(T));
        constexpr int PITCH = MX_TILE * sizeof(T) / 4;
        if constexpr (sizeof(T) == 4) {
            uint32_t m[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const uint2 w = *(const uint2 *)(q + i * PITCH);
                m[0] = larger(m[0], w.x, T());
                m[1] = larger(m[1], w.y, T());
            }
            s[0] = m[0];
            s[1] = m[1];
        } else {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 32; i++) m = larger(m, q[i * PITCH], T());
            s[0] = top_low(m & 0xFFFFu, T());
            s[1] = top_low(m >> 16, T());
        }
        float inv[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (DROP) s[h] = __float_as_uint(__uint_as_float(s[h]) * L.drop.factor);
            s[h] = mx_scale(s[h]);
            inv[h] = mx_inverse(s[h]);
        }
        uint32_t codes[2][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float2 f[2][4];
            uint32_t add[2][8], signs[2] = {0, 0}, w[2][8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float2 x;
                if constexpr (sizeof(T) == 4) {
                    const uint2 u = *(const uint2 *)(q + (8 * i + j) * PITCH);
                    w[0][j] = u.x;
                    w[1][j] = u.y;
                    x = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
                } else {
                    w[0][j] = q[(8 * i + j) * PITCH];
                    x = two_of(w[0][j], T());
                }
                if (DROP) x = mx_mul2(x, make_float2(L.drop.factor, L.drop.factor));
                if (RANDOM) x = make_float2(fabsf(x.x) * inv[0], fabsf(x.y) * inv[1]);   // (one by one the magnitude costs nothing)
                else x = mx_mul2(x, make_float2(inv[0], inv[1]));
                if (j & 1) f[0][j / 2].y = x.x, f[1][j / 2].y = x.y;
                else f[0][j / 2].x = x.x, f[1][j / 2].x = x.y;
                if (RANDOM) {
                    const uint32_t u = s_words[(32 * b + 8 * i + j) * (MX_TILE / 2) + p];
                    add[0][j] = mx_add_low(u);
                    add[1][j] = mx_add_high(u);
                }
            }
            if (RANDOM) {
                if constexpr (sizeof(T) == 4) {
                    signs[0] = signs8<3>(w[0]);
                    signs[1] = signs8<3>(w[1]);
                } else {
                    signs[0] = signs8<1>(w[0]);
                    signs[1] = signs8<3>(w[0]);
                }
            }
            codes[0][i] = codes8<RANDOM>(f[0], signs[0], add[0]);
            codes[1][i] = codes8<RANDOM>(f[1], signs[1], add[1]);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (s[h] == 255u) codes[h][0] = codes[h][1] = codes[h][2] = codes[h][3] = 0;
            if (cc + h < mx_rows8(L.cols))
                *(uint4 *)(L.along_cols.codes + mx_code_at(L.cols, cc + h, r0 / MX_BLOCK + b)) =
                    make_uint4(codes[h][0], codes[h][1], codes[h][2], codes[h][3]);
            const int y = 2 * p + h;
            s_cols[(y & 31) * 16 + (y >> 5) * 4 + b] = (uint8_t)s[h];
        }
        __syncthreads();
    }
    // the tile is a whole group of either matrix and half of one of its panels
    if (ROWS && tid < 128 && r0 < L.rows)
        ((uint32_t *)(L.along_rows.scales + mx_scale_at(L.rows, r0, c0 / MX_BLOCK)))[tid] = ((const uint32_t *)s_rows)[tid];
    if (COLS && tid >= 128 && c0 < L.cols)
        ((uint32_t *)(L.along_cols.scales + mx_scale_at(L.cols, c0, r0 / MX_BLOCK)))[tid - 128] = ((const uint32_t *)s_cols)[tid - 128];
}

// For looking at a matrix: 8 elements a thread, stored one by one (16384 x 4096
// to bf16 170 us, to float32 226; the bytes at the copy rate 26 and 47).
template <typename T>
__global__ void __launch_bounds__(MX_TPB) k_mx_dequantize(const __grid_constant__ mx_dequantize_launch L) {
    mx_begin();
    const int64_t words = (L.m.cols + 7) / 8, all = L.m.rows * words, step = (int64_t)gridDim.x * MX_TPB;
    for (int64_t i = (int64_t)blockIdx.x * MX_TPB + threadIdx.x; i < all; i += step) {
        const int64_t r = i / words, c = (i - r * words) * 8, k = c / MX_BLOCK;
        const uint32_t codes = *(const uint32_t *)(L.m.codes + mx_code_at(L.m.rows, r, k) + (c & 31) / 2);
        const float s = mx_scale_value(L.m.scales[mx_scale_at(L.m.rows, r, k)]);
        T *out = (T *)L.out + r * L.ld + c;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c + j < L.m.cols) mx_from(&out[j], mx_value(codes >> (4 * j)) * s);
    }
}

// -------------------------------------------------------------- dropout
// Bound by memory where rows are whole 16-byte vectors: 16384 x 4096 bf16 in 49
// us, with a residual in 65 (the bytes at the copy rate: 41 and 62).  Other rows
// go two elements a thread: 16384 x 4097 in 116 and 126.
template <typename T>
__device__ __forceinline__ float2 pair_of(const T *x) { return make_float2(mx_f32(x[0]), mx_f32(x[1])); }
__device__ __forceinline__ void pair_from(float *y, float2 v) {
    y[0] = v.x;
    y[1] = v.y;
}
__device__ __forceinline__ void pair_from(__nv_bfloat16 *y, float2 v) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(v.x, v.y);
    y[0] = p.x;
    y[1] = p.y;
}
__device__ __forceinline__ void pair_from(__half *y, float2 v) {
    const __half2 p = __floats2half2_rn(v.x, v.y);
    y[0] = p.x;
    y[1] = p.y;
}

// Two elements; `w`: their random word.  (The halves are compared in the upper
// one: below the threshold there is below it here.)
template <typename T, bool RES>
__device__ __forceinline__ void drop_pair(const mx_dropout_launch &L, uint32_t w, const T *x, const T *res, T *y) {
    const uint32_t threshold = L.drop.threshold << 16;
    float2 f = mx_mul2(pair_of(x), make_float2(L.drop.factor, L.drop.factor));
    if ((w << 16) < threshold) f.x = 0.0f;
    if (w < threshold) f.y = 0.0f;
    if (RES) f = mx_add2(f, pair_of(res));
    pair_from(y, f);
}

template <typename T, bool RES>
__global__ void __launch_bounds__(MX_TPB) k_mx_dropout(const __grid_constant__ mx_dropout_launch L) {
    mx_begin();
    const mx_key key = mx_key_of(L.drop.random);
    const int64_t wide = mx_wide(L.cols), step = (int64_t)gridDim.x * MX_TPB;
    const int64_t first = (int64_t)blockIdx.x * MX_TPB + threadIdx.x;
    const T *x = (const T *)L.x, *res = (const T *)L.residual;
    T *y = (T *)L.y;
    if (L.vectors) {   // 8 elements a thread
        const int64_t words = L.cols / 8, all = L.rows * words;
        for (int64_t i = first; i < all; i += step) {
            mx_vec8<T> v, z;   // (not through the read-only cache: y may be either)
#pragma unroll
            for (int j = 0; j < (int)(sizeof(v) / 16); j++) ((uint4 *)&v)[j] = ((const uint4 *)(x + i * 8))[j];
            if (RES) {
#pragma unroll
                for (int j = 0; j < (int)(sizeof(z) / 16); j++) ((uint4 *)&z)[j] = ((const uint4 *)(res + i * 8))[j];
            }
            int64_t at = i * 8;
            if (!L.flat) {
                const int64_t r = all >> 31 ? i / words : (int64_t)((uint32_t)i / (uint32_t)words);
                at = r * wide + (i - r * words) * 8;
            }
            const uint32_t start = mx_start(key, (uint64_t)at / 2);
            mx_vec8<T> o;
#pragma unroll
            for (int j = 0; j < 8; j += 2) drop_pair<T, RES>(L, mx_word(key, start ^ (j / 2)), v.x + j, z.x + j, o.x + j);
#pragma unroll
            for (int j = 0; j < (int)(sizeof(o) / 16); j++) ((uint4 *)(y + i * 8))[j] = ((const uint4 *)&o)[j];
        }
    } else {
        const int64_t pairs = (L.cols + 1) / 2, all = L.rows * pairs;
        for (int64_t i = first; i < all; i += step) {
            const int64_t r = all >> 31 ? i / pairs : (int64_t)((uint32_t)i / (uint32_t)pairs);
            const int64_t c = (i - r * pairs) * 2, at = r * L.cols + c;
            const bool two = c + 1 < L.cols;
            T v[2], z[2], o[2];
            v[0] = x[at];
            v[1] = two ? x[at + 1] : v[0];
            if (RES) {
                z[0] = res[at];
                z[1] = two ? res[at + 1] : z[0];
            }
            drop_pair<T, RES>(L, mx_word_at(key, (uint64_t)(r * wide + c) / 2), v, z, o);
            y[at] = o[0];
            if (two) y[at + 1] = o[1];
        }
    }
}

// `units` of work, `per_cta` at a time; at most `most` CTAs.
static int grid_for(int64_t units, int per_cta, int64_t most) {
    const int64_t want = (units + per_cta - 1) / per_cta;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

// One chunk a warp, and as many CTAs as that takes: a resident grid whose warps
// take chunk after chunk reaches 0.96 of the copy rate and less (355 M float32:
// encode 707 us against 638, decode 561 against 443).
#define MX_GRID 0x7FFFFFFF
template <typename T>
static int encode(const mx_encode_launch &L, cudaStream_t s) {
    const int grid = grid_for((L.n + 255) / 256, MX_TPB / 32, MX_GRID);
    void (*kern)(const mx_encode_launch);
    if (L.vectors) {
        if (L.base) kern = L.random.on ? k_mx_encode8<T, true, true> : k_mx_encode8<T, true, false>;
        else kern = L.random.on ? k_mx_encode8<T, false, true> : k_mx_encode8<T, false, false>;
    } else {
        if (L.base) kern = L.random.on ? k_mx_encode<T, true, true> : k_mx_encode<T, true, false>;
        else kern = L.random.on ? k_mx_encode<T, false, true> : k_mx_encode<T, false, false>;
    }
    return mx_launch(kern, grid, MX_TPB, 0, 0, s, L);
}

template <typename T>
static int decode(const mx_decode_launch &L, cudaStream_t s) {
    const int grid = grid_for((L.n + 255) / 256, MX_TPB / 32, MX_GRID);
    void (*kern)(const mx_decode_launch);
    if (L.vectors) kern = L.accumulate ? k_mx_decode8<T, true> : k_mx_decode8<T, false>;
    else kern = L.accumulate ? k_mx_decode<T, true> : k_mx_decode<T, false>;
    return mx_launch(kern, grid, MX_TPB, 0, 0, s, L);
}

template <typename T, bool ROWS, bool COLS, bool RANDOM, bool DROP>
static int quantize_as(mx_quantize_launch L, cudaStream_t s) {
    // whole panels: 256 columns where rows are wanted, 256 rows where columns are
    const int64_t x = ROWS ? (L.cols + 255) / 256 * 2 : (L.cols + 127) / 128;
    const int64_t y = COLS ? (L.rows + 255) / 256 * 2 : (L.rows + 127) / 128;
    if (x * y > 0x7FFFFFFF) return cudaErrorInvalidValue;
    L.tiles = (uint32_t)x;
    const size_t smem = mx_tile<T, COLS, RANDOM>::BYTES;
    if (smem > 48 * 1024) {
        const cudaError_t e = mx_allow(k_mx_quantize<T, ROWS, COLS, RANDOM, DROP>, smem);
        if (e != cudaSuccess) return e;
    }
    return mx_launch(k_mx_quantize<T, ROWS, COLS, RANDOM, DROP>, x * y, MX_TPB, smem, 0, s, L);
}

template <typename T, bool RANDOM, bool DROP>
static int quantize_dir(const mx_quantize_launch &L, cudaStream_t s) {
    if (L.along_rows.codes && L.along_cols.codes) return quantize_as<T, true, true, RANDOM, DROP>(L, s);
    if (L.along_rows.codes) return quantize_as<T, true, false, RANDOM, DROP>(L, s);
    return quantize_as<T, false, true, RANDOM, DROP>(L, s);
}

template <typename T>
static int quantize(const mx_quantize_launch &L, cudaStream_t s) {
    if (L.random.on) return L.drop.random.on ? quantize_dir<T, true, true>(L, s) : quantize_dir<T, true, false>(L, s);
    return L.drop.random.on ? quantize_dir<T, false, true>(L, s) : quantize_dir<T, false, false>(L, s);
}

// CTAs an SM (128: 16384 x 4096 bf16 with a residual in 65.5 us; 32: 69)
#define MX_DROPS 128
template <typename T>
static int dropout(const mx_dropout_launch &L, int sms, cudaStream_t s) {
    const int64_t units = L.vectors ? L.rows * (L.cols / 8) : L.rows * ((L.cols + 1) / 2);
    const int grid = grid_for(units, MX_TPB, (int64_t)sms * MX_DROPS);
    return mx_launch(L.residual ? k_mx_dropout<T, true> : k_mx_dropout<T, false>, grid, MX_TPB, 0, 0, s, L);
}

}  // namespace

extern "C" uint32_t mc_mx_hash(uint32_t x) { return mx_mix(x); }

extern "C" void mc_mx_key(mx_random *r) {
    const mx_key k = mx_key_with(r->key, 0);
    r->a = k.a;
    r->b = k.b;
}

extern "C" int mc_launch_mx_encode(const mx_encode_launch *L, int type, void *stream) {
    if (type == FALCOM_TYPE_F32) return encode<float>(*L, (cudaStream_t)stream);
    if (type == FALCOM_TYPE_BF16) return encode<__nv_bfloat16>(*L, (cudaStream_t)stream);
    return encode<__half>(*L, (cudaStream_t)stream);
}

extern "C" int mc_launch_mx_decode(const mx_decode_launch *L, int type, void *stream) {
    if (type == FALCOM_TYPE_F32) return decode<float>(*L, (cudaStream_t)stream);
    if (type == FALCOM_TYPE_BF16) return decode<__nv_bfloat16>(*L, (cudaStream_t)stream);
    return decode<__half>(*L, (cudaStream_t)stream);
}

extern "C" int mc_launch_mx_quantize(const mx_quantize_launch *L, int type, void *stream) {
    if (type == FALCOM_TYPE_F32) return quantize<float>(*L, (cudaStream_t)stream);
    if (type == FALCOM_TYPE_BF16) return quantize<__nv_bfloat16>(*L, (cudaStream_t)stream);
    return quantize<__half>(*L, (cudaStream_t)stream);
}

extern "C" int mc_launch_mx_dequantize(const mx_dequantize_launch *L, int type, int sms, void *stream) {
    const int grid = grid_for(L->m.rows * ((L->m.cols + 7) / 8), MX_TPB, (int64_t)sms * 32);
    return mx_launch(type == FALCOM_TYPE_F32 ? k_mx_dequantize<float> : type == FALCOM_TYPE_BF16 ? k_mx_dequantize<__nv_bfloat16>
                     : k_mx_dequantize<__half>, grid, MX_TPB, 0, 0, (cudaStream_t)stream, *L);
}

extern "C" int mc_launch_mx_dropout(const mx_dropout_launch *L, int type, int sms, void *stream) {
    if (type == FALCOM_TYPE_F32) return dropout<float>(*L, sms, (cudaStream_t)stream);
    if (type == FALCOM_TYPE_BF16) return dropout<__nv_bfloat16>(*L, sms, (cudaStream_t)stream);
    return dropout<__half>(*L, sms, (cudaStream_t)stream);
}
