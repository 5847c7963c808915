// mc_mx4.cu -- 4-bit rounding (vectors with what their receivers hold,
// matrices along rows and columns), reading back, and dropout.  All of it is
// bound by memory: every element is read once and written once.

#include "mc_mx4_device.h"

namespace {

#define MX_TPB 256

// ------------------------------------------------------------- vectors
// A warp has 8 blocks; lane i has element i of each, so loads and stores are
// whole lines at any alignment, and a block's largest magnitude is one
// reduction.  The codes then change lanes: those of 8 elements of a block
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

template <typename T, bool BASE, bool RANDOM>
__global__ void __launch_bounds__(MX_TPB) k_mx_encode(const __grid_constant__ mx_encode_launch L) {
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
        const mx_key k = RANDOM ? mx_key_at(key, (uint64_t)(c * 128)) : key;
        uint32_t codes = 0, scales[2] = {0, 0};
#pragma unroll
        for (int b = 0; b < 8; b++) {
            v[b] = BASE ? mx_f32(raw[b]) - held[b] : mx_f32(raw[b]);
            const uint32_t s = mx_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(v[b]) & 0x7FFFFFFFu));
            scales[b >> 2] |= s << (8 * (b & 3));
            const float y = v[b] * mx_inverse(s);
            uint32_t code;
            if (RANDOM) {
                const uint32_t w = mx_word(k, (uint32_t)(c * 128 + 16 * b + (lane >> 1)));
                code = mx_code_random(y, lane & 1 ? w >> 16 : w & 0xFFFFu);
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
        const int bytes = (left + 1) / 2;
        uint8_t *out = L.codes + c * 128 + 4 * word;
        if (4 * word + 4 <= bytes) *(uint32_t *)out = codes;
        else
            for (int i = 0; 4 * word + i < bytes; i++) out[i] = (uint8_t)(codes >> (8 * i));
        if (lane < (left + 31) / 32) L.scales[c * 8 + lane] = (uint8_t)((lane & 4 ? scales[1] : scales[0]) >> (8 * (lane & 3)));
    }
}

template <typename T, bool ADD>
__global__ void __launch_bounds__(MX_TPB) k_mx_decode(const __grid_constant__ mx_decode_launch L) {
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
// neighbouring columns, which share their random words.
#define MX_TILE 128

template <typename T>
struct mx_vec8 {
    T x[8];
};

template <typename T>
__device__ __forceinline__ mx_vec8<T> load8(const T *p) {
    mx_vec8<T> v;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(v) / 16); i++) ((uint4 *)&v)[i] = __ldg((const uint4 *)p + i);
    return v;
}

template <typename T, bool ROWS, bool COLS, bool RANDOM, bool DROP>
__global__ void __launch_bounds__(MX_TPB) k_mx_quantize(const __grid_constant__ mx_quantize_launch L) {
    extern __shared__ __align__(16) uint8_t s_tile[];
    __shared__ __align__(16) uint8_t s_rows[512], s_cols[512];
    T *tile = (T *)s_tile;
    const int tid = threadIdx.x;
    const uint32_t band = blockIdx.x / L.tiles;
    const int64_t r0 = (int64_t)band * MX_TILE, c0 = (int64_t)(blockIdx.x - band * L.tiles) * MX_TILE;
    const int64_t wide = mx_wide(L.cols);
    mx_key key = {}, drop = {};
    if (RANDOM) key = mx_key_of(L.random);
    if (DROP) drop = mx_key_of(L.drop.random);
    const int tx = tid & 15, ty = tid >> 4;
    const int64_t c = c0 + 8 * tx;
#pragma unroll 2
    for (int i = 0; i < MX_TILE / 16; i++) {
        const int y = ty + 16 * i;
        const int64_t r = r0 + y;
        mx_vec8<T> v;
        memset(&v, 0, sizeof(v));
        if (r < L.rows && c < L.cols) {
            const T *p = (const T *)L.x + r * L.ld + c;
            if (L.vectors && c + 8 <= L.cols) {
                v = load8(p);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (c + j < L.cols) v.x[j] = p[j];
            }
        }
        const uint64_t pair = (uint64_t)(r * wide + c) / 2;
        if (DROP) {
            const mx_key k = mx_key_at(drop, pair);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint32_t w = mx_word(k, (uint32_t)pair + j / 2);
                if ((w & 0xFFFFu) < L.drop.threshold) memset(&v.x[j], 0, sizeof(T));
                if ((w >> 16) < L.drop.threshold) memset(&v.x[j + 1], 0, sizeof(T));
            }
        }
        if (COLS) {
            T *q = tile + y * MX_TILE + 8 * tx;
#pragma unroll
            for (int j = 0; j < (int)(sizeof(v) / 16); j++) ((uint4 *)q)[j] = ((const uint4 *)&v)[j];
        }
        if (ROWS) {
            float f[8];
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                f[j] = mx_f32(v.x[j]);
                if (DROP) f[j] *= L.drop.factor;
                top = max(top, __float_as_uint(f[j]) & 0x7FFFFFFFu);
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const uint32_t s = mx_scale(top);
            const float inv = mx_inverse(s);
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] *= inv;
            uint32_t codes = 0;
            if (RANDOM) {
                const mx_key k = mx_key_at(key, pair);
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const uint32_t w = mx_word(k, (uint32_t)pair + j / 2);
                    codes |= mx_code_random(f[j], w & 0xFFFFu) << (4 * j) | mx_code_random(f[j + 1], w >> 16) << (4 * j + 4);
                }
            } else {
                codes = mx_codes8(f);
            }
            if (s == 255u) codes = 0;
            const int64_t k = c / MX_BLOCK;
            if (r < mx_rows8(L.rows)) *(uint32_t *)(L.along_rows.codes + mx_code_at(L.rows, r, k) + (tx & 3) * 4) = codes;
            if ((tx & 3) == 0) s_rows[(y & 31) * 16 + (y >> 5) * 4 + (tx >> 2)] = (uint8_t)s;
        }
    }
    __syncthreads();
    if (COLS) {
        const int p = tid & 63, b = tid >> 6;
        const int64_t cc = c0 + 2 * p, rr = r0 + 32 * b;
        T v[32][2];
        const T *q = tile + 32 * b * MX_TILE + 2 * p;
#pragma unroll
        for (int i = 0; i < 32; i++) memcpy(v[i], q + i * MX_TILE, 2 * sizeof(T));
        uint32_t top[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 32; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float f = mx_f32(v[i][h]);
                if (DROP) f *= L.drop.factor;
                top[h] = max(top[h], __float_as_uint(f) & 0x7FFFFFFFu);
            }
        const uint32_t s[2] = {mx_scale(top[0]), mx_scale(top[1])};
        const float inv[2] = {mx_inverse(s[0]), mx_inverse(s[1])};
        uint32_t codes[2][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float f[2][8];
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    f[h][j] = mx_f32(v[8 * i + j][h]);
                    if (DROP) f[h][j] *= L.drop.factor;
                    f[h][j] *= inv[h];
                }
            if (RANDOM) {
                codes[0][i] = codes[1][i] = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint64_t pair = (uint64_t)((rr + 8 * i + j) * wide + cc) / 2;
                    const uint32_t w = mx_word(mx_key_at(key, pair), (uint32_t)pair);
                    codes[0][i] |= mx_code_random(f[0][j], w & 0xFFFFu) << (4 * j);
                    codes[1][i] |= mx_code_random(f[1][j], w >> 16) << (4 * j);
                }
            } else {
                codes[0][i] = mx_codes8(f[0]);
                codes[1][i] = mx_codes8(f[1]);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (s[h] == 255u) codes[h][0] = codes[h][1] = codes[h][2] = codes[h][3] = 0;
            if (cc + h < mx_rows8(L.cols))
                *(uint4 *)(L.along_cols.codes + mx_code_at(L.cols, cc + h, rr / MX_BLOCK)) =
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

template <typename T>
__global__ void __launch_bounds__(MX_TPB) k_mx_dequantize(const __grid_constant__ mx_dequantize_launch L) {
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
template <typename T, bool RES>
__device__ __forceinline__ void drop_pair(const mx_dropout_launch &L, mx_key key, uint64_t pair, const T *x, const T *res, T *y) {
    const uint32_t w = mx_word(mx_key_at(key, pair), (uint32_t)pair);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float f = (h ? w >> 16 : w & 0xFFFFu) < L.drop.threshold ? 0.0f : mx_f32(x[h]) * L.drop.factor;
        if (RES) f = f + mx_f32(res[h]);
        mx_from(&y[h], f);
    }
}

template <typename T, bool RES>
__global__ void __launch_bounds__(MX_TPB) k_mx_dropout(const __grid_constant__ mx_dropout_launch L) {
    const mx_key key = mx_key_of(L.drop.random);
    const int64_t wide = mx_wide(L.cols), step = (int64_t)gridDim.x * MX_TPB;
    const int64_t first = (int64_t)blockIdx.x * MX_TPB + threadIdx.x;
    const T *x = (const T *)L.x, *res = (const T *)L.residual;
    T *y = (T *)L.y;
    if (L.vectors) {   // 8 elements a thread
        const int64_t words = L.cols / 8, all = L.rows * words;
        for (int64_t i = first; i < all; i += step) {
            const int64_t r = i / words, c = (i - r * words) * 8;
            const mx_vec8<T> v = load8(x + i * 8);
            mx_vec8<T> o, z;
            if (RES) z = load8(res + i * 8);
            const uint64_t pair = (uint64_t)(r * wide + c) / 2;
#pragma unroll
            for (int j = 0; j < 8; j += 2) drop_pair<T, RES>(L, key, pair + j / 2, v.x + j, z.x + j, o.x + j);
#pragma unroll
            for (int j = 0; j < (int)(sizeof(o) / 16); j++) ((uint4 *)(y + i * 8))[j] = ((const uint4 *)&o)[j];
        }
    } else {
        const int64_t pairs = (L.cols + 1) / 2, all = L.rows * pairs;
        for (int64_t i = first; i < all; i += step) {
            const int64_t r = i / pairs, c = (i - r * pairs) * 2, at = r * L.cols + c;
            const bool two = c + 1 < L.cols;
            T v[2], z[2], o[2];
            v[0] = x[at];
            v[1] = two ? x[at + 1] : v[0];
            if (RES) {
                z[0] = res[at];
                z[1] = two ? res[at + 1] : z[0];
            }
            drop_pair<T, RES>(L, key, (uint64_t)(r * wide + c) / 2, v, z, o);
            y[at] = o[0];
            if (two) y[at + 1] = o[1];
        }
    }
}

static int grid_for(int64_t units, int per_cta, int sms, int per_sm) {
    const int64_t want = (units + per_cta - 1) / per_cta, most = (int64_t)sms * per_sm;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename T>
static void encode(const mx_encode_launch &L, int sms, cudaStream_t s) {
    const int grid = grid_for((L.n + 255) / 256, MX_TPB / 32, sms, 8);
    if (L.base) {
        if (L.random.on) k_mx_encode<T, true, true><<<grid, MX_TPB, 0, s>>>(L);
        else k_mx_encode<T, true, false><<<grid, MX_TPB, 0, s>>>(L);
    } else {
        if (L.random.on) k_mx_encode<T, false, true><<<grid, MX_TPB, 0, s>>>(L);
        else k_mx_encode<T, false, false><<<grid, MX_TPB, 0, s>>>(L);
    }
}

template <typename T>
static void decode(const mx_decode_launch &L, int sms, cudaStream_t s) {
    const int grid = grid_for((L.n + 255) / 256, MX_TPB / 32, sms, 8);
    if (L.accumulate) k_mx_decode<T, true><<<grid, MX_TPB, 0, s>>>(L);
    else k_mx_decode<T, false><<<grid, MX_TPB, 0, s>>>(L);
}

template <typename T, bool ROWS, bool COLS, bool RANDOM, bool DROP>
static int quantize_as(mx_quantize_launch L, cudaStream_t s) {
    // whole panels: 256 columns where rows are wanted, 256 rows where columns are
    const int64_t x = ROWS ? (L.cols + 255) / 256 * 2 : (L.cols + 127) / 128;
    const int64_t y = COLS ? (L.rows + 255) / 256 * 2 : (L.rows + 127) / 128;
    if (x * y > 0x7FFFFFFF) return cudaErrorInvalidValue;
    L.tiles = (uint32_t)x;
    const size_t smem = COLS ? MX_TILE * MX_TILE * sizeof(T) : 0;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(k_mx_quantize<T, ROWS, COLS, RANDOM, DROP>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    k_mx_quantize<T, ROWS, COLS, RANDOM, DROP><<<(unsigned)(x * y), MX_TPB, smem, s>>>(L);
    return cudaSuccess;
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

template <typename T>
static void dropout(const mx_dropout_launch &L, int sms, cudaStream_t s) {
    const int64_t units = L.vectors ? L.rows * (L.cols / 8) : L.rows * ((L.cols + 1) / 2);
    const int grid = grid_for(units, MX_TPB, sms, 32);
    if (L.residual) k_mx_dropout<T, true><<<grid, MX_TPB, 0, s>>>(L);
    else k_mx_dropout<T, false><<<grid, MX_TPB, 0, s>>>(L);
}

}  // namespace

extern "C" uint32_t mc_mx_hash(uint32_t x) { return mx_mix(x); }

extern "C" int mc_launch_mx_encode(const mx_encode_launch *L, int type, int sms, void *stream) {
    if (type == FALCOM_TYPE_F32) encode<float>(*L, sms, (cudaStream_t)stream);
    else if (type == FALCOM_TYPE_BF16) encode<__nv_bfloat16>(*L, sms, (cudaStream_t)stream);
    else encode<__half>(*L, sms, (cudaStream_t)stream);
    return cudaGetLastError();
}

extern "C" int mc_launch_mx_decode(const mx_decode_launch *L, int type, int sms, void *stream) {
    if (type == FALCOM_TYPE_F32) decode<float>(*L, sms, (cudaStream_t)stream);
    else if (type == FALCOM_TYPE_BF16) decode<__nv_bfloat16>(*L, sms, (cudaStream_t)stream);
    else decode<__half>(*L, sms, (cudaStream_t)stream);
    return cudaGetLastError();
}

extern "C" int mc_launch_mx_quantize(const mx_quantize_launch *L, int type, void *stream) {
    int e;
    if (type == FALCOM_TYPE_F32) e = quantize<float>(*L, (cudaStream_t)stream);
    else if (type == FALCOM_TYPE_BF16) e = quantize<__nv_bfloat16>(*L, (cudaStream_t)stream);
    else e = quantize<__half>(*L, (cudaStream_t)stream);
    const int late = cudaGetLastError();
    return e ? e : late;
}

extern "C" int mc_launch_mx_dequantize(const mx_dequantize_launch *L, int type, void *stream) {
    const int64_t all = L->m.rows * ((L->m.cols + 7) / 8), most = 148 * 64;
    const int64_t want = (all + MX_TPB - 1) / MX_TPB;
    const int grid = (int)(want < most ? want : most);
    cudaStream_t s = (cudaStream_t)stream;
    if (type == FALCOM_TYPE_F32) k_mx_dequantize<float><<<grid, MX_TPB, 0, s>>>(*L);
    else if (type == FALCOM_TYPE_BF16) k_mx_dequantize<__nv_bfloat16><<<grid, MX_TPB, 0, s>>>(*L);
    else k_mx_dequantize<__half><<<grid, MX_TPB, 0, s>>>(*L);
    return cudaGetLastError();
}

extern "C" int mc_launch_mx_dropout(const mx_dropout_launch *L, int type, int sms, void *stream) {
    if (type == FALCOM_TYPE_F32) dropout<float>(*L, sms, (cudaStream_t)stream);
    else if (type == FALCOM_TYPE_BF16) dropout<__nv_bfloat16>(*L, sms, (cudaStream_t)stream);
    else dropout<__half>(*L, sms, (cudaStream_t)stream);
    return cudaGetLastError();
}
