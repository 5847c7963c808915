/*
 * mc_mx4.c -- host side of the 4-bit entry points (falcom_mx4_*) and of
 * falcom_dropout: argument checks and launches.  The kernels are in
 * mc_mx4.cu and mc_mx4_product.cu.
 */
#include <cuda_runtime_api.h>
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "mc_call.h"
#include "mc_internal.h"
#include "mc_mx4.h"

static const size_t g_type_size[MX_TYPES] = {4, 2, 2};
#define MX_MOST ((size_t)1 << 31)   /* rows or columns */

static int invalid(const char *who, const char *what) {
    fprintf(stderr, "[ERROR] %s: %s\n", who, what);
    return ERROR_INVALID_PARAM;
}

static int known_type(int dtype) { return dtype >= 0 && dtype < MX_TYPES; }

/* Where a call's arrays lie; the device is that of the first. */
typedef struct {
    const char *who;
    int device, n, ok;
    struct {
        uintptr_t lo, hi;
        int written;
    } span[8];
} mx_call;

static void begin(mx_call *c, const char *who) {
    memset(c, 0, sizeof(*c));
    c->who = who;
    c->device = -1;
    c->ok = 1;
}

static void array(mx_call *c, const char *what, const void *p, size_t bytes, size_t align, int written) {
    if (!c->ok || bytes == 0) return;
    if (c->device < 0) {
        struct cudaPointerAttributes at;
        if (!p || cudaPointerGetAttributes(&at, p) != cudaSuccess ||
            (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)) {
            (void)cudaGetLastError();
            fprintf(stderr, "[ERROR] %s: %s is not device memory\n", c->who, what);
            c->ok = 0;
            return;
        }
        c->device = at.device;
    }
    const uintptr_t lo = (uintptr_t)p, hi = lo + bytes;
    if (!check_argument(c->who, what, p, bytes, align, c->device)) {
        c->ok = 0;
        return;
    }
    for (int i = 0; i < c->n; i++)
        if ((written || c->span[i].written) && lo < c->span[i].hi && c->span[i].lo < hi) {
            fprintf(stderr, "[ERROR] %s: %s overlaps another array of the call\n", c->who, what);
            c->ok = 0;
            return;
        }
    c->span[c->n].lo = lo;
    c->span[c->n].hi = hi;
    c->span[c->n].written = written;
    c->n++;
}

static int sms_of(int device) {
    static int known[64];
    if (device < 0 || device >= 64) return 0;
    int n = __atomic_load_n(&known[device], __ATOMIC_RELAXED);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
            (void)cudaGetLastError();
            return 0;
        }
        __atomic_store_n(&known[device], n, __ATOMIC_RELAXED);
    }
    return n;
}

/* Makes the call's device current.  0: go on (leave(*prev, device) after). */
static int go(const mx_call *c, int *prev, int *sms) {
    if (!c->ok) return ERROR_INVALID_PARAM;
    if (error_pending(c->who)) return ERROR_COMPRESSION;
    *prev = enter(c->device);
    if (*prev == -2) return ERROR_COMPRESSION;
    *sms = sms_of(c->device);
    if (*sms <= 0) {
        leave(*prev, c->device);
        return ERROR_COMPRESSION;
    }
    return ERROR_NONE;
}

static int done(const mx_call *c, int prev, int e) {
    leave(prev, c->device);
    return e == 0 ? ERROR_NONE : launch_failed(c->who, e);
}

static void random_of(mx_call *c, mx_random *out, const falcom_random *r, uint32_t purpose) {
    if (!r) return;
    if (r->counter) array(c, "counter", r->counter, sizeof(*r->counter), 8, 0);
    out->key = mc_mx_hash(mc_mx_hash((uint32_t)r->seed ^ purpose) ^ (uint32_t)(r->seed >> 32));
    out->counter = r->counter;
    out->on = 1;
}

/* p in [0, 1) that is not 1 after rounding to 16 bits; on only where something is dropped */
static int drop_of(mx_call *c, mx_drop *out, const falcom_dropout_args *d) {
    if (!d) return 1;
    if (!(d->p >= 0.0) || floor(d->p * 65536.0 + 0.5) >= 65536.0) return 0;
    out->threshold = (uint32_t)floor(d->p * 65536.0 + 0.5);
    out->factor = (float)(65536.0 / (65536.0 - out->threshold));
    random_of(c, &out->random, &d->random, 0x7F4A7C15u);
    out->random.on = out->threshold > 0;
    return 1;
}

#define ROUNDING 0x9E3779B9u
static const mx_powers g_powers = MX_POWERS;

MC_EXPORT int falcom_mx4_encode(const void *x, int dtype, size_t n, float *base, const falcom_random *random,
                                void *codes, void *scales, void *stream) {
    static const char *who = "falcom_mx4_encode";
    if (!known_type(dtype)) return invalid(who, "unknown type");
    if (n > (size_t)1 << 40) return invalid(who, "too many elements");
    if (n == 0) return ERROR_NONE;
    mx_call c;
    mx_encode_launch L;
    memset(&L, 0, sizeof(L));
    begin(&c, who);
    array(&c, "x", x, n * g_type_size[dtype], g_type_size[dtype], 0);
    if (base) array(&c, "base", base, n * 4, 4, 1);
    array(&c, "codes", codes, (n + 1) / 2, 16, 1);
    array(&c, "scales", scales, (n + 31) / 32, 16, 1);
    random_of(&c, &L.random, random, ROUNDING);
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    L.x = x;
    L.n = (int64_t)n;
    L.base = base;
    L.powers = g_powers;
    L.codes = (uint8_t *)codes;
    L.scales = (uint8_t *)scales;
    return done(&c, prev, mc_launch_mx_encode(&L, dtype, sms, stream));
}

MC_EXPORT int falcom_mx4_decode(const void *codes, const void *scales, size_t n, float weight, int accumulate,
                                void *out, int dtype, void *stream) {
    static const char *who = "falcom_mx4_decode";
    if (!known_type(dtype)) return invalid(who, "unknown type");
    if (n > (size_t)1 << 40 || !isfinite(weight)) return invalid(who, "too many elements, or a weight that is not finite");
    if (n == 0) return ERROR_NONE;
    mx_call c;
    begin(&c, who);
    array(&c, "out", out, n * g_type_size[dtype], g_type_size[dtype], 1);
    array(&c, "codes", codes, (n + 1) / 2, 16, 0);
    array(&c, "scales", scales, (n + 31) / 32, 16, 0);
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    mx_decode_launch L;
    memset(&L, 0, sizeof(L));
    L.codes = (const uint8_t *)codes;
    L.scales = (const uint8_t *)scales;
    L.n = (int64_t)n;
    L.out = out;
    L.weight = weight;
    L.accumulate = accumulate != 0;
    return done(&c, prev, mc_launch_mx_decode(&L, dtype, sms, stream));
}

static int matrix_size_ok(size_t rows, size_t cols) { return rows > 0 && cols > 0 && rows <= MX_MOST && cols <= MX_MOST; }

MC_EXPORT size_t falcom_mx4_codes_bytes(size_t rows, size_t cols) {
    return matrix_size_ok(rows, cols) ? (cols + 255) / 256 * ((rows + 7) / 8 * 8) * 128 : 0;
}

MC_EXPORT size_t falcom_mx4_scales_bytes(size_t rows, size_t cols) {
    return matrix_size_ok(rows, cols) ? (cols + 255) / 256 * ((rows + 127) / 128) * 1024 : 0;
}

static void matrix_of(mx_call *c, mx_matrix *out, const falcom_mx4_matrix *m, const char *what, int written) {
    array(c, what, m->codes, falcom_mx4_codes_bytes(m->rows, m->cols), 16, written);
    array(c, what, m->scales, falcom_mx4_scales_bytes(m->rows, m->cols), 16, written);
    out->codes = (uint8_t *)m->codes;
    out->scales = (uint8_t *)m->scales;
    out->rows = (int64_t)m->rows;
    out->cols = (int64_t)m->cols;
}

/* Bytes from the first to the last element; 0 when the rows overlap. */
static size_t extent(size_t rows, size_t cols, size_t ld, size_t size) {
    if (rows > 1 && (ld < cols || ld > (size_t)1 << 40)) return 0;
    return ((rows - 1) * (rows > 1 ? ld : 0) + cols) * size;
}

MC_EXPORT int falcom_mx4_quantize(const void *x, int dtype, size_t rows, size_t cols, size_t ld,
                                  const falcom_random *random, const falcom_dropout_args *drop,
                                  const falcom_mx4_matrix *along_rows, const falcom_mx4_matrix *along_cols,
                                  void *stream) {
    static const char *who = "falcom_mx4_quantize";
    if (!known_type(dtype)) return invalid(who, "unknown type");
    if (rows > MX_MOST || cols > MX_MOST) return invalid(who, "too many rows or columns");
    if ((along_rows && (along_rows->rows != rows || along_rows->cols != cols)) ||
        (along_cols && (along_cols->rows != cols || along_cols->cols != rows)))
        return invalid(who, "a result has other sizes than x");
    if (rows == 0 || cols == 0 || (!along_rows && !along_cols)) return ERROR_NONE;
    const size_t bytes = extent(rows, cols, ld, g_type_size[dtype]);
    if (bytes == 0) return invalid(who, "rows of x overlap");
    mx_call c;
    mx_quantize_launch L;
    memset(&L, 0, sizeof(L));
    begin(&c, who);
    array(&c, "x", x, bytes, g_type_size[dtype], 0);
    if (along_rows) matrix_of(&c, &L.along_rows, along_rows, "along_rows", 1);
    if (along_cols) matrix_of(&c, &L.along_cols, along_cols, "along_cols", 1);
    random_of(&c, &L.random, random, ROUNDING);
    if (!drop_of(&c, &L.drop, drop)) return invalid(who, "p must lie in [0, 1)");
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    L.x = x;
    L.rows = (int64_t)rows;
    L.cols = (int64_t)cols;
    L.ld = (int64_t)ld;
    L.powers = g_powers;
    L.vectors = ((uintptr_t)x & 15) == 0 && (rows == 1 || ld * g_type_size[dtype] % 16 == 0);
    return done(&c, prev, mc_launch_mx_quantize(&L, dtype, stream));
}

MC_EXPORT int falcom_mx4_dequantize(const falcom_mx4_matrix *m, void *out, int dtype, size_t ld, void *stream) {
    static const char *who = "falcom_mx4_dequantize";
    if (!m || !known_type(dtype)) return invalid(who, "no matrix, or an unknown type");
    if (m->rows > MX_MOST || m->cols > MX_MOST) return invalid(who, "too many rows or columns");
    if (m->rows == 0 || m->cols == 0) return ERROR_NONE;
    const size_t bytes = extent(m->rows, m->cols, ld, g_type_size[dtype]);
    if (bytes == 0) return invalid(who, "rows of out overlap");
    mx_call c;
    mx_dequantize_launch L;
    memset(&L, 0, sizeof(L));
    begin(&c, who);
    array(&c, "out", out, bytes, g_type_size[dtype], 1);
    matrix_of(&c, &L.m, m, "the matrix", 0);
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    L.out = out;
    L.ld = (int64_t)ld;
    return done(&c, prev, mc_launch_mx_dequantize(&L, dtype, stream));
}

MC_EXPORT int falcom_mx4_product(const falcom_mx4_matrix *a, const falcom_mx4_matrix *b, void *out, int dtype,
                                 size_t ld, const falcom_dropout_args *drop, void *stream) {
    static const char *who = "falcom_mx4_product";
    if (!a || !b || !known_type(dtype)) return invalid(who, "a factor is missing, or an unknown type");
    if (a->cols != b->cols) return invalid(who, "the factors have different numbers of columns");
    if (a->rows > MX_MOST || b->rows > MX_MOST || a->cols > MX_MOST) return invalid(who, "too many rows or columns");
    if (a->rows == 0 || b->rows == 0) return ERROR_NONE;
    const size_t bytes = extent(a->rows, b->rows, ld, g_type_size[dtype]);
    if (bytes == 0) return invalid(who, "rows of out overlap");
    mx_call c;
    mx_product_launch L;
    memset(&L, 0, sizeof(L));
    begin(&c, who);
    array(&c, "out", out, bytes, g_type_size[dtype], 1);
    matrix_of(&c, &L.a, a, "a", 0);
    matrix_of(&c, &L.b, b, "b", 0);
    if (!drop_of(&c, &L.drop, drop)) return invalid(who, "p must lie in [0, 1)");
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    L.out = out;
    L.ld = (int64_t)ld;
    L.powers = g_powers;
    return done(&c, prev, mc_launch_mx_product(&L, dtype, sms, stream));
}

MC_EXPORT int falcom_mx4_errors(void) {
    uint32_t word = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = (cudaError_t)mc_mx_errors(&word);
    if (e != cudaSuccess) return ERROR_COMPRESSION;
    return word != 0;
}

MC_EXPORT int falcom_dropout(const void *x, const void *residual, void *y, int dtype, size_t rows, size_t cols,
                             const falcom_dropout_args *drop, void *stream) {
    static const char *who = "falcom_dropout";
    if (!drop || !known_type(dtype)) return invalid(who, "no arguments, or an unknown type");
    if (rows > MX_MOST || cols > MX_MOST) return invalid(who, "too many rows or columns");
    mx_call c;
    mx_dropout_launch L;
    memset(&L, 0, sizeof(L));
    begin(&c, who);
    const size_t size = g_type_size[dtype], bytes = rows * cols * size;
    array(&c, "y", y, bytes, size, 1);
    if (x != y) array(&c, "x", x, bytes, size, 0);
    if (residual && residual != y) array(&c, "residual", residual, bytes, size, 0);
    if (!drop_of(&c, &L.drop, drop)) return invalid(who, "p must lie in [0, 1)");
    if (bytes == 0) return ERROR_NONE;
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    L.x = x;
    L.residual = residual;
    L.y = y;
    L.rows = (int64_t)rows;
    L.cols = (int64_t)cols;
    L.powers = g_powers;
    L.vectors = (((uintptr_t)x | (uintptr_t)y | (uintptr_t)residual) & 15) == 0 && cols % 8 == 0;
    return done(&c, prev, mc_launch_mx_dropout(&L, dtype, sms, stream));
}
