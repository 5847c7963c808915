/*
 * mc_mx4.c -- host side of the 4-bit entry points (falcom_mx4_*) and of
 * falcom_dropout: argument checks and launches.  The kernels are in
 * mc_mx4.cu and mc_mx4_product.cu.
 */
#include <cuda_runtime_api.h>
#include <math.h>
#include <pthread.h>
#include <stdio.h>
#include <string.h>

#include "mc_call.h"
#include "mc_internal.h"
#include "mc_mx4.h"

static const size_t g_type_size[MX_TYPES] = {4, 2, 2};
#define MX_MOST ((size_t)1 << 31)       /* rows or columns */
#define MX_ELEMENTS ((size_t)1 << 46)   /* of a matrix */

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
    mc_mx_key(out);
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

#define VECTOR_ELEMENTS ((size_t)1 << 40)

static size_t codes_of(size_t n) { return (n + 1) / 2; }
/* Where a vector's scales begin in one run of bytes. */
static size_t scales_at(size_t n) { return (codes_of(n) + 15) / 16 * 16; }

MC_EXPORT size_t falcom_mx4_vector_bytes(size_t n) {
    return n <= VECTOR_ELEMENTS ? scales_at(n) + (n + 31) / 32 : 0;
}

/* `scales` NULL: codes is the whole vector. */
static int encode(const char *who, const void *x, int dtype, size_t n, float *base, const falcom_random *random,
                  uint8_t *codes, uint8_t *scales, void *stream) {
    if (!known_type(dtype)) return invalid(who, "unknown type");
    if (n > VECTOR_ELEMENTS) return invalid(who, "too many elements");
    if (n == 0) return ERROR_NONE;
    mx_call c;
    mx_encode_launch L;
    memset(&L, 0, sizeof(L));
    begin(&c, who);
    array(&c, "x", x, n * g_type_size[dtype], g_type_size[dtype], 0);
    if (base) array(&c, "base", base, n * 4, 4, 1);
    L.unit = scales ? 1 : 16;
    if (scales) {
        array(&c, "codes", codes, codes_of(n), 16, 1);
        array(&c, "scales", scales, (n + 31) / 32, 16, 1);
    } else {
        array(&c, "the vector", codes, falcom_mx4_vector_bytes(n), 16, 1);
    }
    random_of(&c, &L.random, random, ROUNDING);
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    L.x = x;
    L.n = (int64_t)n;
    L.base = base;
    L.codes = codes;
    L.scales = scales ? scales : codes + scales_at(n);
    L.vectors = (((uintptr_t)x | (uintptr_t)base) & 15) == 0;
    return done(&c, prev, mc_launch_mx_encode(&L, dtype, stream));
}

MC_EXPORT int falcom_mx4_encode(const void *x, int dtype, size_t n, float *base, const falcom_random *random,
                                void *codes, void *scales, void *stream) {
    static const char *who = "falcom_mx4_encode";
    if (n > 0 && !scales) return invalid(who, "no scales");
    return encode(who, x, dtype, n, base, random, (uint8_t *)codes, (uint8_t *)scales, stream);
}

MC_EXPORT int falcom_mx4_encode_vector(const void *x, int dtype, size_t n, float *base, const falcom_random *random,
                                       void *vector, void *stream) {
    return encode("falcom_mx4_encode_vector", x, dtype, n, base, random, (uint8_t *)vector, NULL, stream);
}

MC_EXPORT int falcom_mx4_decode(const void *codes, const void *scales, size_t n, float weight, int accumulate,
                                void *out, int dtype, void *stream) {
    static const char *who = "falcom_mx4_decode";
    if (!known_type(dtype)) return invalid(who, "unknown type");
    if (n > VECTOR_ELEMENTS || !isfinite(weight)) return invalid(who, "too many elements, or a weight that is not finite");
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
    L.vectors = ((uintptr_t)out & 15) == 0;
    return done(&c, prev, mc_launch_mx_decode(&L, dtype, stream));
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

/* Bytes from the first to the last element; 0 when the rows overlap or lie too far apart. */
static size_t extent(size_t rows, size_t cols, size_t ld, size_t size) {
    if (rows > 1 && (ld < cols || ld > MX_ELEMENTS / rows)) return 0;
    return ((rows - 1) * (rows > 1 ? ld : 0) + cols) * size;
}

static int quantize(const void *x, int dtype, size_t rows, size_t cols, size_t ld, const mx_random *random,
                    const mx_drop *drop, const mx_matrix *along_rows, const mx_matrix *along_cols, void *stream) {
    mx_quantize_launch L;
    memset(&L, 0, sizeof(L));
    if (rows == 0 || cols == 0 || (!along_rows && !along_cols)) return 0;
    L.x = x;
    L.rows = (int64_t)rows;
    L.cols = (int64_t)cols;
    L.ld = (int64_t)ld;
    if (random) L.random = *random;
    if (drop) L.drop = *drop;
    if (along_rows) L.along_rows = *along_rows;
    if (along_cols) L.along_cols = *along_cols;
    L.vectors = ((uintptr_t)x & 15) == 0 && (rows == 1 || ld * g_type_size[dtype] % 16 == 0);
    return mc_launch_mx_quantize(&L, dtype, stream);
}

static int product(const mx_matrix *a, const mx_matrix *b, void *out, int dtype, size_t ld, const mx_drop *drop, int sms,
                   void *stream) {
    mx_product_launch L;
    memset(&L, 0, sizeof(L));
    if (a->rows == 0 || b->rows == 0) return 0;
    L.a = *a;
    L.b = *b;
    L.out = out;
    L.ld = (int64_t)ld;
    if (drop) L.drop = *drop;
    return mc_launch_mx_product(&L, dtype, sms, stream);
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
    mx_random r = {0, 0, NULL, 0, 0};
    mx_drop d = {{0, 0, NULL, 0, 0}, 0, 0};
    mx_matrix by_rows, by_cols;
    mx_call c;
    begin(&c, who);
    if (!drop_of(&c, &d, drop)) return invalid(who, "p must lie in [0, 1)");
    if (rows == 0 || cols == 0 || (!along_rows && !along_cols)) return ERROR_NONE;
    const size_t bytes = extent(rows, cols, ld, g_type_size[dtype]);
    if (bytes == 0) return invalid(who, "rows of x overlap, or lie too far apart");
    array(&c, "x", x, bytes, g_type_size[dtype], 0);
    if (along_rows) matrix_of(&c, &by_rows, along_rows, "along_rows", 1);
    if (along_cols) matrix_of(&c, &by_cols, along_cols, "along_cols", 1);
    random_of(&c, &r, random, ROUNDING);
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    return done(&c, prev, quantize(x, dtype, rows, cols, ld, &r, &d, along_rows ? &by_rows : NULL,
                                   along_cols ? &by_cols : NULL, stream));
}

MC_EXPORT int falcom_mx4_dequantize(const falcom_mx4_matrix *m, void *out, int dtype, size_t ld, void *stream) {
    static const char *who = "falcom_mx4_dequantize";
    if (!m || !known_type(dtype)) return invalid(who, "no matrix, or an unknown type");
    if (m->rows > MX_MOST || m->cols > MX_MOST) return invalid(who, "too many rows or columns");
    if (m->rows == 0 || m->cols == 0) return ERROR_NONE;
    const size_t bytes = extent(m->rows, m->cols, ld, g_type_size[dtype]);
    if (bytes == 0) return invalid(who, "rows of out overlap, or lie too far apart");
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
    return done(&c, prev, mc_launch_mx_dequantize(&L, dtype, sms, stream));
}

MC_EXPORT int falcom_mx4_product(const falcom_mx4_matrix *a, const falcom_mx4_matrix *b, void *out, int dtype,
                                 size_t ld, const falcom_dropout_args *drop, void *stream) {
    static const char *who = "falcom_mx4_product";
    if (!a || !b || !known_type(dtype)) return invalid(who, "a factor is missing, or an unknown type");
    if (a->cols != b->cols) return invalid(who, "the factors have different numbers of columns");
    if (a->rows > MX_MOST || b->rows > MX_MOST || a->cols > MX_MOST) return invalid(who, "too many rows or columns");
    mx_drop d = {{0, 0, NULL, 0, 0}, 0, 0};
    mx_matrix ma, mb;
    mx_call c;
    begin(&c, who);
    if (!drop_of(&c, &d, drop)) return invalid(who, "p must lie in [0, 1)");
    if (a->rows == 0 || b->rows == 0) return ERROR_NONE;
    const size_t bytes = extent(a->rows, b->rows, ld, g_type_size[dtype]);
    if (bytes == 0) return invalid(who, "rows of out overlap, or lie too far apart");
    array(&c, "out", out, bytes, g_type_size[dtype], 1);
    matrix_of(&c, &ma, a, "a", 0);
    matrix_of(&c, &mb, b, "b", 0);
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    return done(&c, prev, product(&ma, &mb, out, dtype, ld, &d, sms, stream));
}

/* A matrix at *at, which moves behind it. */
static size_t matrix_bytes(size_t rows, size_t cols) {
    return falcom_mx4_codes_bytes(rows, cols) + falcom_mx4_scales_bytes(rows, cols);
}

static mx_matrix matrix_in(uint8_t **at, size_t rows, size_t cols) {
    mx_matrix m;
    m.codes = *at;
    m.scales = *at + falcom_mx4_codes_bytes(rows, cols);
    m.rows = (int64_t)rows;
    m.cols = (int64_t)cols;
    *at += matrix_bytes(rows, cols);
    return m;
}

static int rounds_inside(size_t rows, size_t cols) {
    return rows <= MX_ROUND_ROWS && cols <= MX_ROUND_COLS && rows * cols <= MX_ROUND_ELEMENTS;
}

MC_EXPORT size_t falcom_mx4_work_bytes(size_t rows, size_t cols) {
    return rounds_inside(rows, cols) ? 0 : matrix_bytes(rows, cols);
}

MC_EXPORT int falcom_mx4_product_of(const void *x, int x_type, size_t rows, size_t ld_x, const falcom_mx4_matrix *b,
                                    void *out, int dtype, size_t ld, void *work, void *stream) {
    static const char *who = "falcom_mx4_product_of";
    if (!b || !known_type(dtype) || !known_type(x_type)) return invalid(who, "a factor is missing, or an unknown type");
    if (rows > MX_MOST || b->rows > MX_MOST || b->cols > MX_MOST) return invalid(who, "too many rows or columns");
    if (rows == 0 || b->rows == 0) return ERROR_NONE;
    const size_t from = b->cols ? extent(rows, b->cols, ld_x, g_type_size[x_type]) : 0;
    const size_t bytes = extent(rows, b->rows, ld, g_type_size[dtype]);
    if (bytes == 0 || (from == 0 && b->cols)) return invalid(who, "rows of x or of out overlap, or lie too far apart");
    mx_matrix mb;
    mx_call c;
    begin(&c, who);
    array(&c, "out", out, bytes, g_type_size[dtype], 1);
    array(&c, "x", x, from, g_type_size[x_type], 0);
    array(&c, "work", work, falcom_mx4_work_bytes(rows, b->cols), 16, 1);
    matrix_of(&c, &mb, b, "b", 0);
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    if (rounds_inside(rows, b->cols)) {
        mx_product_launch L;
        memset(&L, 0, sizeof(L));
        L.a.rows = (int64_t)rows;
        L.a.cols = mb.cols;
        L.b = mb;
        L.out = out;
        L.ld = (int64_t)ld;
        L.x = x;
        L.ld_x = (int64_t)ld_x;
        L.x_type = x_type;
        L.vectors = ((uintptr_t)x & 15) == 0 && (rows == 1 || ld_x * g_type_size[x_type] % 16 == 0);
        return done(&c, prev, mc_launch_mx_product(&L, dtype, sms, stream));
    }
    uint8_t *at = (uint8_t *)work;
    const mx_matrix a = matrix_in(&at, rows, b->cols);
    int e = quantize(x, x_type, rows, b->cols, ld_x, NULL, NULL, &a, NULL, stream);
    if (e == 0) e = product(&a, &mb, out, dtype, ld, NULL, sms, stream);
    return done(&c, prev, e);
}

/* ------------------------------------------------------------------ layers */
static int layer_ok(const char *who, const falcom_mx4_linear *l) {
    if (!l || !known_type(l->x_type) || !known_type(l->weight_type))
        return invalid(who, "no layer, or an unknown type"), 0;
    if (l->rows > MX_MOST || l->cols > MX_MOST || l->outs > MX_MOST)
        return invalid(who, "too many rows, columns or outputs"), 0;
    return 1;
}

MC_EXPORT size_t falcom_mx4_linear_kept_bytes(const falcom_mx4_linear *l) {
    if (!l) return 0;
    return (l->want_dx ? matrix_bytes(l->cols, l->outs) : 0) + (l->want_dw ? matrix_bytes(l->cols, l->rows) : 0);
}

MC_EXPORT size_t falcom_mx4_linear_work_bytes(const falcom_mx4_linear *l, int backward) {
    if (!l) return 0;
    if (backward) return (l->want_dx ? matrix_bytes(l->rows, l->outs) : 0) + (l->want_dw ? matrix_bytes(l->outs, l->rows) : 0);
    return matrix_bytes(l->rows, l->cols) + matrix_bytes(l->outs, l->cols);
}

static int layer_drop(mx_call *c, mx_drop *out, const falcom_mx4_linear *l) {
    falcom_dropout_args d;
    d.p = l->p;
    d.random = l->random;
    if (l->p == 0.0) d.random.counter = NULL;   /* nothing reads it */
    return drop_of(c, out, &d);
}

MC_EXPORT int falcom_mx4_linear_forward(const falcom_mx4_linear *l, const void *x, size_t ld_x, const void *weight,
                                        size_t ld_weight, void *y, void *kept, void *work, void *stream) {
    static const char *who = "falcom_mx4_linear_forward";
    if (!layer_ok(who, l)) return ERROR_INVALID_PARAM;
    const size_t xs = g_type_size[l->x_type], ws = g_type_size[l->weight_type];
    const int no_x = l->rows == 0 || l->cols == 0, no_w = l->outs == 0 || l->cols == 0;
    const size_t x_bytes = no_x ? 0 : extent(l->rows, l->cols, ld_x, xs), w_bytes = no_w ? 0 : extent(l->outs, l->cols, ld_weight, ws);
    if ((!no_x && x_bytes == 0) || (!no_w && w_bytes == 0) || l->rows * l->outs > MX_ELEMENTS)
        return invalid(who, "rows of x or of the weight overlap, or sizes are out of range");
    mx_drop d = {{0, 0, NULL, 0, 0}, 0, 0};
    mx_call c;
    begin(&c, who);
    if (!layer_drop(&c, &d, l)) return invalid(who, "p must lie in [0, 1)");
    array(&c, "y", y, l->rows * l->outs * xs, xs, 1);
    array(&c, "x", x, x_bytes, xs, 0);
    array(&c, "weight", weight, w_bytes, ws, 0);
    array(&c, "kept", kept, falcom_mx4_linear_kept_bytes(l), 16, 1);
    array(&c, "work", work, falcom_mx4_linear_work_bytes(l, 0), 16, 1);
    if (c.ok && c.n == 0) return ERROR_NONE;   /* nothing at all */
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    uint8_t *at = (uint8_t *)work, *keep = (uint8_t *)kept;
    const mx_matrix a = matrix_in(&at, l->rows, l->cols), b = matrix_in(&at, l->outs, l->cols);
    mx_matrix bt, atr;
    if (l->want_dx) bt = matrix_in(&keep, l->cols, l->outs);
    if (l->want_dw) atr = matrix_in(&keep, l->cols, l->rows);
    int e = quantize(weight, l->weight_type, l->outs, l->cols, ld_weight, NULL, NULL, &b, l->want_dx ? &bt : NULL, stream);
    if (e == 0) e = quantize(x, l->x_type, l->rows, l->cols, ld_x, NULL, &d, &a, l->want_dw ? &atr : NULL, stream);
    if (e == 0) e = product(&a, &b, y, l->x_type, l->outs, NULL, sms, stream);
    return done(&c, prev, e);
}

MC_EXPORT int falcom_mx4_linear_backward(const falcom_mx4_linear *l, const void *dy, size_t ld_dy, const void *kept,
                                         void *dx, void *dw, void *work, void *stream) {
    static const char *who = "falcom_mx4_linear_backward";
    if (!layer_ok(who, l)) return ERROR_INVALID_PARAM;
    if ((dx && !l->want_dx) || (dw && !l->want_dw)) return invalid(who, "forward kept nothing for this gradient");
    const size_t xs = g_type_size[l->x_type], ws = g_type_size[l->weight_type];
    const int none = l->rows == 0 || l->outs == 0;
    const size_t dy_bytes = none ? 0 : extent(l->rows, l->outs, ld_dy, xs);
    if ((!none && dy_bytes == 0) || l->rows * l->cols > MX_ELEMENTS || l->outs * l->cols > MX_ELEMENTS)
        return invalid(who, "rows of dy overlap, or sizes are out of range");
    mx_random r = {0, 0, NULL, 0, 0};
    mx_drop d = {{0, 0, NULL, 0, 0}, 0, 0};
    mx_call c;
    begin(&c, who);
    if (!layer_drop(&c, &d, l)) return invalid(who, "p must lie in [0, 1)");
    if (dx) array(&c, "dx", dx, l->rows * l->cols * xs, xs, 1);
    if (dw) array(&c, "dw", dw, l->outs * l->cols * ws, ws, 1);
    array(&c, "dy", dy, dy_bytes, xs, 0);
    array(&c, "kept", kept, falcom_mx4_linear_kept_bytes(l), 16, 0);
    array(&c, "work", work, falcom_mx4_linear_work_bytes(l, 1), 16, 1);
    random_of(&c, &r, &l->random, ROUNDING);
    if (c.ok && c.n == 0) return ERROR_NONE;
    int prev, sms, rc = go(&c, &prev, &sms);
    if (rc) return rc;
    uint8_t *at = (uint8_t *)work, *keep = (uint8_t *)kept;
    mx_matrix g, gt, bt, atr;
    if (l->want_dx) {
        g = matrix_in(&at, l->rows, l->outs);
        bt = matrix_in(&keep, l->cols, l->outs);
    }
    if (l->want_dw) {
        gt = matrix_in(&at, l->outs, l->rows);
        atr = matrix_in(&keep, l->cols, l->rows);
    }
    int e = quantize(dy, l->x_type, l->rows, l->outs, ld_dy, &r, NULL, dx ? &g : NULL, dw ? &gt : NULL, stream);
    if (e == 0 && dx) e = product(&g, &bt, dx, l->x_type, l->cols, &d, sms, stream);
    if (e == 0 && dw) e = product(&gt, &atr, dw, l->weight_type, l->cols, NULL, sms, stream);
    return done(&c, prev, e);
}

MC_EXPORT int falcom_mx4_errors(void) {
    static pthread_mutex_t lock = PTHREAD_MUTEX_INITIALIZER;
    static uint32_t reported[64];   /* of each device: CTAs that gave up, which the kernels count */
    uint32_t count = 0;
    int device = -1, rc = ERROR_COMPRESSION;
    pthread_mutex_lock(&lock);
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = (cudaError_t)mc_mx_errors(&count);
    if (e == cudaSuccess && device >= 0 && device < 64) {
        rc = count != reported[device] && count != 0;   /* (0 again: the device was reset) */
        reported[device] = count;
    }
    pthread_mutex_unlock(&lock);
    return rc;
}

MC_EXPORT int falcom_dropout(const void *x, const void *residual, void *y, int dtype, size_t rows, size_t cols,
                             const falcom_dropout_args *drop, void *stream) {
    static const char *who = "falcom_dropout";
    if (!drop || !known_type(dtype)) return invalid(who, "no arguments, or an unknown type");
    if (rows > 0 && cols > MX_ELEMENTS / rows) return invalid(who, "too many elements");
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
    L.vectors = (((uintptr_t)x | (uintptr_t)y | (uintptr_t)residual) & 15) == 0 && cols % 8 == 0;
    L.flat = rows == 1 || cols % MX_BLOCK == 0;
    return done(&c, prev, mc_launch_mx_dropout(&L, dtype, sms, stream));
}
