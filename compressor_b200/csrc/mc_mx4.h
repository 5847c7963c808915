/*
 * mc_mx4.h -- what the host side (mc_mx4.c) hands to the kernels of the 4-bit
 * operators and of dropout (mc_mx4.cu, mc_mx4_product.cu).
 */
#ifndef MC_MX4_H
#define MC_MX4_H

#include <cuda_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "falcom_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MX_BLOCK FALCOM_MX4_BLOCK   /* elements of a scale */
#define MX_PANEL 256                /* columns of a matrix whose codes lie together: 128 bytes a row */
#define MX_GROUP 128                /* rows whose scales lie together */
#define MX_TYPES 3

/* Random bits of one purpose. */
typedef struct {
    uint32_t key;              /* hash of purpose and seed */
    int32_t on;
    const int64_t *counter;    /* device memory; NULL counts as 0, and then */
    uint32_t a, b;             /* the key's two words */
} mx_random;

typedef struct {
    mx_random random;
    uint32_t threshold;        /* an element is dropped when its 16 bits are below */
    float factor;              /* of the others */
} mx_drop;

typedef struct {
    uint8_t *codes;            /* [panels][rows up to 8][128], 16-byte pieces exchanged within a row */
    uint8_t *scales;           /* [panels][groups][2][32][4][4] */
    int64_t rows, cols;
} mx_matrix;

typedef struct {
    const void *x;
    int64_t n;
    float *base;               /* or NULL */
    uint8_t *codes, *scales;
    mx_random random;
    int32_t vectors;           /* x and base on 16-byte boundaries */
    int32_t unit;              /* codes are filled up to a multiple of so many bytes: 1, or 16 where scales follow */
} mx_encode_launch;

typedef struct {
    const uint8_t *codes, *scales;
    int64_t n;
    void *out;
    float weight;
    int32_t accumulate;
    int32_t vectors;           /* out on a 16-byte boundary */
} mx_decode_launch;

typedef struct {
    const void *x;
    int64_t rows, cols, ld;
    mx_matrix along_rows, along_cols;   /* codes NULL: not wanted */
    mx_random random;
    mx_drop drop;
    int32_t vectors;           /* every row starts on a 16-byte boundary */
    uint32_t tiles;            /* of 128 columns */
} mx_quantize_launch;

typedef struct {
    mx_matrix m;
    void *out;
    int64_t ld;
} mx_dequantize_launch;

/* Few enough rows and columns to be rounded inside the product, by every CTA
 * for itself, which saves a launch.  Rounding inside and before, in a graph,
 * bf16: 1 x 1024 times 4096 rows of weights 3.3 and 5.4 us, 1 x 4096 5.2 and
 * 7.7, 8 x 4096 7.6 and 7.9, 16 x 2048 6.8 and 6.8: at 32768 elements they
 * meet.  (4096 columns: 48 KB of rounded rows in a CTA of its own.)  The sizes
 * of x alone decide, as they do about the workspace; with many more rows of
 * weights the CTAs round over and over, and 8 x 4096 times 20000 takes 22 us
 * instead of 12, 16 x 1024 times 50257 12.5 instead of 9.9. */
#define MX_ROUND_ROWS 16
#define MX_ROUND_COLS 4096
#define MX_ROUND_ELEMENTS 32768

typedef struct {
    mx_matrix a, b;
    void *out;                 /* [a.rows][ld] */
    int64_t ld;
    mx_drop drop;
    const void *x;             /* not NULL: a as it is before rounding (then without codes and scales) */
    int64_t ld_x;
    int32_t x_type;
    int32_t vectors;           /* every row of x starts on a 16-byte boundary */
} mx_product_launch;

typedef struct {
    const void *x, *residual;
    void *y;
    int64_t rows, cols;
    mx_drop drop;
    int32_t vectors;           /* rows are whole 16-byte vectors of aligned memory */
    int32_t flat;              /* an element's place is its index: rows are whole blocks, or one */
} mx_dropout_launch;

/* All return a CUDA error code (0: queued). */
int mc_launch_mx_encode(const mx_encode_launch *L, int type, void *stream);
int mc_launch_mx_decode(const mx_decode_launch *L, int type, void *stream);
int mc_launch_mx_quantize(const mx_quantize_launch *L, int type, void *stream);
int mc_launch_mx_dequantize(const mx_dequantize_launch *L, int type, int sms, void *stream);
int mc_launch_mx_product(const mx_product_launch *L, int type, int sms, void *stream);
int mc_launch_mx_dropout(const mx_dropout_launch *L, int type, int sms, void *stream);
int mc_mx_errors(uint32_t *word);
uint32_t mc_mx_hash(uint32_t x);
void mc_mx_key(mx_random *r);   /* a and b of key and counter 0 */

#ifdef __cplusplus
}
#endif

#endif
