/*
 * mc_optim.h -- tables shared by the host side (mc_optim.c) and the kernels
 * (mc_optim.cu) of the optimiser entry points.
 */
#ifndef MC_OPTIM_H
#define MC_OPTIM_H

#include <cuda_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "falcom_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define OP_TPB 256
#define OP_WARPS (OP_TPB / 32)
#define OP_BLOCK FALCOM_ADAMW_BLOCK   /* elements a warp holds in registers at once (8 per lane) */
#define OP_NTYPES 3

/* Which arrays of a tensor are aligned (16 bytes; with 32-bit states 4
 * elements): not its states, its states only, or all. */
enum { OP_RAGGED = 0, OP_STATES = 1, OP_ALIGNED = 2 };

/* A unit is a run of elements of one tensor, one CTA's work at a time. */
typedef struct {
    uint32_t tensor;   /* index into the plan's tensors */
    uint32_t index;    /* unit number inside the tensor */
} op_unit;

typedef struct {
    const void *x;
    int64_t n;
    int32_t dtype;
    int32_t head;      /* elements before the first 16-byte boundary (all of a short tensor) */
    int32_t unit;      /* elements of a unit */
    int32_t pad;
} op_norm_tensor;

typedef struct {
    void *p;
    const void *g;
    void *m, *v;
    float *ms, *vs;        /* 8-bit states: one scale per OP_BLOCK elements */
    int64_t n;
    int64_t first_block;   /* OP_BLOCKs of the plan's earlier tensors: the dither's position */
    double weight_decay;
    int32_t how;           /* OP_RAGGED, OP_STATES or OP_ALIGNED */
    int32_t pad;
} op_adamw_tensor;

typedef struct {
    const op_norm_tensor *tensors;
    const op_unit *units;
    uint32_t n_units;
    double scale, max_norm;
    float *out;
    uint32_t *ticket;      /* 0 between calls */
    double *partial;       /* one per CTA */
} op_norm_launch;

typedef struct {
    const op_adamw_tensor *tensors;
    const op_unit *units;
    uint32_t n_units;
    int64_t *step;
    const float *clip;     /* NULL, or {norm, coefficient} */
    const float *lr_dev;   /* NULL, or the learning rate */
    uint32_t *ticket;      /* 0 between calls */
    double lr, beta1, beta2;
    float2 b1, b1c, b2, eps, minus_b2, minus_b2c, one;   /* twice each, for two-element operations; c: 1 - */
    float scale;
    uint32_t seed_key;     /* hash of the seed */
    int32_t advance;       /* this launch's last CTA counts the step */
} op_adamw_launch;

#define OP_NORM_BYTES 32768   /* of a unit */
#define OP_ADAMW_UNIT (OP_WARPS * OP_BLOCK)
/* With 8-bit states a warp has so many blocks of a unit, by the sizes of
 * parameter and gradient types. */
#define OP_ADAMW8_ROUNDS(psize, gsize) ((psize) + (gsize) > 4 ? 1 : 2)

uint32_t mc_op_hash(uint32_t x);
int mc_op_norm_grid(int64_t n_units, int sms);
int mc_op_adamw_grid(int64_t n_units, int sms, int bits, int ptype, int gtype);
/* Both return a CUDA error code (0: queued). */
int mc_launch_norm(const op_norm_launch *L, int grid, void *stream);
int mc_launch_adamw(const op_adamw_launch *L, int bits, int ptype, int gtype, int grid, void *stream);

#ifdef __cplusplus
}
#endif

#endif
