/*
 * mc_optim.c -- host side of the optimiser entry points (falcom_norm_*,
 * falcom_adamw_*): argument checks, the plans' device tables, launches.  The
 * kernels are in mc_optim.cu.
 */
#include <cuda_runtime_api.h>
#include <float.h>
#include <math.h>
#include <pthread.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "mc_call.h"
#include "mc_internal.h"
#include "mc_optim.h"

static const size_t g_type_size[OP_NTYPES] = {4, 2, 2};

/* What both kinds of plans start with. */
typedef struct op_plan {
    uint8_t *table;          /* device memory */
    int device;
    int graphs;              /* captured calls whose graphs still exist (atomic) */
    struct op_plan *next;    /* in the list of destroyed plans that graphs still use */
} op_plan;

struct falcom_norm {
    op_plan base;     /* table: op_norm_tensor[n], then op_unit[n_units] */
    int grid;
    int64_t n_units;
    size_t units_at;
};

struct falcom_adamw {
    op_plan base;     /* table: ticket, error word, op_adamw_tensor[n], op_unit[] of every type pair */
    int bits;
    int64_t *step;
    size_t tensors_at, units_at;
    int64_t n_units[OP_NTYPES * OP_NTYPES];   /* by param_type * OP_NTYPES + grad_type */
    int grid[OP_NTYPES * OP_NTYPES];
    int last;         /* type pair of the launch that counts the step */
};

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

/* [p, p + bytes) is device memory of one device, the plan's (*device, -1
 * before the first range); misalignment and NULL are refused too. */
static int check_range(mc_ptrcache *pc, const char *who, const char *what, size_t i, const void *p, size_t bytes,
                       size_t align, int *device) {
    if (!p || ((uintptr_t)p & (align - 1)) != 0) {
        fprintf(stderr, "[ERROR] %s: %s of tensor %zu is NULL or not %zu-byte aligned\n", who, what, i, align);
        return 0;
    }
    for (int end = 0; end < 2; end++) {
        int dev = -1;
        if (!mc_classify(pc, end ? (const void *)((const uint8_t *)p + bytes - 1) : p, &dev)) {
            fprintf(stderr, "[ERROR] %s: %s of tensor %zu is not device memory\n", who, what, i);
            return 0;
        }
        if (*device < 0) *device = dev;
        if (dev != *device) {
            fprintf(stderr, "[ERROR] %s: %s of tensor %zu is on device %d, others on device %d\n", who, what, i, dev,
                    *device);
            return 0;
        }
    }
    return 1;
}

/* Device copy of a host table, on `device`; NULL when there is no room or
 * no usable device. */
static uint8_t *upload(const char *who, int device, const uint8_t *host, size_t bytes, int *sms) {
    const int prev = enter(device);
    uint8_t *d = NULL;
    if (prev == -2 || cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
        cudaMalloc((void **)&d, bytes) != cudaSuccess) {
        (void)cudaGetLastError();
        fprintf(stderr, "[ERROR] %s: no device memory for %zu bytes of tables on device %d\n", who, bytes, device);
        if (prev != -2) leave(prev, device);
        return NULL;
    }
    /* the copy is complete when the call returns, for every stream */
    if (cudaMemcpy(d, host, bytes, cudaMemcpyHostToDevice) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess) {
        fprintf(stderr, "[ERROR] %s: table upload failed: %s\n", who, cudaGetErrorString(cudaGetLastError()));
        cudaFree(d);
        d = NULL;
    }
    leave(prev, device);
    return d;
}

/* A collector may drop a plan while some stream is being captured: in the
 * relaxed mode freeing does not end the capture. */
static void release(op_plan *plan) {
    const int prev = enter(plan->device);
    if (prev != -2) {
        enum cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        const int relaxed = cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
        cudaFree(plan->table);   /* waits for the device's work first */
        if (relaxed) cudaThreadExchangeStreamCaptureMode(&mode);
        leave(prev, plan->device);
    }
    free(plan);
}

/* A captured call's graph reads the plan's table whenever it runs, so a plan
 * is freed after the graphs that captured it.  The graph (and whatever is
 * instantiated or cloned from it) holds an object whose end drops the count;
 * that happens on a thread of the driver's, where nothing can be freed. */
static int graphs_of(const op_plan *plan) { return __atomic_load_n(&plan->graphs, __ATOMIC_ACQUIRE); }

static void graph_gone(void *plan) { __atomic_fetch_sub(&((op_plan *)plan)->graphs, 1, __ATOMIC_RELEASE); }

static int hold_for_graph(op_plan *plan, cudaStream_t stream) {
    enum cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    cudaGraph_t graph = NULL;
    cudaError_t e = cudaStreamGetCaptureInfo(stream, &status, NULL, &graph, NULL, NULL);
    if (e == cudaSuccess && status != cudaStreamCaptureStatusActive) return cudaSuccess;
    cudaUserObject_t object = NULL;
    __atomic_fetch_add(&plan->graphs, 1, __ATOMIC_RELAXED);
    if (e == cudaSuccess) e = cudaUserObjectCreate(&object, plan, graph_gone, 1, cudaUserObjectNoDestructorSync);
    if (e != cudaSuccess) graph_gone(plan);
    else if ((e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove)) != cudaSuccess)
        cudaUserObjectRelease(object, 1);   /* and so graph_gone */
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e;
}

static op_plan *g_left;   /* destroyed, used by graphs */
static pthread_mutex_t g_left_mu = PTHREAD_MUTEX_INITIALIZER;

/* Frees the destroyed plans that no graph uses any longer, and `plan` when
 * none does (NULL: nothing new). */
static void retire(op_plan *plan) {
    op_plan *free_now = NULL;
    pthread_mutex_lock(&g_left_mu);
    if (plan) {
        plan->next = g_left;
        g_left = plan;
    }
    for (op_plan **at = &g_left; *at;) {
        op_plan *p = *at;
        if (graphs_of(p) > 0) {
            at = &p->next;
            continue;
        }
        *at = p->next;
        p->next = free_now;
        free_now = p;
    }
    pthread_mutex_unlock(&g_left_mu);
    while (free_now) {
        op_plan *p = free_now;
        free_now = p->next;
        release(p);
    }
}

static int current_device(const char *who) {
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) {
        (void)cudaGetLastError();
        fprintf(stderr, "[ERROR] %s: no usable CUDA device\n", who);
        return -1;
    }
    return dev;
}

/* ------------------------------------------------------------------- norm */

/* Units of a tensor: whole ones from its first 16-byte boundary on, the
 * elements before that (*head) go with the first. */
static int64_t norm_units(const void *x, size_t n, size_t size, int32_t *head) {
    const size_t unit = OP_NORM_BYTES / size;
    size_t h = ((16 - ((uintptr_t)x & 15)) & 15) / size;
    if (h > n) h = n;
    if (head) *head = (int32_t)h;
    const size_t k = (n - h + unit - 1) / unit;
    return (int64_t)(k ? k : n > 0);
}

MC_EXPORT falcom_norm *falcom_norm_create(const void *const *tensors, const size_t *numels, const int *dtypes,
                                          size_t n) {
    static const char *who = "falcom_norm_create";
    if (n > UINT32_MAX || (n > 0 && (!tensors || !numels || !dtypes))) {
        fprintf(stderr, "[ERROR] %s: invalid arguments\n", who);
        return NULL;
    }
    retire(NULL);
    int device = -1;
    int64_t n_units = 0;
    mc_ptrcache pc;
    pc.n = 0;
    for (size_t i = 0; i < n; i++) {
        if (dtypes[i] < 0 || dtypes[i] >= OP_NTYPES) {
            fprintf(stderr, "[ERROR] %s: tensor %zu has unknown type %d\n", who, i, dtypes[i]);
            return NULL;
        }
        if (numels[i] > (size_t)1 << 42) {
            fprintf(stderr, "[ERROR] %s: tensor %zu has %zu elements\n", who, i, numels[i]);
            return NULL;
        }
        const size_t sz = g_type_size[dtypes[i]];
        if (numels[i] && !check_range(&pc, who, "address", i, tensors[i], numels[i] * sz, sz, &device)) return NULL;
        n_units += norm_units(tensors[i], numels[i], sz, NULL);
    }
    if (n_units > (int64_t)UINT32_MAX / 2) {
        fprintf(stderr, "[ERROR] %s: too many elements\n", who);
        return NULL;
    }
    if (device < 0 && (device = current_device(who)) < 0) return NULL;
    falcom_norm *plan = (falcom_norm *)calloc(1, sizeof(*plan));
    const size_t units_at = align256(n * sizeof(op_norm_tensor));
    const size_t bytes = align256(units_at + (size_t)n_units * sizeof(op_unit)) + 256;
    uint8_t *host = plan ? (uint8_t *)calloc(1, bytes) : NULL;
    if (!host) {
        fprintf(stderr, "[ERROR] %s: out of memory\n", who);
        free(plan);
        return NULL;
    }
    op_norm_tensor *t = (op_norm_tensor *)host;
    op_unit *u = (op_unit *)(host + units_at);
    for (size_t i = 0; i < n; i++) {
        t[i].x = tensors[i];
        t[i].n = (int64_t)numels[i];
        t[i].dtype = dtypes[i];
        const size_t sz = g_type_size[dtypes[i]];
        t[i].unit = (int32_t)(OP_NORM_BYTES / sz);
        const int64_t k = norm_units(tensors[i], numels[i], sz, &t[i].head);
        for (int64_t j = 0; j < k; j++) {
            u->tensor = (uint32_t)i;
            u->index = (uint32_t)j;
            u++;
        }
    }
    int sms = 0;
    plan->base.device = device;
    plan->n_units = n_units;
    plan->units_at = units_at;
    plan->base.table = upload(who, device, host, bytes, &sms);
    free(host);
    if (!plan->base.table) {
        free(plan);
        return NULL;
    }
    plan->grid = mc_op_norm_grid(n_units, sms);
    return plan;
}

MC_EXPORT size_t falcom_norm_work_bytes(const falcom_norm *plan) {
    return plan ? 16 + (size_t)plan->grid * sizeof(double) : 0;
}

MC_EXPORT int falcom_norm_run(falcom_norm *plan, double scale, double max_norm, float *out, void *work,
                              void *stream) {
    static const char *who = "falcom_norm_run";
    if (!plan || !out || !work || !isfinite(scale) || !(max_norm > 0.0)) {
        fprintf(stderr, "[ERROR] %s: invalid arguments\n", who);
        return ERROR_INVALID_PARAM;
    }
    if (!check_argument(who, "out", out, 2 * sizeof(float), 4, plan->base.device) ||
        !check_argument(who, "work", work, falcom_norm_work_bytes(plan), 8, plan->base.device))
        return ERROR_INVALID_PARAM;
    if (error_pending(who)) return ERROR_COMPRESSION;
    const int prev = enter(plan->base.device);
    if (prev == -2) return ERROR_COMPRESSION;
    int e = hold_for_graph(&plan->base, (cudaStream_t)stream);
    op_norm_launch L;
    memset(&L, 0, sizeof(L));
    L.tensors = (const op_norm_tensor *)plan->base.table;
    L.units = (const op_unit *)(plan->base.table + plan->units_at);
    L.n_units = plan->n_units;
    L.scale = scale;
    L.max_norm = max_norm;
    L.out = out;
    L.ticket = (uint32_t *)work;
    L.partial = (double *)((uint8_t *)work + 16);
    if (e == 0) e = mc_launch_norm(&L, plan->grid, stream);
    leave(prev, plan->base.device);
    return e == 0 ? ERROR_NONE : launch_failed(who, e);
}

MC_EXPORT int falcom_norm_graphs(const falcom_norm *plan) { return plan ? graphs_of(&plan->base) : 0; }

MC_EXPORT void falcom_norm_destroy(falcom_norm *plan) {
    if (plan) retire(&plan->base);
}

/* ------------------------------------------------------------------ AdamW */
typedef struct {
    uintptr_t lo, hi;
    int written;
} span;

static int span_cmp(const void *a, const void *b) {
    const span *x = (const span *)a, *y = (const span *)b;
    return x->lo < y->lo ? -1 : x->lo > y->lo;
}

/* No written array shares a byte with any other array. */
static int spans_disjoint(span *s, size_t n) {
    qsort(s, n, sizeof(*s), span_cmp);
    uintptr_t any = 0, written = 0;
    for (size_t i = 0; i < n; i++) {
        if (s[i].lo < (s[i].written ? any : written)) return 0;
        if (s[i].hi > any) any = s[i].hi;
        if (s[i].written && s[i].hi > written) written = s[i].hi;
    }
    return 1;
}

static void add_span(span *s, size_t *k, const void *p, size_t bytes, int written) {
    s[*k].lo = (uintptr_t)p;
    s[*k].hi = (uintptr_t)p + bytes;
    s[*k].written = written;
    (*k)++;
}

static int check_tensors(const char *who, const falcom_adamw_tensor *t, size_t n, int bits, int64_t *step,
                         int *device, span *spans) {
    size_t k = 0;
    mc_ptrcache pc;
    pc.n = 0;
    for (size_t i = 0; i < n; i++) {
        if (t[i].param_type < 0 || t[i].param_type >= OP_NTYPES || t[i].grad_type < 0 || t[i].grad_type >= OP_NTYPES) {
            fprintf(stderr, "[ERROR] %s: tensor %zu has an unknown type\n", who, i);
            return 0;
        }
        if (!(t[i].weight_decay >= 0.0) || !isfinite(t[i].weight_decay) || t[i].n > (size_t)1 << 39) {
            fprintf(stderr, "[ERROR] %s: weight decay or length of tensor %zu is out of range\n", who, i);
            return 0;
        }
        if (t[i].n == 0) continue;
        const size_t ps = g_type_size[t[i].param_type], gs = g_type_size[t[i].grad_type];
        const size_t ss = bits == 32 ? 4 : 1, blocks = (t[i].n + OP_BLOCK - 1) / OP_BLOCK;
        if (!check_range(&pc, who, "param", i, t[i].param, t[i].n * ps, ps, device) ||
            !check_range(&pc, who, "grad", i, t[i].grad, t[i].n * gs, gs, device) ||
            !check_range(&pc, who, "m", i, t[i].m, t[i].n * ss, ss, device) ||
            !check_range(&pc, who, "v", i, t[i].v, t[i].n * ss, ss, device))
            return 0;
        if (bits == 8 && (!check_range(&pc, who, "m_scale", i, t[i].m_scale, 4 * blocks, 4, device) ||
                          !check_range(&pc, who, "v_scale", i, t[i].v_scale, 4 * blocks, 4, device)))
            return 0;
        add_span(spans, &k, t[i].param, t[i].n * ps, 1);
        add_span(spans, &k, t[i].grad, t[i].n * gs, 0);
        add_span(spans, &k, t[i].m, t[i].n * ss, 1);
        add_span(spans, &k, t[i].v, t[i].n * ss, 1);
        if (bits == 8) {
            add_span(spans, &k, t[i].m_scale, 4 * blocks, 1);
            add_span(spans, &k, t[i].v_scale, 4 * blocks, 1);
        }
    }
    if (!check_range(&pc, who, "step", n, step, sizeof(*step), 8, device)) return 0;
    add_span(spans, &k, step, sizeof(*step), 1);
    if (!spans_disjoint(spans, k)) {
        fprintf(stderr, "[ERROR] %s: an array that is written overlaps another array\n", who);
        return 0;
    }
    return 1;
}

static int64_t adamw_units(const falcom_adamw_tensor *t, int bits) {
    const size_t unit = (size_t)OP_ADAMW_UNIT * (bits == 32 ? 1 : OP_ADAMW8_ROUNDS(g_type_size[t->param_type],
                                                                                   g_type_size[t->grad_type]));
    return (int64_t)((t->n + unit - 1) / unit);
}

MC_EXPORT falcom_adamw *falcom_adamw_create(const falcom_adamw_tensor *tensors, size_t n, int state_bits,
                                            int64_t *step) {
    static const char *who = "falcom_adamw_create";
    if (n > UINT32_MAX || (n > 0 && !tensors) || (state_bits != 32 && state_bits != 8)) {
        fprintf(stderr, "[ERROR] %s: invalid arguments (state_bits must be 32 or 8)\n", who);
        return NULL;
    }
    retire(NULL);
    int device = -1;
    span *spans = (span *)malloc((6 * n + 1) * sizeof(*spans));
    if (!spans) {
        fprintf(stderr, "[ERROR] %s: out of memory\n", who);
        return NULL;
    }
    int ok = check_tensors(who, tensors, n, state_bits, step, &device, spans);
    free(spans);
    if (!ok) return NULL;

    int64_t counts[OP_NTYPES * OP_NTYPES] = {0}, total = 0;
    for (size_t i = 0; i < n; i++) {
        const int64_t k = adamw_units(&tensors[i], state_bits);
        counts[tensors[i].param_type * OP_NTYPES + tensors[i].grad_type] += k;
        total += k;
    }
    if (total > (int64_t)UINT32_MAX / 2) {
        fprintf(stderr, "[ERROR] %s: too many elements\n", who);
        return NULL;
    }
    falcom_adamw *plan = (falcom_adamw *)calloc(1, sizeof(*plan));
    const size_t tensors_at = 256;
    const size_t units_at = align256(tensors_at + n * sizeof(op_adamw_tensor));
    const size_t bytes = align256(units_at + (size_t)total * sizeof(op_unit)) + 256;
    uint8_t *host = plan ? (uint8_t *)calloc(1, bytes) : NULL;
    if (!host) {
        fprintf(stderr, "[ERROR] %s: out of memory\n", who);
        free(plan);
        return NULL;
    }
    op_adamw_tensor *t = (op_adamw_tensor *)(host + tensors_at);
    op_unit *fill[OP_NTYPES * OP_NTYPES], *u = (op_unit *)(host + units_at);
    for (int c = 0; c < OP_NTYPES * OP_NTYPES; c++) {
        fill[c] = u;
        u += counts[c];
    }
    int64_t blocks = 0;
    for (size_t i = 0; i < n; i++) {
        const falcom_adamw_tensor *a = &tensors[i];
        t[i].p = a->param;
        t[i].g = a->grad;
        t[i].m = a->m;
        t[i].v = a->v;
        t[i].ms = a->m_scale;
        t[i].vs = a->v_scale;
        t[i].n = (int64_t)a->n;
        t[i].first_block = blocks;
        t[i].weight_decay = a->weight_decay;
        if ((((uintptr_t)a->m | (uintptr_t)a->v) & 15) != 0) t[i].how = OP_RAGGED;
        else if (((uintptr_t)a->param & (4 * g_type_size[a->param_type] - 1)) != 0 ||
                 ((uintptr_t)a->grad & (4 * g_type_size[a->grad_type] - 1)) != 0) t[i].how = OP_STATES;
        else t[i].how = OP_ALIGNED;
        blocks += (int64_t)((a->n + OP_BLOCK - 1) / OP_BLOCK);
        const int c = a->param_type * OP_NTYPES + a->grad_type;
        const int64_t k = adamw_units(a, state_bits);
        for (int64_t j = 0; j < k; j++) {
            fill[c]->tensor = (uint32_t)i;
            fill[c]->index = (uint32_t)j;
            fill[c]++;
        }
    }
    int sms = 0;
    plan->base.device = device;
    plan->bits = state_bits;
    plan->step = step;
    plan->tensors_at = tensors_at;
    plan->units_at = units_at;
    plan->base.table = upload(who, device, host, bytes, &sms);
    free(host);
    if (!plan->base.table) {
        free(plan);
        return NULL;
    }
    for (int c = 0; c < OP_NTYPES * OP_NTYPES; c++) {
        plan->n_units[c] = counts[c];
        if (counts[c]) plan->last = c;
        plan->grid[c] = mc_op_adamw_grid(counts[c], sms, state_bits, c / OP_NTYPES, c % OP_NTYPES);
    }
    return plan;
}

MC_EXPORT int falcom_adamw_step(falcom_adamw *plan, const falcom_adamw_args *a, void *stream) {
    static const char *who = "falcom_adamw_step";
    if (!plan || !a || !(a->lr >= 0.0) || !isfinite(a->lr) || !(a->beta1 >= 0.0 && a->beta1 < 1.0) ||
        !(a->beta2 >= 0.0 && a->beta2 < 1.0) || !((float)a->eps >= FLT_MIN) || !isfinite((float)a->eps) ||
        !isfinite((float)a->grad_scale)) {
        fprintf(stderr, "[ERROR] %s: invalid arguments\n", who);
        return ERROR_INVALID_PARAM;
    }
    if ((a->clip && !check_argument(who, "clip", a->clip, 2 * sizeof(float), 4, plan->base.device)) ||
        (a->lr_device && !check_argument(who, "lr_device", a->lr_device, sizeof(float), 4, plan->base.device)))
        return ERROR_INVALID_PARAM;
    if (error_pending(who)) return ERROR_COMPRESSION;
    const int prev = enter(plan->base.device);
    if (prev == -2) return ERROR_COMPRESSION;
    int e = hold_for_graph(&plan->base, (cudaStream_t)stream);
    op_adamw_launch L;
    memset(&L, 0, sizeof(L));
    L.tensors = (const op_adamw_tensor *)(plan->base.table + plan->tensors_at);
    L.units = (const op_unit *)(plan->base.table + plan->units_at);
    L.step = plan->step;
    L.clip = a->clip;
    L.lr_dev = a->lr_device;
    L.ticket = (uint32_t *)plan->base.table;
    L.lr = a->lr;
    L.beta1 = a->beta1;
    L.beta2 = a->beta2;
    L.b1.x = L.b1.y = (float)a->beta1;
    L.b2.x = L.b2.y = (float)a->beta2;
    L.b1c.x = L.b1c.y = (float)(1.0 - a->beta1);
    L.one.x = L.one.y = 1.0f;
    L.minus_b2.x = L.minus_b2.y = -L.b2.x;
    L.minus_b2c.x = L.minus_b2c.y = -(float)(1.0 - a->beta2);
    L.eps.x = L.eps.y = (float)a->eps;
    L.scale = (float)a->grad_scale;
    L.seed_key = mc_op_hash(mc_op_hash((uint32_t)a->seed ^ 0x9E3779B9u) ^ (uint32_t)(a->seed >> 32));
    for (int c = 0; c < OP_NTYPES * OP_NTYPES && e == 0; c++) {
        /* a plan without elements still counts its steps */
        if (plan->n_units[c] > 0 || c == plan->last) {
            L.n_units = plan->n_units[c];
            L.advance = c == plan->last;
            e = mc_launch_adamw(&L, plan->bits, c / OP_NTYPES, c % OP_NTYPES, plan->grid[c], stream);
        }
        L.units += plan->n_units[c];
    }
    leave(prev, plan->base.device);
    return e == 0 ? ERROR_NONE : launch_failed(who, e);
}

MC_EXPORT int falcom_adamw_errors(falcom_adamw *plan) {
    if (!plan) return ERROR_INVALID_PARAM;
    const int prev = enter(plan->base.device);
    if (prev == -2) return ERROR_COMPRESSION;
    uint32_t word = 0;
    /* steps may be in flight on streams that the copy does not wait for */
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(&word, plan->base.table + 4, 4, cudaMemcpyDeviceToHost);
    leave(prev, plan->base.device);
    if (e != cudaSuccess) return ERROR_COMPRESSION;
    return word != 0;
}

MC_EXPORT int falcom_adamw_graphs(const falcom_adamw *plan) { return plan ? graphs_of(&plan->base) : 0; }

MC_EXPORT void falcom_adamw_destroy(falcom_adamw *plan) {
    if (plan) retire(&plan->base);
}
