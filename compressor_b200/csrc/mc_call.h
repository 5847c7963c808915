/*
 * mc_call.h -- what entry points that take device pointers and a stream have
 * in common: argument checks, the current device, errors.
 */
#ifndef MC_CALL_H
#define MC_CALL_H

#include <cuda_runtime_api.h>
#include <stdint.h>
#include <stdio.h>

#include "mc_internal.h"

static inline int device_byte(const void *p, int device) {
    struct cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        (void)cudaGetLastError();
        return 0;
    }
    return (at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged) && at.device == device;
}

/* An argument of a run or step: `bytes` of device memory of `device`.  Its
 * last byte is asked about where another allocation could start before it:
 * they start at multiples of 256 bytes. */
static inline int check_argument(const char *who, const char *what, const void *p, size_t bytes, size_t align, int device) {
    const uintptr_t first = (uintptr_t)p, last = first + bytes - 1;
    if (p && (first & (align - 1)) == 0 && device_byte(p, device) &&
        (first / 256 == last / 256 || device_byte((const void *)last, device)))
        return 1;
    fprintf(stderr, "[ERROR] %s: %s is NULL, not %zu-byte aligned or not %zu bytes of device memory of device %d\n",
            who, what, align, bytes, device);
    return 0;
}

/* Makes `device` current; returns the device to restore, or -2 on failure. */
static inline int enter(int device) {
    int prev = -1;
    if (cudaGetDevice(&prev) != cudaSuccess || (prev != device && cudaSetDevice(device) != cudaSuccess)) {
        (void)cudaGetLastError();
        return -2;
    }
    return prev;
}

static inline void leave(int prev, int device) {
    if (prev >= 0 && prev != device) cudaSetDevice(prev);
}

/* An error that the caller's earlier work left stays the caller's. */
static inline int error_pending(const char *who) {
    const cudaError_t e = cudaPeekAtLastError();
    if (e == cudaSuccess) return 0;
    fprintf(stderr, "[ERROR] %s: a CUDA error is already pending (%s); nothing launched\n", who,
            cudaGetErrorString(e));
    return 1;
}

static inline int launch_failed(const char *who, int e) {
    fprintf(stderr, "[ERROR] %s: launch failed: %s\n", who, cudaGetErrorString((cudaError_t)e));
    return ERROR_COMPRESSION;
}

#endif
