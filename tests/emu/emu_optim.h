// emu_optim.h -- what mc_optim.cu and mc_optim.c use beyond emu.h and
// fake_cudart.cpp (test infrastructure only).
#pragma once

extern "C" inline __attribute__((used)) cudaError_t cudaDeviceGetAttribute(int *v, cudaDeviceAttr, int) {
    *v = 2;   // two SMs: grids that stride over their units even in small cases
    return cudaSuccess;
}

extern "C" inline __attribute__((used)) cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode *) {
    return cudaSuccess;
}

// Stream capture: between the two calls of emu_optim_capture every stream is
// being captured into one graph (kernels run all the same), which lives until
// emu_optim_graph_gone.
#include <utility>
#include <vector>
inline bool emu_capturing = false;
inline std::vector<std::pair<cudaHostFn_t, void *>> emu_objects;
extern "C" __attribute__((used, visibility("default"))) inline void emu_optim_capture(int on) { emu_capturing = on != 0; }
extern "C" __attribute__((used, visibility("default"))) inline void emu_optim_graph_gone() {
    for (auto &o : emu_objects) o.first(o.second);
    emu_objects.clear();
}
extern "C" inline __attribute__((used)) cudaError_t cudaStreamGetCaptureInfo(cudaStream_t, cudaStreamCaptureStatus *st,
                                                                             unsigned long long *, cudaGraph_t *g,
                                                                             const cudaGraphNode_t **, size_t *) {
    *st = emu_capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
    if (g) *g = (cudaGraph_t)&emu_capturing;
    return cudaSuccess;
}
extern "C" inline __attribute__((used)) cudaError_t cudaUserObjectCreate(cudaUserObject_t *o, void *p, cudaHostFn_t f,
                                                                         unsigned, unsigned) {
    emu_objects.emplace_back(f, p);
    *o = (cudaUserObject_t)&emu_objects;
    return cudaSuccess;
}
extern "C" inline __attribute__((used)) cudaError_t cudaGraphRetainUserObject(cudaGraph_t, cudaUserObject_t, unsigned,
                                                                              unsigned) {
    return cudaSuccess;
}
extern "C" inline __attribute__((used)) cudaError_t cudaUserObjectRelease(cudaUserObject_t, unsigned) {
    return cudaSuccess;
}
inline float emu_e4m3(unsigned code) {
    const int e = code >> 3 & 15, f = code & 7;
    float v = e ? ldexpf(1.0f + f / 8.0f, e - 7) : ldexpf(f / 8.0f, -6);
    if ((code & 0x7F) == 0x7F) v = NAN;
    return code & 0x80 ? -v : v;
}
inline unsigned __byte_perm(unsigned a, unsigned b, unsigned sel) {
    const unsigned long long ab = (unsigned long long)b << 32 | a;
    unsigned r = 0;
    for (int i = 0; i < 4; i++) r |= (unsigned)(ab >> 8 * (sel >> 4 * i & 7) & 0xFF) << 8 * i;
    return r;
}

template <class T>
inline T __shfl_sync(unsigned, T v, int src) {   // emu_shfl knows lane ^ arg: from src's own side
    return emu_shfl(v, false, (int)(threadIdx.x & 31) ^ src);
}
inline int __all_sync(unsigned, int p) { return __ballot_sync(0xffffffffu, p) == 0xffffffffu; }

// Test hook: so many lanes find that their wait has run out, whatever the
// barrier says.
inline std::atomic<int> emu_late_waits{0};
extern "C" __attribute__((used, visibility("default"))) inline void emu_optim_late_waits(int n) { emu_late_waits = n; }
inline bool emu_wait_is_late() {
    int n = emu_late_waits;
    while (n > 0 && !emu_late_waits.compare_exchange_weak(n, n - 1)) {
    }
    return n > 0;
}

// An mbarrier: arrivals expected, arrivals missing in this phase, phase.
inline void emu_mbar_init(uint32_t bar, uint64_t count) {
    __atomic_store_n((uint64_t *)emu_smem_ptr(bar), count << 40 | count << 8, __ATOMIC_SEQ_CST);
}
inline void emu_mbar_arrive(uint32_t bar) {
    uint64_t *p = (uint64_t *)emu_smem_ptr(bar), old = __atomic_load_n(p, __ATOMIC_SEQ_CST), now;
    do {
        const uint64_t count = old >> 40, missing = (old >> 8 & 0xFFFFFFFF) - 1;
        now = missing ? count << 40 | missing << 8 | (old & 1) : count << 40 | count << 8 | ((old & 1) ^ 1);
    } while (!__atomic_compare_exchange_n(p, &old, now, false, __ATOMIC_SEQ_CST, __ATOMIC_SEQ_CST));
}
inline bool emu_mbar_done(uint32_t bar, uint32_t parity) {
    return (__atomic_load_n((uint64_t *)emu_smem_ptr(bar), __ATOMIC_SEQ_CST) & 1) != parity;
}
