// emu_product.h -- host emulation of what compressor_b200/csrc/mc_mx4_product.cu
// uses of the hardware (test infrastructure only): clusters of CTAs whose
// threads are host threads, shared memory with mbarriers and bulk copies,
// tensor memory, and block-scaled 4-bit matrix instructions that read the
// descriptors, the swizzle and the scales as they lie.
//
// Copies and matrix instructions happen when they are issued.  Shared and
// tensor memory start out full of NaN, so that what was never written shows in
// a result that uses it.  Waits are bounded in units of emu_second.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cmath>
#include <condition_variable>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <memory>
#include <mutex>
#include <thread>
#include <type_traits>
#include <vector>

inline void emu_fail(const char *what) {
    fprintf(stderr, "emu: %s\n", what);
    abort();
}

struct EmuMeet {   // a barrier of n threads
    std::mutex m;
    std::condition_variable cv;
    int n, count = 0;
    unsigned gen = 0;
    explicit EmuMeet(int n_) : n(n_) {}
    void wait() {
        std::unique_lock<std::mutex> lk(m);
        const unsigned g = gen;
        if (++count == n) {
            count = 0;
            gen++;
            cv.notify_all();
        } else {
            cv.wait(lk, [&] { return gen != g; });
        }
    }
};

enum { EMU_WINDOW = 256 * 1024, EMU_STATIC = 1024, EMU_DYNAMIC = 8208 };
struct EmuCta {
    alignas(1024) uint8_t mem[EMU_WINDOW];
    uint32_t tmem[128][512];
    uint32_t dynamic = 0, columns = 0;   // bytes; allocated columns
    EmuMeet all;
    std::vector<std::unique_ptr<EmuMeet>> warps, named;
    std::vector<uint64_t> slot;
    int copies = 0;
    EmuCta(int threads, size_t bytes) : dynamic((uint32_t)bytes), all(threads), slot(threads) {
        memset(mem, 0xFF, sizeof(mem));
        memset(tmem, 0xFF, sizeof(tmem));
        for (int i = 0; i < threads / 32; i++) warps.emplace_back(new EmuMeet(32));
        for (int i = 0; i < 16; i++) named.emplace_back(new EmuMeet(64));
    }
};
struct EmuCluster {
    std::mutex m;
    std::condition_variable cv;
    std::vector<std::unique_ptr<EmuCta>> cta;
    EmuMeet all;
    EmuCluster(int ctas, int threads, size_t bytes) : all(ctas * threads) {
        for (int i = 0; i < ctas; i++) cta.emplace_back(new EmuCta(threads, bytes));
    }
};
struct EmuUint3 {
    unsigned x, y, z;
};
inline thread_local EmuUint3 threadIdx, blockIdx, gridDim;
inline thread_local EmuCluster *emu_cluster;
inline thread_local EmuCta *emu_cta;
inline thread_local int emu_rank;

// Test hooks: how long a second is; from which of its copies on a CTA of that
// rank loses them (-1: none).
inline std::atomic<double> emu_second{100.0};
inline std::atomic<int> emu_lost_rank{-1}, emu_lost_from{0};

template <class F>
inline void emu_launch(int64_t grid, int threads, size_t bytes, int cluster, F f) {
    if (bytes > 227 * 1024 || grid % cluster || threads % 32) emu_fail("a launch that the hardware refuses");
    for (int64_t first = 0; first < grid; first += cluster) {
        EmuCluster c(cluster, threads, bytes);
        std::vector<std::thread> pool;
        for (int r = 0; r < cluster; r++)
            for (int t = 0; t < threads; t++)
                pool.emplace_back([&, r, t] {
                    threadIdx = {(unsigned)t, 0, 0};
                    blockIdx = {(unsigned)(first + r), 0, 0};
                    gridDim = {(unsigned)grid, 1, 1};
                    emu_cluster = &c;
                    emu_cta = c.cta[r].get();
                    emu_rank = r;
                    f();
                });
        for (auto &t : pool) t.join();
        for (auto &cta : c.cta)
            if (cta->columns) emu_fail("tensor memory was not freed");
    }
}

// ------------------------------------------------------------- shared memory
inline uint8_t *emu_slot(int i) { return emu_cta->mem + EMU_STATIC + 512 * i; }   // of a __shared__ variable
inline uint8_t *emu_dynamic() { return emu_cta->mem + EMU_DYNAMIC; }
inline uint8_t *emu_at(uint32_t at, uint32_t bytes, int rank = -1) {
    EmuCta *c = rank < 0 ? emu_cta : emu_cluster->cta.at(rank).get();
    const bool fixed = at >= EMU_STATIC && at + bytes <= EMU_DYNAMIC, dynamic = at >= EMU_DYNAMIC && at + bytes <= EMU_DYNAMIC + c->dynamic;
    if (!fixed && !dynamic) emu_fail("an address outside of the CTA's shared memory");
    return c->mem + at;
}
template <class T>
inline T emu_load(uint32_t at, int rank = -1) {
    if (at % sizeof(T)) emu_fail("a misaligned load from shared memory");
    T v;
    memcpy(&v, emu_at(at, sizeof(T), rank), sizeof(T));
    return v;
}
template <class T>
inline void emu_store(uint32_t at, T v, int rank = -1) {
    if (at % sizeof(T)) emu_fail("a misaligned store to shared memory");
    memcpy(emu_at(at, sizeof(T), rank), &v, sizeof(T));
}

inline void __syncthreads() { emu_cta->all.wait(); }
inline void __syncwarp() { emu_cta->warps[threadIdx.x / 32]->wait(); }
template <class T>
inline T emu_exchange(T v, int src) {
    static_assert(sizeof(T) <= 8, "");
    const int w = threadIdx.x / 32;
    uint64_t bits = 0;
    memcpy(&bits, &v, sizeof(T));
    emu_cta->slot[threadIdx.x] = bits;
    emu_cta->warps[w]->wait();
    bits = emu_cta->slot[32 * w + src];
    emu_cta->warps[w]->wait();
    memcpy(&v, &bits, sizeof(T));
    return v;
}
template <class T>
inline T __shfl_sync(unsigned, T v, int src) { return emu_exchange(v, src); }
template <class T>
inline T __shfl_xor_sync(unsigned, T v, int o) { return emu_exchange(v, (int)(threadIdx.x & 31) ^ o); }
inline int __all_sync(unsigned, int p) {
    int all = 1;
    for (int i = 0; i < 32; i++) all &= emu_exchange(p, i) != 0;
    return all;
}

// ------------------------------------------------------------------ mbarriers
struct EmuBar {
    uint16_t count, missing;
    int32_t bytes;
    bool phase() const { return count >> 15; }
};
static_assert(sizeof(EmuBar) == 8, "");
template <class F>
inline void emu_bar(uint32_t bar, int rank, F f) {   // under the cluster's lock; flips the phase where it is complete
    if (bar % 8) emu_fail("a misaligned mbarrier");
    std::lock_guard<std::mutex> lk(emu_cluster->m);
    EmuBar *b = (EmuBar *)emu_at(bar, 8, rank);
    f(*b);
    if (b->missing == 0 && b->bytes == 0) {
        b->count ^= 0x8000;
        b->missing = b->count & 0x7FFF;
        emu_cluster->cv.notify_all();
    }
}
inline void emu_arrive(uint32_t bar, int rank, int expect = 0) {
    emu_bar(bar, rank, [&](EmuBar &b) {
        if (b.missing == 0) emu_fail("one arrival too many");
        b.bytes += expect;
        b.missing--;
    });
}
inline bool emu_done(uint32_t bar, uint32_t parity, double seconds) {
    std::unique_lock<std::mutex> lk(emu_cluster->m);
    const EmuBar *b = (const EmuBar *)emu_at(bar, 8);
    return emu_cluster->cv.wait_for(lk, std::chrono::duration<double>(seconds * emu_second), [&] { return b->phase() != (parity != 0); });
}
inline void emu_bar_init(uint32_t bar, uint32_t count) {
    std::lock_guard<std::mutex> lk(emu_cluster->m);
    EmuBar b = {(uint16_t)count, (uint16_t)count, 0};
    memcpy(emu_at(bar, 8), &b, 8);
}

// --------------------------------------------------------------------- copies
struct EmuRange {
    const uint8_t *lo, *hi;
};
inline std::vector<EmuRange> emu_global;   // what copies may read
inline void emu_copy(uint32_t dst, const uint8_t *src, uint32_t bytes, uint32_t bar, int bar_rank, uint32_t zeros = 0) {
    if (dst % 16 || (uintptr_t)src % 16 || bytes % 16) emu_fail("a copy that is not on 16-byte boundaries");
    bool inside = bytes == 0;
    for (auto &r : emu_global) inside |= src >= r.lo && src + bytes <= r.hi;
    if (!inside) emu_fail("a copy from outside of its matrix");
    uint8_t *to = emu_at(dst, bytes + zeros);
    const int number = __atomic_fetch_add(&emu_cta->copies, 1, __ATOMIC_SEQ_CST);
    if (emu_lost_rank == emu_rank && number >= emu_lost_from) return;
    memcpy(to, src, bytes);
    memset(to + bytes, 0, zeros);
    emu_bar(bar, bar_rank, [&](EmuBar &b) { b.bytes -= (int32_t)(bytes + zeros); });
}
// A tensor map of rows of words: what cuTensorMapEncodeTiled is given here.
struct EmuMap {
    const uint8_t *base;
    uint64_t rows;
    uint32_t words, box;
};
inline CUresult emu_encode_map(CUtensorMap *map, CUtensorMapDataType type, cuuint32_t rank, void *base, const cuuint64_t *size,
                               const cuuint64_t *stride, const cuuint32_t *box, const cuuint32_t *, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
    if (rank != 2 || type != CU_TENSOR_MAP_DATA_TYPE_UINT32 || stride[0] != size[0] * 4 || box[0] != size[0] || box[0] > 256 || box[1] > 256 ||
        (uintptr_t)base % 16)
        return CUDA_ERROR_INVALID_VALUE;
    const EmuMap m = {(const uint8_t *)base, size[1], box[0], box[1]};
    memcpy(map, &m, sizeof(m));
    return CUDA_SUCCESS;
}
inline void emu_copy_box(uint32_t dst, const CUtensorMap *map, int32_t row, uint32_t bar) {   // the first CTA's barrier is told
    EmuMap m;
    memcpy(&m, map, sizeof(m));
    if (row < 0) emu_fail("a box at a negative row");
    const uint64_t left = (uint64_t)row < m.rows ? m.rows - row : 0, rows = left < m.box ? left : m.box;
    emu_copy(dst, m.base + (rows ? (uint64_t)row * m.words * 4 : 0), (uint32_t)rows * m.words * 4, bar, 0, (uint32_t)(m.box - rows) * m.words * 4);
}

// -------------------------------------------------------------- tensor memory
inline void emu_tmem_alloc(uint32_t dst, uint32_t columns) {
    if (threadIdx.x & 31) return;
    if (columns < 32 || columns > 512 || (columns & (columns - 1)) || emu_cta->columns) emu_fail("columns of tensor memory");
    emu_cta->columns = columns;
    emu_store<uint32_t>(dst, 512 - columns);
}
inline void emu_tmem_free(uint32_t at, uint32_t columns) {
    if (threadIdx.x & 31) return;
    if (columns != emu_cta->columns || at != 512 - columns) emu_fail("freeing other columns than were allocated");
    emu_cta->columns = 0;
}
inline uint32_t &emu_cell(EmuCta *c, uint32_t lane, uint32_t column) {
    if (lane >= 128 || column >= 512 || column < 512 - c->columns) emu_fail("an address outside of the allocated columns");
    return c->tmem[lane][column];
}
inline uint32_t emu_desc_at(uint64_t desc) { return (uint32_t)(desc & 0x3FFF) << 4; }
inline uint32_t emu_desc_rows8(uint64_t desc) { return (uint32_t)(desc >> 32 & 0x3FFF) << 4; }   // bytes from 8 rows to the next
// 32 rows of 16 bytes to 4 columns, for each quarter of the lanes; without a swizzle 8 rows are 128 bytes
inline void emu_copy_scales(EmuCta *c, int rank, uint32_t to, uint64_t desc) {
    if (desc >> 61 != 0 || emu_desc_rows8(desc) != 128) emu_fail("a descriptor of scales");
    for (int r = 0; r < 32; r++)
        for (int w = 0; w < 4; w++) {
            const uint32_t v = emu_load<uint32_t>(emu_desc_at(desc) + r / 8 * 128 + r % 8 * 16 + 4 * w, rank);
            for (int q = 0; q < 4; q++) emu_cell(c, 32 * q + r, (to & 0xFFFF) + w) = v;
        }
}
// Byte k of row r of a matrix of 128-byte rows with the 128-byte swizzle.
inline uint8_t emu_code(uint64_t desc, uint32_t r, uint32_t k, int rank) {
    uint32_t at = emu_desc_at(desc) + r / 8 * emu_desc_rows8(desc) + r % 8 * 128 + k;
    at ^= (at >> 7 & 7) << 4;
    return emu_load<uint8_t>(at, rank);
}
inline double emu_scale(EmuCta *c, uint32_t at, uint32_t r, uint32_t byte) {
    const uint32_t s = emu_cell(c, r % 32, (at & 0xFFFF) + r / 32) >> 8 * byte & 255;
    return s == 255 ? NAN : ldexp(1.0, (int)s - 127);
}
// d[m][n] (+)= sum over 64 k of a[m][k] b[n][k], scales of 32 k each.  ctas: 1, or 2 with a's rows and b's shared out.
inline void emu_mma(int ctas, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t add) {
    static const float value[16] = {0, .5f, 1, 1.5f, 2, 3, 4, 6, -0.f, -.5f, -1, -1.5f, -2, -3, -4, -6};
    const uint32_t n_all = (idesc >> 17 & 63) * 8, m_all = (idesc >> 27 & 3) * 128, id_b = idesc >> 4 & 3, id_a = idesc >> 29 & 3;
    if ((idesc >> 7 & 7) != 1 || (idesc >> 10 & 7) != 1 || !(idesc >> 23 & 1) || m_all != 128u * ctas || n_all == 0 || n_all > 256 || n_all % (8 * ctas) ||
        a >> 61 != 2 || b >> 61 != 2 || (id_a & 1) || (id_b & 1))
        emu_fail("a matrix instruction's descriptors");
    for (int c = 0; c < ctas; c++) {
        const int rank = ctas == 2 ? c : emu_rank;
        EmuCta *cta = emu_cluster->cta[rank].get();
        std::vector<float> rows(128 * 64), cols(n_all * 64);
        for (uint32_t r = 0; r < 128; r++)
            for (uint32_t k = 0; k < 64; k++) {
                const uint8_t byte = emu_code(a, r, k / 2, rank);
                rows[r * 64 + k] = value[k & 1 ? byte >> 4 : byte & 15] * (float)emu_scale(cta, sa, r, id_a + k / 32);
            }
        for (uint32_t n = 0; n < n_all; n++)
            for (uint32_t k = 0; k < 64; k++) {
                const uint32_t part = n_all / ctas;
                const uint8_t byte = emu_code(b, n % part, k / 2, ctas == 2 ? (int)(n / part) : emu_rank);
                cols[n * 64 + k] = value[k & 1 ? byte >> 4 : byte & 15] * (float)emu_scale(cta, sb, n, id_b + k / 32);
            }
        for (uint32_t r = 0; r < 128; r++)
            for (uint32_t n = 0; n < n_all; n++) {
                double sum = 0;
                for (uint32_t k = 0; k < 64; k++) sum += (double)rows[r * 64 + k] * cols[n * 64 + k];
                uint32_t &cell = emu_cell(cta, r, (d & 0xFFFF) + n);
                float old = 0.0f, now;
                if (add) memcpy(&old, &cell, 4);
                now = (float)(old + sum);
                memcpy(&cell, &now, 4);
            }
    }
}
inline void emu_tmem_load(uint32_t at, uint32_t *r, int columns) {
    const uint32_t lanes = at >> 16;
    if (lanes != threadIdx.x / 32 % 4 * 32) emu_fail("a warp that reads other lanes than its own");
    for (int j = 0; j < columns; j++) r[j] = emu_cell(emu_cta, lanes + (threadIdx.x & 31), (at & 0xFFFF) + j);
}

// ------------------------------------------------------------------- the rest
template <class T>
inline T __ldg(const T *p) {
    if ((uintptr_t)p & (sizeof(T) - 1)) emu_fail("a misaligned load");
    return *p;
}
template <class A, class B>
inline auto min(A a, B b) -> decltype(a < b ? a : b) { return a < b ? a : b; }
template <class A, class B>
inline auto max(A a, B b) -> decltype(a < b ? a : b) { return a < b ? b : a; }
inline float __uint_as_float(unsigned u) {
    float f;
    memcpy(&f, &u, 4);
    return f;
}
inline unsigned __float_as_uint(float f) {
    unsigned u;
    memcpy(&u, &f, 4);
    return u;
}
inline unsigned __byte_perm(unsigned a, unsigned b, unsigned sel) {
    const unsigned long long ab = (unsigned long long)b << 32 | a;
    unsigned r = 0;
    for (int i = 0; i < 4; i++) r |= (unsigned)(ab >> 8 * (sel >> 4 * i & 7) & 0xFF) << 8 * i;
    return r;
}
template <class T>
inline T atomicExch(T *p, T v) { return __atomic_exchange_n(p, v, __ATOMIC_SEQ_CST); }
template <class T>
inline T atomicAdd(T *p, T v) { return __atomic_fetch_add(p, v, __ATOMIC_SEQ_CST); }
