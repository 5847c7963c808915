// mc_mx4_product.cu -- out[t][n] = sum over k of a[t][k] * b[n][k], both
// factors in microscaled 4-bit form, on the tensor cores (tcgen05.mma,
// kind::mxf4 with a scale per 32 elements), sums in float32.
//
// The matrices lie in memory as the tensor cores want them in shared memory:
// panels of 256 columns, in a panel 128 bytes a row with the 128-byte swizzle
// already applied, and the scales in pieces of 128 rows by 4.  So a tile of
// any rows is one contiguous run, and a bulk copy brings it in.

#include <cuda.h>

#include <type_traits>

#include "mc_mx4_device.h"

namespace {

// ------------------------------------------------------------ instructions
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_g2s(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// Every wait is bounded: false when it ran out (some seconds).  The clock is
// looked at late and rarely, and so is `failed` (or NULL), which ends the wait.
__device__ __noinline__ bool mbar_wait_long(uint32_t bar, uint32_t parity, uint32_t seconds, const volatile uint32_t *failed) {
    uint64_t t0, t;
    for (int i = 0; i < 256; i++)
        if (mbar_try_wait(bar, parity)) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    for (uint32_t i = 0; i < 1u << 26; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
        if (t - t0 > seconds * 1000000000ull || (failed && *failed)) return false;
    }
    return false;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t seconds, const volatile uint32_t *failed = NULL) {
    return mbar_try_wait(bar, parity) || mbar_wait_long(bar, parity, seconds, failed);
}

// The same for a barrier at which threads of another CTA of the cluster arrive.
__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, uint32_t seconds) {
    return mbar_try_wait_cluster(bar, parity) || (mbar_wait_long(bar, parity, seconds, NULL) && mbar_try_wait_cluster(bar, parity));
}

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
template <int COLUMNS>
__device__ __forceinline__ void tmem_alloc(uint32_t dst) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "n"(COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int COLUMNS>
__device__ __forceinline__ void tmem_free(uint32_t at) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "n"(COLUMNS));
}
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 512 bytes of scales (128 rows, 4 each) to 4 columns, for all four quarters of the lanes
__device__ __forceinline__ void tc_copy_scales(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                       uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(add) : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 16 columns of a warp's 32 lanes
__device__ __forceinline__ void tc_ld16(uint32_t at, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t at, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
                 : "=f"(v) : "r"(at), "r"(rank) : "memory");
    return v;
}

// Shared memory matrix, rows of 128 bytes with the 128-byte swizzle, 8 rows
// 1024 bytes further on.
__device__ __forceinline__ uint64_t desc_codes(uint32_t at) {
    return (uint64_t)(at >> 4 & 0x3FFF) | 1ull << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61;
}
// 16 bytes a row, 8 rows 128 bytes further on, no swizzle.
__device__ __forceinline__ uint64_t desc_scales(uint32_t at) {
    return (uint64_t)(at >> 4 & 0x3FFF) | 1ull << 16 | 8ull << 32 | 1ull << 46;
}

// CTAs in which a wait ran out.  Sums that may lack a part are then never said
// to be done, and who waits for them leaves NaN.
__device__ uint32_t g_mx_error;
#define MX_NAN 0x7FFFFFFFu

// ------------------------------------------------------------------ narrow
// Few tiles.  One tile of 128 x BN a CTA: b's rows are the instruction's M (128
// lanes of the sum), a's rows its N, so that neighbouring lanes are
// neighbouring elements of a row of `out`, and few rows of a (tokens) cost a
// narrow instruction instead of an empty one.  What bounds it is the way to b:
// an SM's shared memory is shared out in stages to the CTAs that it gets, 3 at
// most (1 x 50257 x 1024 in a graph: 6.8 us, 4.2 of them for the bytes at the
// copy rate; with 100 KB for each of 2 CTAs 9.3).  From 65 rows of a on tensor
// memory admits 2 CTAs of an SM, from 129 on one, and the rest stays empty.  The
// CTAs of a cluster have the same tile and a share of the panels each; their
// sums meet in the order of the ranks.  TX: a is not in 4 bits yet but has
// elements of this type; each CTA rounds what it needs (void: it is).
template <int BN, bool ROUND>
struct mx_cfg {
    static constexpr int GROUPS = BN > 128 ? 2 : 1;                  // of a's rows with scales
    static constexpr int B_BYTES = 128 * 128, A_BYTES = BN * 128, A_ALL = A_BYTES + GROUPS * 1024;   // of a panel
    static constexpr int STAGE = B_BYTES + 1024 + (ROUND ? 0 : A_ALL);
    static constexpr int SUMS = (BN * 512 + STAGE - 1) / STAGE;      // stages that a cluster's sums lie over
    static constexpr int SCALES = 8 + 8 * GROUPS;                    // columns of a panel's scales: each stage has its own
    static constexpr int COLUMNS = BN <= 64 ? 128 : 2 * BN;
    static constexpr int SLOTS = (COLUMNS - BN) / SCALES, FIT = 222 * 1024 / STAGE;
    static constexpr int MOST = SLOTS < FIT ? SLOTS : FIT;
    // CTAs that wait for columns may hold up others of their cluster, which have theirs: so whatever CTAs of these
    // kernels share an SM have columns for all.  Each takes over a fifth of the SM's 228 KB of shared memory for each
    // quarter of its 512 columns.
    static constexpr int LEAST = COLUMNS * 368;
    static_assert(SUMS <= MOST, "");
    // E2M1 both, E8M0 scales, M = 128
    static constexpr uint32_t IDESC = 1u << 7 | 1u << 10 | (uint32_t)(BN / 8) << 17 | 1u << 23 | 1u << 27;
};

#define MX_THREADS 192   // warps 0 to 3: results; 4: copies; 5: instructions

template <typename T, bool DROP>
__device__ __forceinline__ void put(const mx_product_launch &L, mx_key key, int64_t wide, int64_t t, int64_t n, float v) {
    if (DROP) {
        const uint32_t w = mx_word_at(key, (uint64_t)(t * wide + n) / 2);
        v = ((n & 1) ? w >> 16 : w & 0xFFFFu) < L.drop.threshold ? 0.0f : v * L.drop.factor;
    }
    mx_from((T *)L.out + t * L.ld + n, v);
}

// Rounds a's rows (all of them, 16 at most) of panels p0 to p1 to shared
// memory, `stride` bytes a panel: BN rows of codes, then scales.
template <typename TX, int BN>
__device__ __forceinline__ void round_rows(const mx_product_launch &L, uint32_t to, int stride, int p0, int p1) {
    const int units = (p1 - p0) * 32, all = (int)L.a.rows * units;   // of 8 elements; whole warps
    for (int u = threadIdx.x; u < all; u += 128) {
        const int r = u / units, q = u - r * units;
        const int64_t c = (int64_t)p0 * MX_PANEL + 8 * q;
        const TX *x = (const TX *)L.x + r * L.ld_x + c;
        mx_vec8<TX> v;
        memset(&v, 0, sizeof(v));
        if (L.vectors && c + 8 <= L.a.cols) {
            v = load8(x);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c + j < L.a.cols) v.x[j] = x[j];
        }
        uint32_t w[2 * sizeof(TX)], m = 0;
        memcpy(w, &v, sizeof(v));
#pragma unroll
        for (int j = 0; j < (int)(2 * sizeof(TX)); j++) m = larger(m, w[j], TX());
        uint32_t top = top_of(m, TX());
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t s = mx_scale(top);
        uint32_t codes = row_codes<TX, false, false>(w, mx_inverse(s), 1.0f, NULL);
        if (s == 255u) codes = 0;
        const int j = q / 4 & 7;   // block of the panel
        const uint32_t at = to + q / 32 * stride;
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + r * 128 + ((j ^ (r & 7)) * 16) + (q & 3) * 4), "r"(codes) : "memory");
        if ((q & 3) == 0)
            asm volatile("st.shared.b8 [%0], %1;" ::"r"(at + BN * 128 + (j >> 2) * 512 + r * 16 + (j & 3)), "r"(s) : "memory");
    }
}

// This rank's share of the rows [from, to) of a cluster's sums, [row][128]
// float32 at `sums` of each rank, added in the order of the ranks.  The others'
// come from far: 16 loads at a time.
template <typename T, int SPLIT, bool DROP>
__device__ __forceinline__ void meet(const mx_product_launch &L, mx_key key, int64_t wide, uint32_t sums, int64_t t0, int64_t n, int from, int to,
                                     bool inside) {
    constexpr int ROWS = 16 / SPLIT;
    const uint32_t mine = sums + threadIdx.x * 4;
#pragma unroll 1
    for (int c = from; c < to; c += ROWS) {
        float u[ROWS][SPLIT];
#pragma unroll
        for (int j = 0; j < ROWS; j++)
#pragma unroll
            for (int q = 0; q < SPLIT; q++)
                if (c + j < to) u[j][q] = ld_cluster(mine + (c + j) * 512, q);
#pragma unroll
        for (int j = 0; j < ROWS; j++) {
            float v = u[j][0];
#pragma unroll
            for (int q = 1; q < SPLIT; q++) v += u[j][q];
            if (c + j < to && inside) put<T, DROP>(L, key, wide, t0 + c + j, n, v);
        }
    }
}

// What failed leaves NaN.
__device__ __noinline__ void nan_sums(uint32_t at, int rows) {
    for (int c = 0; c < rows; c++) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + c * 512), "r"(MX_NAN) : "memory");
}
template <typename T, bool DROP>
__device__ __noinline__ void nan_out(const mx_product_launch &L, mx_key key, int64_t wide, int64_t t0, int64_t n, int rows) {
    for (int c = 0; c < rows; c++) put<T, DROP>(L, key, wide, t0 + c, n, __uint_as_float(MX_NAN));
}

template <typename T, int BN, bool DROP, typename TX>
__global__ void __launch_bounds__(MX_THREADS) k_mx_product(const __grid_constant__ mx_product_launch L, int tiles_n, int split, int stages) {
    constexpr bool ROUND = !std::is_same<TX, void>::value;
    typedef mx_cfg<BN, ROUND> C;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) uint64_t s_full[C::MOST], s_empty[C::MOST], s_done, s_quiet, s_stopped, s_rounded;
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem = (smem_u32(s_raw) + 1023) & ~1023u, own = smem + stages * C::STAGE;
    const int rank = blockIdx.x % split, tile = blockIdx.x / split;
    const int64_t n0 = (int64_t)(tile % tiles_n) * 128, t0 = (int64_t)(tile / tiles_n) * BN;
    const int64_t cols = L.a.cols;
    const int panels = (int)((cols + MX_PANEL - 1) / MX_PANEL);
    const int p0 = (int)((int64_t)panels * rank / split), p1 = (int)((int64_t)panels * (rank + 1) / split);

    if (warp == 5) tmem_alloc<C::COLUMNS>(smem_u32(&s_tmem));
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; i++) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_empty[i]), 1);
        }
        mbar_init(smem_u32(&s_done), 1);
        mbar_init(smem_u32(&s_quiet), 1);
        mbar_init(smem_u32(&s_stopped), 1);
        mbar_init(smem_u32(&s_rounded), 128);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        s_failed = 0;
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = s_tmem;
    mx_begin();

    if (warp == 4 && elect_one()) {
        const int64_t rows_b = mx_rows8(L.b.rows), rows_a = mx_rows8(L.a.rows);
        const int64_t groups_b = (L.b.rows + 127) / 128, groups_a = (L.a.rows + 127) / 128;
        const uint32_t nb = (uint32_t)min((int64_t)128, rows_b - n0) * 128, na = ROUND ? 0 : (uint32_t)min((int64_t)BN, rows_a - t0) * 128;
        const uint32_t ga = ROUND ? 0 : (uint32_t)min((int64_t)C::GROUPS, groups_a - t0 / 128) * 1024;
        const uint8_t *b = L.b.codes + ((int64_t)p0 * rows_b + n0) * 128, *sb = L.b.scales + ((int64_t)p0 * groups_b + n0 / 128) * 1024;
        const uint8_t *a = L.a.codes + ((int64_t)p0 * rows_a + t0) * 128, *sa = L.a.scales + ((int64_t)p0 * groups_a + t0 / 128) * 1024;
        int s = 0, round = 0;   // stage, times round
        bool ok = true;
        int p = p0;
        for (; p < p1; p++, b += rows_b * 128, sb += groups_b * 1024, a += rows_a * 128, sa += groups_a * 1024) {
            if (round > 0) ok = mbar_wait(smem_u32(&s_empty[s]), (round - 1) & 1, 4);
            if (!ok) break;
            const uint32_t at = smem + s * C::STAGE, bar = smem_u32(&s_full[s]);
            mbar_expect_tx(bar, nb + na + 1024 + ga);
            bulk_g2s(at, b, nb, bar);
            bulk_g2s(at + C::B_BYTES, sb, 1024, bar);
            if (!ROUND) {
                bulk_g2s(at + C::B_BYTES + 1024, a, na, bar);
                bulk_g2s(at + C::B_BYTES + 1024 + C::A_BYTES, sa, ga, bar);
            }
            if (++s == stages) {
                s = 0;
                round++;
            }
        }
        if (!ok) s_failed = 1;
        // no copy may outlive the CTA, whoever gave up: the last round of each stage
        for (int left = min(p - p0, stages); left > 0; left--) {
            if (s-- == 0) {
                s = stages - 1;
                round--;
            }
            mbar_wait(smem_u32(&s_full[s]), round & 1, 2);
        }
        mbar_arrive(smem_u32(&s_quiet));
    }
    if (warp == 5 && elect_one()) {
        bool ok = !ROUND || mbar_wait(smem_u32(&s_rounded), 0, 8);
        int s = 0, round = 0;   // stage, times round
        for (int p = p0; p < p1 && ok; p++) {
            const int i = p - p0;
            // a full stage is one whose last panel is done with, and so are that panel's columns of scales
            ok = mbar_wait(smem_u32(&s_full[s]), round & 1, 4);
            if (!ok) break;
            tc_after_sync();
            const uint32_t at = smem + s * C::STAGE, sb = at + C::B_BYTES;
            const uint32_t a = ROUND ? own + i * C::A_ALL : sb + 1024, sa = a + C::A_BYTES;
            const uint32_t cols_b = tmem + BN + s * C::SCALES, cols_a = cols_b + 8;
            const int steps = (int)min((int64_t)4, (cols - (int64_t)p * MX_PANEL + 63) / 64);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                tc_copy_scales(cols_b + h * 4, desc_scales(sb + h * 512));
#pragma unroll
                for (int g = 0; g < C::GROUPS; g++)
                    tc_copy_scales(cols_a + (h * C::GROUPS + g) * 4, desc_scales(sa + g * 1024 + h * 512));
            }
            const uint64_t db = desc_codes(at), da = desc_codes(a);
            for (int j = 0; j < steps; j++) {
                const uint32_t id = (j & 1) * 2, h = j >> 1;
                tc_mma(tmem, db + 2 * j, da + 2 * j, C::IDESC | id << 4 | id << 29, cols_b + h * 4,
                       cols_a + h * C::GROUPS * 4, i > 0 || j > 0);
            }
            tc_commit(smem_u32(&s_empty[s]));
            if (++s == stages) {
                s = 0;
                round++;
            }
        }
        if (ok) {
            tc_commit(smem_u32(&s_done));
        } else {   // what was issued ends before the memory goes
            s_failed = 1;
            tc_commit(smem_u32(&s_stopped));
            mbar_wait(smem_u32(&s_stopped), 0, 2);
        }
    }
    if constexpr (ROUND) {
        if (warp < 4) {
            round_rows<TX, BN>(L, own, C::A_ALL, p0, p1);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // for the tensor core
            mbar_arrive(smem_u32(&s_rounded));
        }
    }
    __syncwarp();

    bool failed = false;
    if (warp < 4) failed = !mbar_wait(smem_u32(&s_done), 0, 16, &s_failed);
    if (failed) {
        s_failed = 1;
        mbar_wait(smem_u32(&s_quiet), 0, 60);   // no copy that is late may come over what is left instead of the sums
    }
    tc_after_sync();
    const int64_t n = n0 + 32 * warp + lane;
    const int valid = (int)min((int64_t)BN, L.a.rows - t0);
    mx_key key = {};
    if (DROP) key = mx_key_of(L.drop.random);
    const int64_t wide = mx_wide(L.b.rows);
    const uint32_t mine = tmem + ((uint32_t)(32 * warp) << 16);
    if (split == 1) {
        if (warp < 4) {
            for (int c = 0; c < BN; c += 16) {
                if (c >= valid) break;
                uint32_t r[16];
                __syncwarp();
                tc_ld16(mine + c, r);
                tc_wait_ld();
                if (n < L.b.rows && !failed)
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (c + j < valid) put<T, DROP>(L, key, wide, t0 + c + j, n, panels ? __uint_as_float(r[j]) : 0.0f);
            }
            if (failed && n < L.b.rows) nan_out<T, DROP>(L, key, wide, t0, n, valid);
        }
    } else {
        // [BN][128] float32 over the stages, which are all used up
        if (warp < 4)
            for (int c = 0; c < BN && c < valid; c += 16) {
                uint32_t r[16];
                __syncwarp();
                tc_ld16(mine + c, r);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; j++)
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(smem + ((c + j) * 128 + 32 * warp + lane) * 4), "r"(r[j]) : "memory");
            }
        if (failed) nan_sums(smem + threadIdx.x * 4, valid);
        __syncwarp();
        cluster_sync();
        if (warp < 4) {
            const int from = valid * rank / split, to = valid * (rank + 1) / split;
            const bool inside = n < L.b.rows;
            if (split == 2) meet<T, 2, DROP>(L, key, wide, smem, t0, n, from, to, inside);
            else if (split == 4) meet<T, 4, DROP>(L, key, wide, smem, t0, n, from, to, inside);
            else meet<T, 8, DROP>(L, key, wide, smem, t0, n, from, to, inside);
        }
        __syncwarp();
        cluster_sync();
    }
    tc_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && s_failed) atomicAdd(&g_mx_error, 1u);
    if (warp == 5) tmem_free<C::COLUMNS>(tmem);
}

// ------------------------------------------------------------------- wide
// Many tiles of 256 x 256, each by a pair of CTAs on neighbouring SMs
// (cta_group::2): each has half of a's rows and half of b's in shared memory,
// and the sums of its half of a's rows, so a panel costs an SM 35 KB of copies
// instead of 51.  A pair takes tile after tile, and a tile's results leave
// while the next one is summed.  Here a's rows are the lanes and b's the
// columns of the sum, so that a lane has neighbouring elements of a row of
// `out` in its registers, rounds two at a time and stores 16 bytes at a time.
// Two sums of 256 columns and the scales of 5 panels are more than the 512
// columns there are, so the sums overlap by 128: those are read first, and the
// next tile's first instruction waits for that alone.  Bound by the tensor pipe
// at the clock that the power limit leaves (8192^3: 187 us, 5.9 PFLOP/s; 128 x
// 256 a CTA 207), or by the way out of the results.
struct mx_wide_cfg {
    static constexpr int BN = 256, THREADS = 320;                    // warps 0 to 7: results; 8: copies; 9: instructions
    static constexpr int A_BYTES = 128 * 128, B_BYTES = BN / 2 * 128;
    static constexpr int STAGE = A_BYTES + B_BYTES + 1024 + 2048, STAGES = 5;
    static constexpr int PITCH = 256 + 16, OUT = 32 * PITCH;         // two warps' part of the results: 32 rows, 256 bytes each
    static constexpr int SMEM = STAGES * STAGE + 4 * OUT + 1024;
    static constexpr int SECOND = 128, SCALES_AT = 384, SCALES = 24; // columns: a stage's scales have their own
    static constexpr uint32_t IDESC = 1u << 7 | 1u << 10 | (uint32_t)(BN / 8) << 17 | 1u << 23 | 2u << 27;
    static_assert(SMEM <= 227 * 1024 && SMEM >= 512 * 368 && SCALES_AT + STAGES * SCALES <= 512 && SECOND + BN <= SCALES_AT, "");
};

// The forms for a pair.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t at) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "n"(512));
}
__device__ __forceinline__ void tc_copy_scales_pair(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void tc_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                            uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(add) : "memory");
}
// Arrives at the barrier of both CTAs.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// Arrives at the first CTA's barrier.  Relaxed: the arriving thread has read
// sums (tcgen05.wait::ld) that may be written over now and hands on nothing
// that it wrote; a release at cluster scope would wait for its stores of
// results (over 1000 clocks).
__device__ __forceinline__ void mbar_arrive_first(uint32_t bar) {
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
                 "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(bar) : "memory");
}
// A word of the second CTA's.
__device__ __forceinline__ void st_second(uint32_t at, uint32_t v) {
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 1;\n\tst.shared::cluster.b32 [a], %1;\n\t}"
                 ::"r"(at), "r"(v) : "memory");
}
// A box of rows from `row` on to this CTA's shared memory, which the first
// CTA's barrier is told.
__device__ __forceinline__ void load_rows_pair(uint32_t dst, const CUtensorMap *map, int32_t row, uint32_t bar) {
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %3, 0;\n\t"
                 "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%2, %4}], [a];\n\t}"
                 ::"r"(dst), "l"(map), "r"(0), "r"(bar), "r"(row) : "memory");
}

__device__ __forceinline__ void st_shared16(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t at) {
    uint4 r;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
    return r;
}
__device__ __forceinline__ void bar_pair(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// 16 bytes of results.
__device__ __forceinline__ uint4 pack16(const float *v, float) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *(const uint32_t *)&p;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 p = __floats2half2_rn(a, b);
    return *(const uint32_t *)&p;
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float *v, T t) {
    return make_uint4(pack2(v[0], v[1], t), pack2(v[2], v[3], t), pack2(v[4], v[5], t), pack2(v[6], v[7], t));
}

// The 16 bytes that begin `from` (0, 2, ..., 16) bytes into a and then b.
__device__ __forceinline__ uint4 joined(uint4 a, uint4 b, uint32_t from) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const bool two = from & 8, one = from & 4;
#pragma unroll
    for (int i = 0; i < 6; i++) w[i] = two ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; i++) w[i] = one ? w[i + 1] : w[i];
    const uint32_t sel = from & 2 ? 0x5432u : 0x3210u;
    return make_uint4(__byte_perm(w[0], w[1], sel), __byte_perm(w[1], w[2], sel), __byte_perm(w[2], w[3], sel),
                      __byte_perm(w[3], w[4], sel));
}

// Every other of 32 rows of up to 256 bytes (`count` elements) from shared
// memory to `out` (of the first row), from row `first` (0 or 1) on.  16 lanes
// have a row, 16 bytes each.  A row that does not begin on a 16-byte boundary
// leaves in the 15 whole pieces that lie in it, put together from two, and 16 /
// SIZE elements at its two ends, one a lane (8192 x 50257 x 1024 to bf16: 295
// us; with 4-byte stores of whole rows 750, on boundaries 225, at the rate of
// a fill 213).
template <typename T>
__device__ __forceinline__ void rows_out(uint32_t buf, uint8_t *out, int64_t ld_bytes, int rows, int count, int first, int lane, bool even) {
    constexpr int SIZE = sizeof(T), PITCH = mx_wide_cfg::PITCH, BATCH = 4;
    const int h = lane & 15, r0 = first + 2 * (lane >> 4);   // rows r0, r0 + 4, ...
    uint8_t *g = out + r0 * ld_bytes;
    uint32_t at = buf + r0 * PITCH;
    // (all loads of a batch before its stores: one after the other they would wait for each other)
    if (even && count * SIZE == 256) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = ld_shared16(at + 4 * i * PITCH + 16 * h);
#pragma unroll
        for (int i = 0; i < 8; i++, g += 4 * ld_bytes)
            if (r0 + 4 * i < rows) *(uint4 *)(g + 16 * h) = v[i];
    } else if (count * SIZE == 256) {
#pragma unroll 1
        for (int r = r0; r < 32; r += 4 * BATCH, at += 4 * BATCH * PITCH) {
            uint4 now[BATCH], last[BATCH];
            uint32_t end[BATCH], off[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const uint32_t row = at + 4 * i * PITCH;
                off[i] = ((uint32_t)(uintptr_t)g + 4 * i * (uint32_t)ld_bytes) & 15;
                now[i] = ld_shared16(row + 16 * h);
                last[i] = ld_shared16(row + 16 * h - (h && off[i] ? 16 : 0));   // (a row that is on a boundary: itself)
                // the elements at the ends: 16 - off bytes of them in front
                const uint32_t e = row + (h * SIZE & 15) + (h * SIZE < 16 - off[i] ? 0 : 240);
                if (SIZE == 4) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(end[i]) : "r"(e) : "memory");
                else asm volatile("{\n\t.reg .b16 x;\n\tld.shared.b16 x, [%1];\n\tcvt.u32.u16 %0, x;\n\t}" : "=r"(end[i]) : "r"(e) : "memory");
            }
#pragma unroll
            for (int i = 0; i < BATCH; i++, g += 4 * ld_bytes) {   // (no branches: the two rows of a warp may differ)
                const bool in = r + 4 * i < rows;
                const uint4 v = joined(last[i], now[i], 16 - off[i]);
                if (in && (h > 0 || off[i] == 0)) *(uint4 *)(g + (int)(16 * h - off[i])) = v;
                uint8_t *e = g + h * SIZE + (h * SIZE < 16 - off[i] ? 0 : 240);
                if (in && off[i] != 0 && h * SIZE < 16) {
                    if (SIZE == 4) *(uint32_t *)e = end[i];
                    else *(uint16_t *)e = (uint16_t)end[i];
                }
            }
        }
    } else {   // the last columns of the matrix
        for (int r = first; r < rows; r += 2)
            for (int i = lane; i < count; i += 32) {
                if (SIZE == 4) {
                    uint32_t v;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(buf + r * PITCH + 4 * i) : "memory");
                    ((uint32_t *)(out + r * ld_bytes))[i] = v;
                } else {
                    uint16_t v;
                    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(buf + r * PITCH + 2 * i) : "memory");
                    ((uint16_t *)(out + r * ld_bytes))[i] = v;
                }
            }
    }
}

// Codes as rows of 128 bytes, scales as rows of 1024, of all panels.
struct mx_maps {
    CUtensorMap a_codes, b_codes, a_scales, b_scales;
};

template <typename T, bool DROP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(mx_wide_cfg::THREADS, 1)
    k_mx_product_wide(const __grid_constant__ mx_product_launch L, const __grid_constant__ mx_maps M, int tiles_n, int tiles) {
    typedef mx_wide_cfg C;
    constexpr int CHUNK = 128 / sizeof(T), PARTS = 64 / CHUNK, E = 16 / sizeof(T), BN = C::BN, COPIES = 8, ISSUE = 9;
    extern __shared__ uint8_t s_raw[];
    // s_full: both CTAs' copies, at the first; s_done, s_free: for even and for odd tiles
    __shared__ __align__(8) uint64_t s_full[C::STAGES], s_empty[C::STAGES], s_done[2], s_free[2], s_stopped;
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t smem = (smem_u32(s_raw) + 1023) & ~1023u;
    const int64_t cols = L.a.cols;
    const int panels = (int)((cols + MX_PANEL - 1) / MX_PANEL), last_steps = (int)((cols - 1) % MX_PANEL) / 64 + 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; i++) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_empty[i]), 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_u32(&s_done[i]), 1);
            mbar_init(smem_u32(&s_free[i]), 16);   // the result warps of both
        }
        mbar_init(smem_u32(&s_stopped), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        s_failed = 0;
    }
    __syncthreads();
    cluster_sync();
    if (warp == ISSUE) tmem_alloc_pair(smem_u32(&s_tmem));
    tc_before_sync();
    __syncthreads();
    cluster_sync();
    tc_after_sync();
    const uint32_t tmem = s_tmem;
    mx_begin();

    if (warp == COPIES) {
        // One lane for each of a panel's four copies: codes of a and of b, scales of a and of b.  Boxes are whole: what
        // lies behind a matrix's last row belongs to rows or columns of the sum that nobody stores.
        const CUtensorMap *map = lane == 0 ? &M.a_codes : lane == 1 ? &M.b_codes : lane == 2 ? &M.a_scales : &M.b_scales;
        const int stride = (int)(lane == 0 ? mx_rows8(L.a.rows) : lane == 1 ? mx_rows8(L.b.rows) : ((lane == 2 ? L.a.rows : L.b.rows) + 127) / 128);
        const uint32_t to = smem + (lane == 0 ? 0 : lane == 1 ? C::A_BYTES : C::A_BYTES + C::B_BYTES + (lane == 2 ? 0 : 1024));
        int s = 0, used = 0;   // stage; stages used so far, up to all
        uint32_t parity = 1;   // of the wait for an empty stage
        bool ok = true;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const int n0 = tile % tiles_n * BN, t0 = tile / tiles_n * 256 + 128 * rank;
            int row = lane == 0 ? t0 : lane == 1 ? n0 + BN / 2 * rank : lane == 2 ? t0 / 128 : n0 / 128;
            for (int p = 0; p < panels; p++, row += stride) {
                const uint32_t bar = smem_u32(&s_full[s]);
                if (lane == 0) {
                    if (used == C::STAGES) ok = mbar_wait(smem_u32(&s_empty[s]), parity, 4);
                    if (ok && rank == 0) mbar_expect_tx(bar, 2 * C::STAGE);
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                if (lane < 4) load_rows_pair(to + s * C::STAGE, map, row, bar);
                used = min(used + 1, C::STAGES);
                if (++s == C::STAGES) {
                    s = 0;
                    parity ^= 1;
                }
            }
        }
        if (lane == 0 && !ok) s_failed = 1;
        // no copy may outlive the pair, whoever gave up: the last round of each stage
        if (lane == 0 && rank == 0)
            for (; used > 0; used--) {
                if (s-- == 0) {
                    s = C::STAGES - 1;
                    parity ^= 1;
                }
                mbar_wait(smem_u32(&s_full[s]), parity ^ 1, 2);
            }
    }
    if (warp == ISSUE && rank == 0 && elect_one()) {
        const uint64_t codes = desc_codes(smem), scales = desc_scales(smem + C::A_BYTES + C::B_BYTES);
        int s = 0, count = 0;
        uint32_t parity = 0;
        bool ok = true;
        for (int tile = pair; tile < tiles; tile += pairs, count++) {
            const uint32_t sum = tmem + (count & 1) * C::SECOND;
            // the tile before has left the overlap
            if (count > 0) ok = mbar_wait_cluster(smem_u32(&s_free[(count - 1) & 1]), (count - 1) >> 1 & 1, 4);
            tc_after_sync();
            for (int p = 0; p < panels && ok; p++) {
                ok = mbar_wait_cluster(smem_u32(&s_full[s]), parity, 4);
                // a full stage is one whose last panel is done with, and so are that panel's columns of scales
                if (!ok) break;
                tc_after_sync();
                const uint64_t da = codes + s * (C::STAGE >> 4), db = da + (C::A_BYTES >> 4);
                const uint64_t sa = scales + s * (C::STAGE >> 4), sb = sa + (1024 >> 4);
                const uint32_t cols_a = tmem + C::SCALES_AT + s * C::SCALES, cols_b = cols_a + 8;
                const int steps = p + 1 < panels ? 4 : last_steps;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    tc_copy_scales_pair(cols_a + h * 4, sa + h * (512 >> 4));
#pragma unroll
                    for (int g = 0; g < 2; g++) tc_copy_scales_pair(cols_b + (h * 2 + g) * 4, sb + g * (1024 >> 4) + h * (512 >> 4));
#pragma unroll
                    for (int j = 2 * h; j < 2 * h + 2; j++) {
                        const uint32_t id = (j & 1) * 2;
                        if (j < steps)
                            tc_mma_pair(sum, da + 2 * j, db + 2 * j, C::IDESC | id << 4 | id << 29, cols_a + h * 4, cols_b + h * 8,
                                        p > 0 || j > 0);
                    }
                }
                tc_commit_pair(smem_u32(&s_empty[s]));
                if (++s == C::STAGES) {
                    s = 0;
                    parity ^= 1;
                }
            }
            if (!ok) break;
            tc_commit_pair(smem_u32(&s_done[count & 1]));
        }
        if (!ok) {   // what was issued ends before the memory goes
            s_failed = 1;
            st_second(smem_u32((const void *)&s_failed), 1);
            tc_commit_pair(smem_u32(&s_stopped));
            mbar_wait(smem_u32(&s_stopped), 0, 2);
        }
    }
    __syncwarp();
    if (warp < COPIES) {
        const int set = warp >> 2, quarter = warp & 3;
        const uint32_t buf = smem + C::STAGES * C::STAGE + quarter * C::OUT;
        const int64_t ld_bytes = L.ld * (int64_t)sizeof(T), wide = mx_wide(L.b.rows);
        const bool even = (((uintptr_t)L.out | (uintptr_t)ld_bytes) & 15) == 0;
        mx_key key = {};
        if (DROP) key = mx_key_of(L.drop.random);
        int count = 0;
        bool failed = false;   // the tiles that follow are not summed either
        for (int tile = pair; tile < tiles; tile += pairs, count++) {
            const int64_t n0 = (int64_t)(tile % tiles_n) * BN, t0 = (int64_t)(tile / tiles_n) * 256 + 128 * rank + 32 * quarter;
            const int rows = (int)max((int64_t)0, min((int64_t)32, L.a.rows - t0)), columns = (int)min((int64_t)BN, L.b.rows - n0);
            uint8_t *out = (uint8_t *)L.out + t0 * ld_bytes + n0 * (int64_t)sizeof(T);
            if (!failed) failed = !mbar_wait(smem_u32(&s_done[count & 1]), count >> 1 & 1, 20, &s_failed);
            if (failed) s_failed = 1;
            tc_after_sync();
            const uint32_t mine = tmem + (count & 1) * C::SECOND + ((uint32_t)(32 * quarter) << 16);
            // first the overlap: columns 128 on of even tiles, the first 128 of odd ones
            for (int k = 0; k < 2 * PARTS; k++) {
                const int both = ((k < PARTS) == ((count & 1) == 0) ? 128 : 0) + k % PARTS * 2 * CHUNK, c = both + set * CHUNK;
                const bool some = both < columns && rows > 0;   // the same for both warps
                float v[CHUNK];
                if (some) {
#pragma unroll
                    for (int j = 0; j < CHUNK; j += 16) tc_ld16(mine + c + j, (uint32_t *)v + j);
                    tc_wait_ld();
                    if (failed)
#pragma unroll
                        for (int j = 0; j < CHUNK; j++) v[j] = __uint_as_float(MX_NAN);
                }
                if (k == PARTS - 1) {   // the overlap is read, and all of the tile before
                    tc_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_first(smem_u32(&s_free[count & 1]));
                }
                if (!some) continue;
                if (DROP) {
                    const uint64_t pos = (uint64_t)((t0 + lane) * wide + n0 + c) / 2;
                    uint32_t start = 0;
#pragma unroll
                    for (int j = 0; j < CHUNK; j += 2) {
                        if (j % 8 == 0) start = mx_start(key, pos + j / 2);
                        const uint32_t w = mx_word(key, start ^ (j / 2 & 3));
                        v[j] = (w & 0xFFFFu) < L.drop.threshold ? 0.0f : v[j] * L.drop.factor;
                        v[j + 1] = (w >> 16) < L.drop.threshold ? 0.0f : v[j + 1] * L.drop.factor;
                    }
                }
                bar_pair(1 + quarter);   // the last part has left the buffer
#pragma unroll
                for (int j = 0; j < CHUNK; j += E) st_shared16(buf + lane * C::PITCH + (set * CHUNK + j) * sizeof(T), pack16(v + j, T()));
                bar_pair(1 + quarter);
                rows_out<T>(buf, out + both * (int64_t)sizeof(T), ld_bytes, rows, min(2 * CHUNK, columns - both), set, lane, even);
            }
        }
    }
    tc_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && s_failed) atomicAdd(&g_mx_error, 1u);
    cluster_sync();   // nothing of the pair is in use any more
    tc_after_sync();
    if (warp == ISSUE) tmem_free_pair(tmem);
    __syncwarp();
    cluster_sync();
}

typedef CUresult (*mx_encode_fn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// `words` 32-bit words a row, `box` rows a copy.
static bool map_rows(mx_encode_fn encode, CUtensorMap *map, const uint8_t *base, int64_t rows, int words, int box) {
    const cuuint64_t size[2] = {(cuuint64_t)words, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)words * 4};
    const cuuint32_t part[2] = {(cuuint32_t)words, (cuuint32_t)box}, step[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, (void *)base, size, stride, part, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static mx_encode_fn encoder() {
    static mx_encode_fn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            return (mx_encode_fn) nullptr;
        }
        return (mx_encode_fn)p;
    }();
    return fn;
}

template <typename T, bool DROP>
static int product_wide(const mx_product_launch &L, int sms, cudaStream_t s) {
    typedef mx_wide_cfg C;
    auto kern = k_mx_product_wide<T, DROP>;
    const cudaError_t e = mx_allow(kern, C::SMEM);
    if (e != cudaSuccess) return e;
    const int64_t tiles_n = (L.b.rows + C::BN - 1) / C::BN, tiles = tiles_n * ((L.a.rows + 255) / 256);
    if (tiles > 0x3FFFFFFF) return cudaErrorInvalidValue;
    const int pairs = (int)(tiles < sms / 2 ? tiles : sms / 2);
    const int64_t panels = (L.a.cols + MX_PANEL - 1) / MX_PANEL;
    const mx_encode_fn encode = encoder();
    mx_maps M;
    if (!encode || !map_rows(encode, &M.a_codes, L.a.codes, panels * ((L.a.rows + 7) / 8 * 8), 32, 128) ||
        !map_rows(encode, &M.b_codes, L.b.codes, panels * ((L.b.rows + 7) / 8 * 8), 32, C::BN / 2) ||
        !map_rows(encode, &M.a_scales, L.a.scales, panels * ((L.a.rows + 127) / 128), 256, 1) ||
        !map_rows(encode, &M.b_scales, L.b.scales, panels * ((L.b.rows + 127) / 128), 256, 2))
        return cudaErrorNotSupported;
    return mx_launch(kern, 2 * pairs, C::THREADS, C::SMEM, 0, s, L, M, (int)tiles_n, (int)tiles);
}

template <typename T, int BN, bool DROP, typename TX = void>
static int product_as(const mx_product_launch &L, int sms, cudaStream_t s) {
    constexpr bool ROUND = !std::is_same<TX, void>::value;
    typedef mx_cfg<BN, ROUND> C;
    const int64_t tiles_n = (L.b.rows + 127) / 128, tiles_t = (L.a.rows + BN - 1) / BN, tiles = tiles_n * tiles_t;
    const int64_t panels = (L.a.cols + MX_PANEL - 1) / MX_PANEL;
    int split = 1;
    while (split < 8 && tiles * split * 2 <= sms && split * 2 <= panels) split *= 2;
    if (tiles * split > 0x7FFFFFFF) return cudaErrorInvalidValue;
    // as many stages as the CTAs of an SM have room for, and use for
    const int64_t ctas = (tiles * split + sms - 1) / sms, each = (panels + split - 1) / split;
    const int own = 1024 + (ROUND ? (int)each * C::A_ALL : 0), least = split > 1 ? C::SUMS : 1;
    int stages = (222 * 1024 / (int)(ctas < 3 ? ctas : 3) - own) / C::STAGE;
    if (stages > each) stages = (int)each;
    if (stages < least) stages = least;
    if (stages > C::MOST) stages = C::MOST;
    const int need = own + stages * C::STAGE, smem = need < C::LEAST ? C::LEAST : need;
    auto kern = k_mx_product<T, BN, DROP, TX>;
    const cudaError_t e = mx_allow(kern, 225 * 1024);
    if (e != cudaSuccess) return e;
    return mx_launch(kern, tiles * split, MX_THREADS, smem, split, s, L, (int)tiles_n, split, stages);
}

template <typename T, bool DROP>
static int product_for(const mx_product_launch &L, int sms, cudaStream_t s) {
    const int64_t t = L.a.rows;
    if (t <= 16) return product_as<T, 16, DROP>(L, sms, s);
    if (t <= 32) return product_as<T, 32, DROP>(L, sms, s);
    if (t <= 64) return product_as<T, 64, DROP>(L, sms, s);
    if (t <= 128) return product_as<T, 128, DROP>(L, sms, s);
    const int64_t tiles = (L.b.rows + 255) / 256 * ((t + 255) / 256) * 2;
    // fewer tiles than SMs: their panels are shared out
    if (tiles * 2 <= sms || L.a.cols == 0 || L.b.rows <= 128) return product_as<T, 256, DROP>(L, sms, s);
    return product_wide<T, DROP>(L, sms, s);
}

template <typename T>
static int product(const mx_product_launch &L, int sms, cudaStream_t s) {
    if (L.x) {
        if (L.x_type == FALCOM_TYPE_F32) return product_as<T, 16, false, float>(L, sms, s);
        if (L.x_type == FALCOM_TYPE_BF16) return product_as<T, 16, false, __nv_bfloat16>(L, sms, s);
        return product_as<T, 16, false, __half>(L, sms, s);
    }
    return L.drop.random.on ? product_for<T, true>(L, sms, s) : product_for<T, false>(L, sms, s);
}

}  // namespace

extern "C" int mc_launch_mx_product(const mx_product_launch *L, int type, int sms, void *stream) {
    if (type == FALCOM_TYPE_F32) return product<float>(*L, sms, (cudaStream_t)stream);
    if (type == FALCOM_TYPE_BF16) return product<__nv_bfloat16>(*L, sms, (cudaStream_t)stream);
    return product<__half>(*L, sms, (cudaStream_t)stream);
}

extern "C" int mc_mx_errors(uint32_t *word) { return cudaMemcpyFromSymbol(word, g_mx_error, sizeof(*word)); }
