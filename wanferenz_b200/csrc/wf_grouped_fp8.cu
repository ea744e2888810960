// wf_grouped_fp8.cu - the experts' block-scaled FP8 product on tcgen05.
//
//   out[r, n] = sum_k (a[row(r), k] * a_s[row(r), k/128]) * (w[e, n, k] * w_s[e, n/128, k/128])
//   for expert e and r in [offsets[e], offsets[e+1]), row(r) = rows[r] (or r)
//
// Weight rows are the M side of the MMA, tokens the N side: an expert's rows are cut
// into tiles of about equal width, multiples of 32 up to 256, so a few rows cost a few
// columns and an expert pads to 32 rows once.  A pair of CTAs (cta_group::2) works on 256
// weight rows: each holds 128 of them (one block of weight scales) and half of the
// tokens in shared memory, and the products of its own 128 rows in its TMEM, so a
// 256-wide tile moves 32 KB into each SM per 128-wide K step, half of what single
// CTAs of 128 x 128 would.
//
// Scales.  With e8m0 on both sides the tensor core applies them (kind::mxf8f6f4; a
// byte per 128 K repeated for its four 32-wide products) and sums the whole of K in
// TMEM.  Otherwise each 128-wide K step's product goes to a fresh accumulator, and the
// worker warps scale and add it in 32-bit registers while the next step multiplies.
// For many rows per expert those sums are all that counts, and the sides change places
// (k_grouped_f32_wide): a token per TMEM lane, so that a thread's scale is one register.
// (A scale per column comes from shared memory, 4 bytes a lane and column whether the
// lanes read the same ones or not: 131 KB a K step, as many cycles as the whole product.)
//
// Measured on a B200.  Few rows per expert, bound by the weights' stream (5.5 TB/s while it
// runs): 96 rows over 64 experts of 2048 x 2048, e8m0, 40 us (floor 32); 1536 rows over 64 of
// 2048 x 1024, f32, 35.4 us (21.7).  Many: one expert of 16384 rows, 4096 x 4096, e8m0, 2.7 to 2.8
// PFLOP/s in a call by itself, 2.3 in a loop under the 1 kW cap; 16386 rows over 32 of these
// experts 264 us by itself (floor 174) and 298 in a loop, with a row list to pack 277 and 332: the
// tensor cores wait for the one accumulator at the end of each tile.  With f32 scales 397 and 444,
// with a list 417 and 461: a worker's load of products, its wait and its additions follow one
// another, neither the tensor pipe (36 %) nor the issue slots (35 %) are full.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/wfb200.h"
#include "wf_host.h"
#include "wf_ptx.cuh"
#include "wf_tcgen05.cuh"

namespace wf {
namespace grp {

using namespace tc;

__device__ int g_err;  // error flags of the grouped products since the last wf_grouped_read_error

constexpr int MAX_E = 512;
constexpr int SGRP = 8;                 // K steps per group of scales
// Rows per expert up to which tiles are narrow (32 experts of 2048 x 2048, rows in order, narrow
// against wide tiles in us: e8m0 48 rows 27.8 / 34.1, 64 31.2 / 35.1, 96 40.2 / 36.8; f32 48 rows
// 32.1 / 32.3, 64 37.0 / 33.9) ...
constexpr int NARROW_E8 = 64, NARROW_F32 = 48;
// ... and up to which a row list is gathered in place, by TMA copies of four rows, instead of
// packed into expert order first (the same with e8m0 and narrow tiles: gathered 4 rows 28.1, 8 30.4,
// 16 33.3, 32 40.0; packed 16 29.9, 32 30.3).  The TMA unit takes about 80 cycles for a four-row
// copy, as long as for a box of 128 rows.
constexpr int GATHER = 12;
constexpr int W_PROD = 0, W_MMA = 1, WORKERS = 8;
constexpr int SMEM_MAX = 232448;
constexpr int TAB_BYTES = 2 * MAX_E * 4 + (MAX_E + 1) * 8;  // per expert: first row, rows, first token tile

// NT: tokens per tile, at most.  Narrow tiles, for few rows per expert, leave room for ten stages and
// for accumulators ahead of the workers: there the weights' stream from HBM is all that counts, and
// nothing may pause it.
template <bool E8, int NT>
struct Plan {
    // e8m0: 4 scale warps, one per TMEM lane quadrant; f32: 2
    static constexpr int SCALE0 = E8 ? 4 : 2, SCALERS = E8 ? 4 : 2, WORK0 = SCALE0 + SCALERS;
    static constexpr int THREADS = 32 * (WORK0 + WORKERS);
    static constexpr int ABYTES = 128 * 128, BBYTES = NT / 2 * 128, STAGE = ABYTES + BBYTES;
    static constexpr int STAGES = NT == 256 ? 6 : 10;
    // TMEM: sums of whole tiles (e8m0) and two groups of scale factors, or products of K steps (f32)
    static constexpr int NACC = E8 ? (NT == 256 ? 1 : 4) : 512 / NT;
    static constexpr int SFB = NT / 32 < 4 ? 4 : NT / 32;  // columns of a K step's token scale factors
    static constexpr uint32_t COL_SFA = 256, COL_SFB = COL_SFA + 2 * SGRP * 4;
    static constexpr int NBAR = 2 * STAGES + 2 * NACC + 5;
    static constexpr int OFF_S = STAGES * STAGE;         // scales: [2][SGRP][NT] f32 or [2][NT] x 8 bytes
    static constexpr int OFF_TAB = OFF_S + 2 * SGRP * NT * 4;
    static constexpr int OFF_BAR = OFF_TAB + TAB_BYTES;
    static constexpr int SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
    static_assert(SMEM <= SMEM_MAX && OFF_BAR % 8 == 0, "shared memory");
    static_assert(E8 ? NACC * NT <= 256 && COL_SFB + 2 * SGRP * SFB <= 512 : NT == 64, "tensor memory");
};

// The bound of the waits on another role: a wait ends `cycles` after its first miss.  A bound lowered
// by wf_set_wait_limit is kept by polling; try_wait may suspend the thread for longer.
struct Bound {
    long long cycles;
    uint32_t poll;
};
struct Args {
    CUtensorMap tmW;     // weights [E*N, K], box 128 x 128
    CUtensorMap tmA[4];  // rows [M, K], boxes of 128, 64, 32 and 16 rows; the first of one row to gather
    const void *a_s, *w_s;
    const int *offsets, *rows;
    __nv_bfloat16 *out;
    Bound limit;
    int M, R, E, N, K, a_f32, w_f32;
    int gather;          // the tensor map's rows are those of `rows`, else the product's own
};

// ---- CTA pairs ------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's `p` in CTA 0 of the pair.
__device__ __forceinline__ uint32_t leader_addr(const void *p) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}
// The pair's barriers hand over TMEM (ordered by the tcgen05 fences) and copies of the
// async proxy, no ordinary memory, so arrivals and waits keep the default CTA scope:
// cluster scope would flush stores on every arrival and drop the L1 on every wait
// (measured: over 1000 cycles of each K step's hand-over).
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool wait_once(uint64_t *bar, uint32_t parity, uint32_t poll) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %3, 0;\n\t"
        "@q mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@!q mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(poll)
        : "memory");
    return ok != 0;
}
// Bounded wait; a wait that runs out sets the error flag and tells the CTA's other roles.
__device__ __forceinline__ bool twait(uint64_t *bar, uint32_t parity, volatile int *abort, const Bound &limit) {
    if (wait_once(bar, parity, limit.poll)) return true;
    const long long t0 = clock64();
    while (!wait_once(bar, parity, limit.poll)) {
        if (*abort) return false;
        if (clock64() - t0 > limit.cycles) {
            atomicOr(&g_err, kErrTimeout);
            *abort = 1;
            return false;
        }
    }
    return true;
}

__device__ __forceinline__ void tmem_alloc2(uint32_t *dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Arrive on `bar` of the CTAs in `mask` once every tcgen05 operation this thread issued so far is complete.
__device__ __forceinline__ void commit2(uint64_t *bar, uint16_t mask = 3) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(mask)
        : "memory");
}

// Whether `v` holds in all `n` threads of the named barrier.
__device__ __forceinline__ bool bar_all(int id, int n, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %3, 0;\n\t"
        "bar.red.and.pred q, %1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(id), "r"(n), "r"((uint32_t)v)
        : "memory");
    return r != 0;
}

__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r != 0;
}

// ---- MMA: M = 256 over the pair, both operands K-major E4M3 ----------------
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
}
// kind::f8f6f4, f32 accumulator
__device__ __forceinline__ uint32_t idesc_f8(int n) { return 1u << 4 | (uint32_t)(n >> 3) << 17 | (256u >> 4) << 24; }
// kind::mxf8f6f4, UE8M0 scales, byte sf_id of the scale words
__device__ __forceinline__ uint32_t idesc_mx(int n, uint32_t sf_id) {
    return sf_id << 4 | (uint32_t)(n >> 3) << 17 | 1u << 23 | (256u >> 7) << 27 | sf_id << 29;
}

// ---- TMA into this CTA's memory, completion on the leader's barrier --------
__device__ __forceinline__ void tma_load2(void *dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
// The same with an L2 policy.
__device__ __forceinline__ void tma_load2_hint(void *dst, const CUtensorMap *map, int c0, int c1, uint32_t bar, uint64_t pol) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar), "l"(pol)
        : "memory");
}
// Four rows of the tensor map, 128 bytes each, to 512 consecutive (swizzled) bytes.
__device__ __forceinline__ void tma_gather4(void *dst, const CUtensorMap *map, int c0, int4 r, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// ---- tiles -----------------------------------------------------------------
struct Tile {
    int e, n0, r0, nrow, width;
};

// Every expert's rows, clamped to the R rows there are, and its first token tile, in shared memory.
// (Tiles are counted in 64 bits: offsets that fall again may give every expert all the rows.)
struct Table {
    int *lo, *cnt;
    long long *first;
    __device__ explicit Table(uint8_t *at)
        : lo(reinterpret_cast<int *>(at)), cnt(lo + MAX_E), first(reinterpret_cast<long long *>(cnt + MAX_E)) {}
    // By all threads; complete for the caller's next barrier.
    __device__ void fill(const Args &p, int nt) const {
        for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
            const int a = min(max(p.offsets[e], 0), p.R), b = min(max(p.offsets[e + 1], 0), p.R);
            lo[e] = a;
            cnt[e] = max(b - a, 0);
        }
        __syncthreads();
        if (threadIdx.x >= 32) return;
        const int lane = threadIdx.x;
        long long sum = 0, own[MAX_E / 32];
#pragma unroll
        for (int j = 0; j < MAX_E / 32; ++j) {
            const int e = lane * (MAX_E / 32) + j;
            own[j] = sum;
            if (e < p.E) sum += (cnt[e] + nt - 1) / nt;
        }
        long long incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
#pragma unroll
        for (int j = 0; j < MAX_E / 32; ++j) {
            const int e = lane * (MAX_E / 32) + j;
            if (e < p.E) first[e] = incl - sum + own[j];
        }
        if (lane == 31) first[p.E] = incl;
    }
};

// Tiles of a CTA (pair) in order; within an expert the tile of 256 weight rows runs fastest.
struct Walk {
    Table tab;
    int E, nn, step, e;
    long long i;
    // Cuts an expert's rows into tiles whose widths differ by 32 at most, or of `fixed` rows.
    __device__ bool next(Tile &t, int fixed = 0) {
        while (e < E && i >= tab.first[e + 1] * nn) ++e;
        if (e >= E) return false;
        const int local = (int)(i - tab.first[e] * nn);
        const int nt = (int)(tab.first[e + 1] - tab.first[e]), c = tab.cnt[e];
        t.e = e;
        t.n0 = local % nn * 256;
        const int j = local / nn;
        int at = j * fixed;
        t.width = fixed;
        if (!fixed) {  // cta_group::2 takes N in steps of 32
            const int units = (c + 31) / 32, each = units / nt, more = units - each * nt;
            t.width = 32 * (each + (j < more));
            at = 32 * (j * each + min(j, more));
        }
        t.r0 = tab.lo[e] + at;
        t.nrow = min(t.width, c - at);
        i += step;
        return true;
    }
};

__device__ __forceinline__ float scale_at(const void *s, int f32, size_t i) {
    if (f32) return __ldg((const float *)s + i);
    const uint32_t b = __ldg((const uint8_t *)s + i);
    return b == 255 ? __uint_as_float(0x7fffffffu) : e8m0_to_f32(b);
}

// The row of `a` that row r of the product reads, clamped into a; `valid` says whether it was inside.
__device__ __forceinline__ int source_row(const Args &p, int r, bool &valid) {
    const int s = p.rows ? __ldg(p.rows + r) : r;
    valid = s >= 0 && s < p.M;
    return valid ? s : 0;
}

// Rows of the tile that CTA `rank` of the pair loads: in fours to gather, else in sixteens.
__device__ __forceinline__ int rows_held(const Tile &t, int half, int rank, int gather) {
    const int n = min(max(t.nrow - half * rank, 0), half);
    return gather ? (n + 3) & ~3 : (n + 15) & ~15;
}

template <bool E8, int NT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Plan<E8, NT>::THREADS, 1)
    k_grouped_fp8(const __grid_constant__ Args p) {
    using L = Plan<E8, NT>;
    constexpr int STAGES = L::STAGES, STAGE = L::STAGE, ABYTES = L::ABYTES, NACC = L::NACC, HALF = NT / 2;
    constexpr uint32_t COL_SFA = L::COL_SFA, COL_SFB = L::COL_SFB;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bar = reinterpret_cast<uint64_t *>(base + L::OFF_BAR);
    // full, ready-for-MMA and freed accumulators live in the leader; empty, acc_ready in both
    uint64_t *full = bar, *empty = bar + STAGES, *acc_ready = empty + STAGES, *acc_free = acc_ready + NACC;
    uint64_t *sf_full = acc_free + NACC, *sf_empty = sf_full + 2, *fin = sf_empty + 2;
    uint32_t *tmem_base = reinterpret_cast<uint32_t *>(bar + L::NBAR);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_base + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const int nks = p.K / 128, nn = (p.N + 255) / 256, nb = (p.N + 127) / 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
        for (int j = 0; j < NACC; ++j) {
            mbar_init(acc_ready + j, 1);
            mbar_init(acc_free + j, 2 * WORKERS);
        }
        for (int j = 0; j < 2; ++j) {
            mbar_init(sf_full + j, E8 ? 2 * L::SCALERS : L::SCALERS);
            mbar_init(sf_empty + j, E8 ? 1 : WORKERS);
        }
        mbar_init(fin, 1);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == W_MMA) tmem_alloc2(tmem_base, 512);
    pdl_wait();
    const Table tab(base + L::OFF_TAB);
    tab.fill(p, NT);
    fence_before_sync();
    __syncthreads();
    cluster_sync();
    fence_after_sync();
    const uint32_t tm = *tmem_base;
    Walk walk{tab, p.E, nn, (int)(gridDim.x / 2), 0, (long long)(blockIdx.x / 2)};
    Tile t;

    if (warp == W_PROD) {
        int gs = 0;
        bool ok = true;
        // Narrow tiles read most weights once, wide ones several times: evict-first took 1536 rows
        // over 64 experts of 2048 x 1024 from 41.0 to 38.9 us and cost wide tiles 6 %.
        const uint64_t pol = policy_evict_first();
        while (ok && walk.next(t)) {
            // The pair's rows of the tile, half each; columns behind the tile's last row hold what
            // the stage held before and are not stored.
            const int half = t.width / 2, mine = rows_held(t, half, rank, p.gather);
            const uint32_t bytes = 2 * ABYTES + 128 * (rows_held(t, half, 0, p.gather) + rows_held(t, half, 1, p.gather));
            int src[4];
            if (p.gather) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    bool valid;
                    src[j] = source_row(p, t.r0 + min(half * rank + 4 * lane + j, t.nrow - 1), valid);
                }
            }
            for (int ks = 0; ks < nks; ++ks, ++gs) {
                const int st = gs % STAGES;
                if (gs >= STAGES) ok = twait(empty + st, (gs / STAGES - 1) & 1, abort, p.limit);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                uint8_t *dst = base + st * STAGE;
                const uint32_t fb = leader_addr(full + st);
                if (lane == 0) {
                    if (rank == 0) mbar_arrive_expect_tx(full + st, bytes);
                    if constexpr (NT == 256) tma_load2(dst, &p.tmW, ks * 128, t.e * p.N + t.n0 + 128 * rank, fb);
                    else tma_load2_hint(dst, &p.tmW, ks * 128, t.e * p.N + t.n0 + 128 * rank, fb, pol);
                }
                __syncwarp();
                if (p.gather) {
                    if (4 * lane < mine)
                        tma_gather4(dst + ABYTES + lane * 512, &p.tmA[0], ks * 128, make_int4(src[0], src[1], src[2], src[3]), fb);
                } else if (lane < 4 && mine & 128 >> lane) {
                    // a sum of boxes, one a lane: a copy costs the TMA unit about as much whatever its
                    // height (boxes of 16 rows alone took 1.46 times as long for one expert of
                    // 16384 rows, 4096 x 4096)
                    const int at = mine & ~(0xff >> lane);
                    tma_load2(dst + ABYTES + at * 128, &p.tmA[lane], ks * 128, t.r0 + half * rank + at, fb);
                }
            }
        }
        // The last stages' releases arrive from the leader: none may find this CTA gone.
        for (int u = max(0, gs - STAGES); ok && u < gs; ++u) ok = twait(empty + u % STAGES, (u / STAGES) & 1, abort, p.limit);
        if (*abort) {
            // The copies issued must land before the CTA's memory goes.  A pair that gave up in
            // different places has no barrier to tell, so both wait some milliseconds.
            const long long t0 = clock64();
            while (clock64() - t0 < 8000000) {}
        }
    } else if (warp == W_MMA) {
        // The whole warp walks the loop and one elected lane issues, so that descriptors stay in
        // uniform registers (a loop run by one lane alone moves every operand there by itself:
        // 850 cycles per K step, more than its product takes).
        if (rank == 0) {
            const bool leader = elect_one();
            const uint64_t ad0 = smem_desc_sw128(base), bd0 = smem_desc_sw128(base + ABYTES);
            int st = 0, sg = 0, acc = 0;      // stage, group of scales, accumulator
            uint32_t phase = 0, aphase = 1;   // (a fresh barrier passes a wait for the phase before)
            bool ok = true;
            while (ok && walk.next(t)) {
                const int width = __shfl_sync(0xffffffffu, t.width, 0);
                if (E8) ok = twait(acc_free + acc, aphase, abort, p.limit);
                if (!__all_sync(0xffffffffu, ok)) break;
                for (int ks = 0; ks < nks; ++ks) {
                    const int g = ks % SGRP, b = sg & 1;
                    if (E8) {
                        if (g == 0) ok = twait(sf_full + b, (sg / 2) & 1, abort, p.limit);
                    } else {
                        ok = twait(acc_free + acc, aphase, abort, p.limit);
                    }
                    ok = ok && twait(full + st, phase, abort, p.limit);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    fence_after_sync();
                    if (leader) {
                        const uint64_t ad = ad0 + st * (STAGE / 16), bd = bd0 + st * (STAGE / 16);
                        if (E8) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                mma_mx(tm + NT * acc, ad + 2 * j, bd + 2 * j, idesc_mx(width, j), tm + COL_SFA + 4 * (SGRP * b + g),
                                       tm + COL_SFB + L::SFB * (SGRP * b + g), (ks | j) != 0);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) mma_f8(tm + NT * acc, ad + 2 * j, bd + 2 * j, idesc_f8(width), j != 0);
                        }
                        commit2(empty + st);
                        if (!E8) commit2(acc_ready + acc);
                        if (E8 && (g == SGRP - 1 || ks == nks - 1)) commit2(sf_empty + b);
                    }
                    __syncwarp();
                    if (g == SGRP - 1 || ks == nks - 1) ++sg;
                    if (++st == STAGES) { st = 0; phase ^= 1; }
                    if (!E8 && ++acc == NACC) { acc = 0; aphase ^= 1; }
                }
                if (E8) {
                    if (ok && leader) commit2(acc_ready + acc);
                    __syncwarp();
                    if (++acc == NACC) { acc = 0; aphase ^= 1; }
                }
            }
            if (leader) commit2(fin, 1);  // TMEM and the peer's operands go only when every MMA is done,
            wf_wait(fin, 0, &g_err);      // also when the CTA gives up (twait would return at once)
        }
    } else if (warp < L::SCALE0) {
        // (no role)
    } else if (warp < L::WORK0) {
        if constexpr (E8) {
            // Scale factors into TMEM.  Every lane quadrant holds all of them, so each warp writes
            // its own copy; the global loads are shared through shared memory.
            uint2 *sb = reinterpret_cast<uint2 *>(base + L::OFF_S);
            const int i = threadIdx.x - 32 * L::SCALE0;  // this thread loads tokens i and i + 128
            const uint32_t lanes = tm + ((uint32_t)(32 * (warp & 3)) << 16);
            const uint8_t *as = (const uint8_t *)p.a_s, *ws = (const uint8_t *)p.w_s;
            const bool wide = nks % 8 == 0 && reinterpret_cast<uintptr_t>(as) % 8 == 0;
            int sg = 0;
            bool ok = true;
            while (ok && walk.next(t)) {
                size_t ai[(NT + 127) / 128];
#pragma unroll
                for (int h = 0; h < (NT + 127) / 128; ++h) {
                    bool valid;
                    ai[h] = (size_t)source_row(p, t.r0 + min(i + 128 * h, t.nrow - 1), valid) * nks;
                }
                // the second CTA's rows may lie past N: any scale does, nothing of them is stored
                const size_t wi = ((size_t)t.e * nb + min(t.n0 / 128 + rank, nb - 1)) * nks;
                for (int k0 = 0; k0 < nks; k0 += SGRP, ++sg) {
                    const int b = sg & 1;
#pragma unroll
                    for (int h = 0; h < (NT + 127) / 128; ++h) {
                        if (i + 128 * h >= t.width) break;
                        uint2 v = make_uint2(0, 0);
                        if (wide) {
                            v = __ldg(reinterpret_cast<const uint2 *>(as + ai[h] + k0));
                        } else {
#pragma unroll
                            for (int g = 0; g < SGRP; ++g)
                                if (k0 + g < nks) (g < 4 ? v.x : v.y) |= (uint32_t)__ldg(as + ai[h] + k0 + g) << (8 * (g & 3));
                        }
                        sb[b * NT + 128 * h + i] = v;
                    }
                    uint32_t wb[SGRP];
#pragma unroll
                    for (int g = 0; g < SGRP; ++g) wb[g] = k0 + g < nks ? __ldg(ws + wi + k0 + g) * 0x01010101u : 0u;
                    if (sg >= 2) ok = twait(sf_empty + b, (sg / 2 - 1) & 1, abort, p.limit);
                    ok = bar_all(1, 32 * L::SCALERS, ok);  // the warps agree: none is left at a barrier
                    if (!ok) break;
                    fence_after_sync();
                    uint2 v[NT / 32];
#pragma unroll
                    for (int c = 0; c < NT / 32; ++c) v[c] = sb[b * NT + 32 * c + lane];
#pragma unroll
                    for (int g = 0; g < SGRP; ++g) {
                        if (k0 + g >= nks) break;
                        uint32_t f[NT / 32];
#pragma unroll
                        for (int c = 0; c < NT / 32; ++c) f[c] = __byte_perm(g < 4 ? v[c].x : v[c].y, 0, 0x1111 * (g & 3));
                        if constexpr (NT == 256) tmem_st8(lanes + COL_SFB + L::SFB * (SGRP * b + g), f);
                        else tmem_st4(lanes + COL_SFB + L::SFB * (SGRP * b + g), f[0], f[1], f[0], f[1]);
                        tmem_st4(lanes + COL_SFA + 4 * (SGRP * b + g), wb[g], wb[g], wb[g], wb[g]);
                    }
                    tmem_wait_st();
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) arrive_at(leader_addr(sf_full + b));
                }
            }
            for (int u = max(0, sg - 2); ok && u < sg; ++u) ok = twait(sf_empty + (u & 1), (u / 2) & 1, abort, p.limit);
        } else {
            // token scale x weight scale of each K step into shared memory
            float *sa = reinterpret_cast<float *>(base + L::OFF_S);
            const int i = threadIdx.x - 32 * L::SCALE0;  // this thread: tokens i, i + 64, ...
            int sg = 0;
            bool ok = true;
            while (ok && walk.next(t)) {
                size_t ai[NT / 64];
#pragma unroll
                for (int h = 0; h < NT / 64; ++h) {
                    bool valid;
                    ai[h] = (size_t)source_row(p, t.r0 + min(i + 64 * h, t.nrow - 1), valid) * nks;
                }
                const size_t wi = ((size_t)t.e * nb + min(t.n0 / 128 + rank, nb - 1)) * nks;
                for (int k0 = 0; k0 < nks; k0 += SGRP, ++sg) {
                    const int b = sg & 1;
                    if (sg >= 2) ok = twait(sf_empty + b, (sg / 2 - 1) & 1, abort, p.limit);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    // all loads of the group before the first use: one trip to memory, not one per step
                    float w[SGRP], v[NT / 64][SGRP];
#pragma unroll
                    for (int g = 0; g < SGRP; ++g) {
                        const int k = min(k0 + g, nks - 1);
                        w[g] = scale_at(p.w_s, p.w_f32, wi + k);
#pragma unroll
                        for (int h = 0; h < NT / 64; ++h) v[h][g] = 64 * h < t.width ? scale_at(p.a_s, p.a_f32, ai[h] + k) : 0.f;
                    }
#pragma unroll
                    for (int g = 0; g < SGRP; ++g)
#pragma unroll
                        for (int h = 0; h < NT / 64; ++h)
                            if (64 * h < t.width) sa[(b * SGRP + g) * NT + i + 64 * h] = v[h][g] * w[g];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sf_full + b);
                }
            }
        }
    } else {
        // workers: warp (q, half) takes the 32 weight rows of TMEM lane quadrant q and half of the
        // widest tile's tokens
        const int q = warp & 3, half = (warp - L::WORK0) >> 2;
        const uint32_t col = tm + ((uint32_t)(32 * q) << 16) + HALF * half;
        const float *sa = reinterpret_cast<const float *>(base + L::OFF_S) + HALF * half;
        int sg = 0, acc = 0;
        uint32_t aphase = 0;
        bool ok = true;
        while (ok && walk.next(t)) {
            const int mine = min(t.nrow - HALF * half, HALF);  // tokens of this warp that are stored
            uint32_t keep[HALF / 32];  // those whose row of `a` exists; the others' results are zero
#pragma unroll
            for (int c = 0; c < HALF / 32; ++c) {
                bool valid = true;
                if (32 * c + lane < mine) source_row(p, t.r0 + HALF * half + 32 * c + lane, valid);
                keep[c] = __ballot_sync(0xffffffffu, valid);
            }
            const int n = t.n0 + 128 * rank + 32 * q + lane;
            __nv_bfloat16 *o = p.out + (size_t)(t.r0 + HALF * half) * p.N + n;
            if constexpr (E8) {
                ok = twait(acc_ready + acc, aphase, abort, p.limit);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                fence_after_sync();
                __nv_bfloat162 y[HALF / 2];
#pragma unroll
                for (int c = 0; c < HALF / 32; ++c) {
                    if (HALF * half + 32 * c >= t.width) break;
                    uint32_t v[32];
                    tmem_ld32(col + NT * acc + 32 * c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        y[16 * c + j] = __floats2bfloat162_rn(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                }
                fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive_at(leader_addr(acc_free + acc));
                if (++acc == NACC) { acc = 0; aphase ^= 1; }
                if (n < p.N) {
#pragma unroll
                    for (int j = 0; j < HALF; ++j)
                        if (j < mine)
                            o[(size_t)j * p.N] = !(keep[j / 32] >> (j % 32) & 1) ? __float2bfloat16_rn(0.f)
                                                 : j & 1                        ? __high2bfloat16(y[j / 2])
                                                                                : __low2bfloat16(y[j / 2]);
                }
            } else {
                float sum[HALF];
#pragma unroll
                for (int j = 0; j < HALF; ++j) sum[j] = 0.f;
                for (int ks = 0; ks < nks; ++ks) {
                    const int g = ks % SGRP, b = sg & 1;
                    if (g == 0) ok = twait(sf_full + b, (sg / 2) & 1, abort, p.limit);
                    ok = ok && twait(acc_ready + acc, aphase, abort, p.limit);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    fence_after_sync();
                    const float *s = sa + (b * SGRP + g) * NT;
#pragma unroll
                    for (int c = 0; c < HALF / 32; ++c) {
                        if (HALF * half + 32 * c < t.width) {
                            uint32_t v[32];
                            tmem_ld32(col + NT * acc + 32 * c, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                const float4 f = *reinterpret_cast<const float4 *>(s + 32 * c + j);
                                sum[32 * c + j] += f.x * __uint_as_float(v[j]);
                                sum[32 * c + j + 1] += f.y * __uint_as_float(v[j + 1]);
                                sum[32 * c + j + 2] += f.z * __uint_as_float(v[j + 2]);
                                sum[32 * c + j + 3] += f.w * __uint_as_float(v[j + 3]);
                            }
                        }
                    }
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        arrive_at(leader_addr(acc_free + acc));
                        if (g == SGRP - 1 || ks == nks - 1) mbar_arrive(sf_empty + b);
                    }
                    if (g == SGRP - 1 || ks == nks - 1) ++sg;
                    if (++acc == NACC) { acc = 0; aphase ^= 1; }
                }
                if (!ok) break;
                if (n < p.N) {
#pragma unroll
                    for (int j = 0; j < HALF; ++j)
                        if (j < mine) o[(size_t)j * p.N] = __float2bfloat16_rn(keep[j / 32] >> (j % 32) & 1 ? sum[j] : 0.f);
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    cluster_sync();  // the pair's operands, barriers and TMEM are read by both
    if (warp == W_MMA) {
        fence_after_sync();
        tmem_dealloc2(tm, 512);
    }
}

// ---------------------------------------------------------------------------
// f32 scales, many rows per expert: 128 tokens x 256 weight rows a tile, one CTA each
// ---------------------------------------------------------------------------
namespace wide {
constexpr int MT = 128, NW = 256, STAGES = 4, ABYTES = MT * 128, STAGE = ABYTES + NW * 128;
constexpr int W_WORK0 = 4, THREADS = 32 * (W_WORK0 + WORKERS);
constexpr int NBAR = 2 * STAGES + 5;
constexpr int OFF_TAB = STAGES * STAGE, OFF_BAR = OFF_TAB + TAB_BYTES, SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
static_assert(SMEM <= SMEM_MAX && OFF_BAR % 8 == 0, "shared memory");
// Registers: a worker holds 128 sums and 64 loaded products; the split of what the block was
// launched with (REGS a thread, checked before the first launch) must not ask for more.
constexpr int REGS = 168;
static_assert(256 * 216 + 128 * 72 <= THREADS * REGS, "register split");

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
    // f32 += e4m3 x e4m3, M = 128, N = 256, both operands K-major
    constexpr uint32_t idesc = 1u << 4 | (NW >> 3) << 17 | (MT >> 4) << 24;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&v)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,"
        "%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]), "=r"(v[32]),
          "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]), "=r"(v[40]),
          "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]), "=r"(v[48]),
          "=r"(v[49]), "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]), "=r"(v[56]),
          "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
        : "r"(taddr)
        : "memory");
}
// (d0, d1) += s * (a, b), two 32-bit operations in one instruction
__device__ __forceinline__ void fma2(float &d0, float &d1, float s, uint32_t a, uint32_t b) {
    asm("{\n\t.reg .b64 d, s, v;\n\t"
        "mov.b64 d, {%0, %1};\n\tmov.b64 s, {%2, %2};\n\tmov.b64 v, {%3, %4};\n\t"
        "fma.rn.f32x2 d, s, v, d;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "+f"(d0), "+f"(d1)
        : "f"(s), "r"(a), "r"(b));
}
}  // namespace wide

__global__ void __launch_bounds__(wide::THREADS, 1) k_grouped_f32_wide(const __grid_constant__ Args p) {
    using namespace wide;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bar = reinterpret_cast<uint64_t *>(base + OFF_BAR);
    uint64_t *full = bar, *empty = bar + STAGES, *acc_ready = empty + STAGES, *acc_free = acc_ready + 2, *fin = acc_free + 2;
    uint32_t *tmem_base = reinterpret_cast<uint32_t *>(bar + NBAR);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_base + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int nks = p.K / 128, nn = (p.N + NW - 1) / NW, nb = (p.N + 127) / 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
        for (int j = 0; j < 2; ++j) { mbar_init(acc_ready + j, 1); mbar_init(acc_free + j, WORKERS); }
        mbar_init(fin, 1);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == W_MMA) { tmem_alloc(tmem_base, 512); tmem_relinquish(); }
    pdl_wait();
    const Table tab(base + OFF_TAB);
    tab.fill(p, MT);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tm = *tmem_base;
    Walk walk{tab, p.E, nn, (int)gridDim.x, 0, (long long)blockIdx.x};
    Tile t;

    if (warp < W_WORK0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == W_PROD) {
            int gs = 0;
            bool ok = true;
            while (ok && walk.next(t, MT)) {
                const int mine = (t.nrow + 15) & ~15;  // rows loaded; lanes behind the last row are not stored
                for (int ks = 0; ks < nks; ++ks, ++gs) {
                    const int st = gs % STAGES;
                    if (gs >= STAGES) ok = twait(empty + st, (gs / STAGES - 1) & 1, abort, p.limit);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    uint8_t *dst = base + st * STAGE;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(full + st, NW * 128 + mine * 128);
                        tma_load_2d(dst + ABYTES, &p.tmW, ks * 128, t.e * p.N + t.n0, full + st);
                        tma_load_2d(dst + ABYTES + 128 * 128, &p.tmW, ks * 128, t.e * p.N + t.n0 + 128, full + st);
                    }
                    __syncwarp();
                    if (lane < 4 && mine & 128 >> lane) {
                        const int at = mine & ~(0xff >> lane);
                        tma_load_2d(dst + at * 128, &p.tmA[lane], ks * 128, t.r0 + at, full + st);
                    }
                }
            }
            // The copies issued must land before the CTA's memory goes, whoever gives up and whenever:
            // a role whose wait runs out after this one has left its loop ends the CTA all the same.
            for (int u = max(0, gs - STAGES); u < gs; ++u) wf_wait(full + u % STAGES, (u / STAGES) & 1, &g_err);
        } else if (warp == W_MMA) {
            const bool leader = elect_one();
            const uint64_t ad0 = smem_desc_sw128(base), bd0 = smem_desc_sw128(base + ABYTES);
            int st = 0, acc = 0;
            uint32_t phase = 0, aphase = 1;
            bool ok = true;
            while (ok && walk.next(t, MT)) {
                for (int ks = 0; ks < nks; ++ks) {
                    ok = twait(acc_free + acc, aphase, abort, p.limit) && twait(full + st, phase, abort, p.limit);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    fence_after_sync();
                    if (leader) {
                        const uint64_t ad = ad0 + st * (STAGE / 16), bd = bd0 + st * (STAGE / 16);
#pragma unroll
                        for (int j = 0; j < 4; ++j) mma(tm + NW * acc, ad + 2 * j, bd + 2 * j, j != 0);
                        commit(empty + st);
                        commit(acc_ready + acc);
                    }
                    __syncwarp();
                    if (++st == STAGES) { st = 0; phase ^= 1; }
                    acc ^= 1;
                    if (!acc) aphase ^= 1;
                }
            }
            if (leader) commit(fin);  // TMEM goes only when every MMA is done,
            wf_wait(fin, 0, &g_err);  // also when the CTA gives up (twait would return at once)
        }
    } else {
        // worker (q, half): the 32 tokens of TMEM lane quadrant q, 128 weight rows (one block of scales)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int q = warp & 3, half = (warp - W_WORK0) >> 2;
        const uint32_t col = tm + ((uint32_t)(32 * q) << 16) + 128 * half;
        int acc = 0;
        uint32_t aphase = 0;
        bool ok = true;
        while (ok && walk.next(t, MT)) {
            const int row = 32 * q + lane;
            bool valid;
            const size_t ai = (size_t)source_row(p, t.r0 + min(row, t.nrow - 1), valid) * nks;
            // the second block may lie past N: any scale does, nothing of it is stored
            const size_t wi = ((size_t)t.e * nb + min(t.n0 / 128 + half, nb - 1)) * nks;
            float sum[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) sum[j] = 0.f;
            float next = scale_at(p.a_s, p.a_f32, ai) * scale_at(p.w_s, p.w_f32, wi);
            for (int ks = 0; ks < nks; ++ks) {
                const float s = next;
                const int k1 = min(ks + 1, nks - 1);  // the next step's scale is on its way during this one
                const float an = scale_at(p.a_s, p.a_f32, ai + k1), wn = scale_at(p.w_s, p.w_f32, wi + k1);
                ok = twait(acc_ready + acc, aphase, abort, p.limit);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                fence_after_sync();
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t v[64];
                    tmem_ld64(col + NW * acc + 64 * c, v);
                    tmem_wait_ld();
                    if (c == 1) {
                        fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(acc_free + acc);
                    }
#pragma unroll
                    for (int j = 0; j < 64; j += 2) fma2(sum[64 * c + j], sum[64 * c + j + 1], s, v[j], v[j + 1]);
                }
                next = an * wn;
                acc ^= 1;
                if (!acc) aphase ^= 1;
            }
            if (!ok) break;
            if (row < t.nrow) {
                const int n0 = t.n0 + 128 * half;
                uint4 *o = reinterpret_cast<uint4 *>(p.out + (size_t)(t.r0 + row) * p.N + n0);
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    if (n0 + 8 * c >= p.N) break;
                    uint32_t y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(valid ? sum[8 * c + 2 * j] : 0.f, valid ? sum[8 * c + 2 * j + 1] : 0.f);
                        y[j] = *reinterpret_cast<const uint32_t *>(&b);
                    }
                    o[c] = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == W_MMA) {
        fence_after_sync();
        tmem_dealloc(tm, 512);
    }
}

// The listed rows of a in the product's order (rows that do not exist: row 0, their results are zeroed).
// A warp per row, eight 16-byte pieces a lane in flight.
constexpr int PACK_WARPS = 8;
__global__ void __launch_bounds__(32 * PACK_WARPS) k_pack_rows(const uint4 *a, const int *rows, const int *offsets, uint4 *out,
                                                               int E, int M, int R, int chunks) {
    pdl_wait();
    pdl_launch_dependents();
    // rows behind the last expert's are left out; the offsets need not rise
    int end = 0;
    for (int e = threadIdx.x; e <= E; e += 32 * PACK_WARPS) end = max(end, __ldg(offsets + e));
    __shared__ int ends[PACK_WARPS];
    end = __reduce_max_sync(0xffffffffu, end);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) ends[warp] = end;
    const long long r0 = (long long)blockIdx.x * PACK_WARPS + warp, step = (long long)gridDim.x * PACK_WARPS;
    int s = r0 < R ? __ldg(rows + r0) : 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PACK_WARPS; ++w) end = max(end, ends[w]);
    end = min(end, R);
    for (long long r = r0; r < end; r += step) {
        const uint4 *src = a + (size_t)(s >= 0 && s < M ? s : 0) * chunks;
        uint4 *dst = out + r * chunks;
        if (r + step < end) s = __ldg(rows + r + step);
        for (int c0 = lane; c0 < chunks; c0 += 256) {
            uint4 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + 32 * j < chunks) v[j] = __ldg(src + c0 + 32 * j);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + 32 * j < chunks) dst[c0 + 32 * j] = v[j];
        }
    }
}

// Memory of a call: what it writes must lie apart from what its CTAs read at other times.
struct Span {
    const void *at;
    int64_t bytes;
    bool meets(const Span &o) const {
        const uintptr_t x = (uintptr_t)at, y = (uintptr_t)o.at;
        return bytes > 0 && o.bytes > 0 && x < y + (uintptr_t)o.bytes && y < x + (uintptr_t)bytes;
    }
};

int tensor_map(CUtensorMap *m, const void *base, uint64_t rows, uint64_t K, uint32_t box_rows) {
    host::EncodeTiledFn enc = host::encode_fn();
    if (!enc) return host::fail(WF_E_CUDA, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[2] = {K, rows}, strides[1] = {K};
    const cuuint32_t box[2] = {128, box_rows}, estr[2] = {1, 1};
    if (enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return host::fail(WF_E_SHAPE, "cuTensorMapEncodeTiled failed");
    return WF_OK;
}

// `kernel` with `ctas` CTAs for each of the units of work that fit the device, at most one per tile of
// `nt` rows x 256 weight rows.
template <void (*kernel)(const Args)>
cudaError_t launch(const Args &p, int ctas, int nt, int threads, int smem, int sms, cudaStream_t st, int regs = 0) {
    static std::atomic<uint64_t> ready[64];
    cudaError_t e = host::allow_smem((const void *)kernel, 0, smem, ready);
    if (e != cudaSuccess) return e;
    if (regs) {  // a register split of more than the block is launched with would wait for ever
        static const cudaFuncAttributes attr = [] {
            cudaFuncAttributes a = {};
            if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess) a.numRegs = 0;
            return a;
        }();
        if (attr.numRegs < regs) return cudaErrorInvalidConfiguration;
    }
    const int64_t tiles = ((int64_t)p.R / nt + (p.E < p.R ? p.E : p.R)) * ((p.N + 255) / 256), most = sms / ctas;
    return host::launch_pdl(kernel, dim3(ctas * (unsigned)(tiles < most ? tiles : most)), threads, smem, st, p);
}
template <bool E8, int NT>
cudaError_t launch_pairs(const Args &p, int sms, cudaStream_t st) {
    return launch<k_grouped_fp8<E8, NT>>(p, 2, NT, Plan<E8, NT>::THREADS, Plan<E8, NT>::SMEM, sms, st);
}

}  // namespace grp
}  // namespace wf

using wf::host::cuda_fail;
using wf::host::fail;

extern "C" {

size_t wf_grouped_fp8_workspace_bytes(int32_t row_list, int64_t R, int32_t E, int64_t K) {
    if (R <= 0 || R > (1 << 30) || E <= 0 || E > wf::grp::MAX_E || K <= 0 || K > (1 << 20)) return 0;
    return row_list && R > (int64_t)E * wf::grp::GATHER ? (size_t)R * K : 0;
}

int wf_grouped_fp8_gemm(const void *a, const void *a_s, int32_t a_scale_kind, const void *w, const void *w_s,
                        int32_t w_scale_kind, const int32_t *offsets, const int32_t *rows, int64_t M, int64_t R,
                        int32_t E, int64_t N, int64_t K, void *out, void *workspace,
                        size_t workspace_bytes, void *stream) {
    if (!a || !a_s || !w || !w_s || !offsets || !out) return fail(WF_E_ARG, "null pointer");
    if (a_scale_kind < 0 || a_scale_kind > 1 || w_scale_kind < 0 || w_scale_kind > 1) return fail(WF_E_DTYPE, "bad scale kind");
    if (M <= 0 || M > (1 << 30) || R <= 0 || R > (1 << 30)) return fail(WF_E_SHAPE, "M and R must be in 1..2^30");
    if (!rows && R > M) return fail(WF_E_SHAPE, "R exceeds the M rows of a (no row list)");
    if (E <= 0 || E > wf::grp::MAX_E) return fail(WF_E_SHAPE, "E must be in 1..512");
    if (N <= 0 || N % 8 || N > (1 << 20) || E * N > (1 << 30)) return fail(WF_E_SHAPE, "N must be a multiple of 8, E * N at most 2^30");
    if (K <= 0 || K % 128 || K > (1 << 20)) return fail(WF_E_SHAPE, "K must be a positive multiple of 128, at most 2^20");
    if ((uintptr_t)a % 16 || (uintptr_t)w % 16 || (uintptr_t)out % 16 || (uintptr_t)offsets % 4 || (uintptr_t)rows % 4 ||
        (a_scale_kind == WF_SCALE_F32 && (uintptr_t)a_s % 4) || (w_scale_kind == WF_SCALE_F32 && (uintptr_t)w_s % 4))
        return fail(WF_E_ARG, "a, w and out must be 16-byte aligned, f32 scales and row lists 4-byte");
    wf::grp::Args p;
    const bool pack = rows && R > (int64_t)E * wf::grp::GATHER;
    if (pack) {
        if (!workspace || workspace_bytes < (size_t)R * K) return fail(WF_E_ARG, "workspace too small (see wf_grouped_fp8_workspace_bytes)");
        if ((uintptr_t)workspace % 16) return fail(WF_E_ARG, "workspace must be 16-byte aligned");
    }
    const int64_t nks = K / 128, a_sb = a_scale_kind == WF_SCALE_F32 ? 4 : 1, w_sb = w_scale_kind == WF_SCALE_F32 ? 4 : 1;
    const wf::grp::Span in[] = {{a, M * K},      {a_s, M * nks * a_sb},    {w, E * N * K}, {w_s, E * ((N + 127) / 128) * nks * w_sb},
                                {offsets, (E + 1) * 4}, {rows, rows ? R * 4 : 0}};
    const wf::grp::Span y = {out, R * N * 2}, ws = {workspace, pack ? R * K : 0};
    for (const wf::grp::Span &x : in)
        if (x.meets(y) || x.meets(ws)) return fail(WF_E_ARG, "out or the workspace overlaps an input");
    if (y.meets(ws)) return fail(WF_E_ARG, "out overlaps the workspace");
    p.gather = rows && !pack;
    int rc = wf::grp::tensor_map(&p.tmW, w, (uint64_t)E * N, K, 128);
    if (p.gather) {
        if (!rc) rc = wf::grp::tensor_map(&p.tmA[0], a, M, K, 1);
        for (int j = 1; j < 4; ++j) p.tmA[j] = p.tmA[0];
    } else {
        for (int j = 0; j < 4 && !rc; ++j) rc = wf::grp::tensor_map(&p.tmA[j], pack ? workspace : a, pack ? R : M, K, 128 >> j);
    }
    if (rc) return rc;
    p.a_s = a_s; p.w_s = w_s; p.offsets = offsets; p.rows = rows; p.out = (__nv_bfloat16 *)out;
    p.limit.cycles = wf::host::wait_limit();
    p.limit.poll = p.limit.cycles < wf::kWaitLimitCycles;
    p.M = (int)M; p.R = (int)R; p.E = E; p.N = (int)N; p.K = (int)K;
    p.a_f32 = a_scale_kind == WF_SCALE_F32; p.w_f32 = w_scale_kind == WF_SCALE_F32;
    const int sms = wf::host::sm_count();
    if (sms <= 0) return fail(WF_E_CUDA, "no CUDA device");
    const bool e8 = !p.a_f32 && !p.w_f32, few = R <= (int64_t)E * (e8 ? wf::grp::NARROW_E8 : wf::grp::NARROW_F32);
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = cudaSuccess;
    if (pack) {
        const int64_t ctas = (R + wf::grp::PACK_WARPS - 1) / wf::grp::PACK_WARPS, most = 16 * (int64_t)sms;
        e = wf::host::launch_pdl(wf::grp::k_pack_rows, dim3((unsigned)(ctas < most ? ctas : most)), 32 * wf::grp::PACK_WARPS, 0,
                                 st, (const uint4 *)a, rows, offsets, (uint4 *)workspace, (int)E, (int)M, (int)R,
                                 (int)(K / 16));
    }
    if (e == cudaSuccess)
        e = few ? (e8 ? wf::grp::launch_pairs<true, 64>(p, sms, st) : wf::grp::launch_pairs<false, 64>(p, sms, st))
            : e8 ? wf::grp::launch_pairs<true, 256>(p, sms, st)
                 : wf::grp::launch<wf::grp::k_grouped_f32_wide>(p, 1, wf::grp::wide::MT, wf::grp::wide::THREADS,
                                                                wf::grp::wide::SMEM, sms, st, wf::grp::wide::REGS);
    return e == cudaSuccess ? WF_OK : cuda_fail(e, "grouped_fp8_gemm launch");
}

int wf_grouped_read_error(void *stream) {
    int err = 0;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&err, wf::grp::g_err, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return cuda_fail(e, "read error word");
    if (!err) return WF_OK;
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(wf::grp::g_err, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return cuda_fail(e, "clear error word");
    return fail(WF_E_TIMEOUT, "a device wait timed out");
}

}  // extern "C"
