// wf_grouped_fp8.cu - the experts' block-scaled FP8 product on tcgen05.
//
//   out[r, n] = sum_k (a[row(r), k] * a_s[row(r), k/128]) * (w[e, n, k] * w_s[e, n/128, k/128])
//   for expert e and r in [offsets[e], offsets[e+1]), row(r) = rows[r] (or r)
//
// Weight rows are the M side of the MMA (128 per tile, exactly one block of weight
// scales), tokens the N side: an expert's rows are cut into tiles of equal width, a
// multiple of 16, so a few rows cost a few columns and nothing is padded to 128.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/wfb200.h"
#include "wf_host.h"
#include "wf_ptx.cuh"
#include "wf_tcgen05.cuh"

namespace wf {
namespace grp {

using namespace tc;

__device__ int g_err;  // error flags of the grouped products since the last wf_grouped_read_error

constexpr int MAX_E = 512;
constexpr int NT = 128;                 // tokens per tile, at most
constexpr int STAGES = 6;
constexpr int ABYTES = 128 * 128, BBYTES = NT * 128, STAGE = ABYTES + BBYTES;
constexpr int NACC = 4;                 // K-step accumulators in TMEM
constexpr int SGRP = 8;                 // K steps per group of scales
constexpr int W_PROD = 0, W_MMA = 1, W_SCALE0 = 2, W_WORK0 = 4, WORKERS = 8;
constexpr int THREADS = 32 * (W_WORK0 + WORKERS);
constexpr int NBAR = 2 * STAGES + 2 * NACC + 4 + 1;
constexpr int OFF_SA = STAGES * STAGE;                   // [2][SGRP][NT] f32
constexpr int OFF_LO = OFF_SA + 2 * SGRP * NT * 4;       // [MAX_E] first row
constexpr int OFF_CNT = OFF_LO + MAX_E * 4;              // [MAX_E] rows
constexpr int OFF_T = OFF_CNT + MAX_E * 4;               // [MAX_E + 1] first token tile
constexpr int OFF_MASK = OFF_T + (MAX_E + 4) * 4;        // [2][4] valid columns
constexpr int OFF_BAR = OFF_MASK + 32;
constexpr int SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
static_assert(SMEM <= 232448 && OFF_BAR % 8 == 0, "shared memory");

struct Args {
    CUtensorMap tmW, tmA;  // weights [E*N, K], box 128 x 128; tokens [M, K], box 128 x 1 (gather)
    const void *a_s, *w_s;
    const int *offsets, *rows;
    __nv_bfloat16 *out;
    long long limit;
    int M, R, E, N, K, a_f32, w_f32;
};

__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor of kind::f8f6f4: E4M3 x E4M3 -> f32, M = 128, both operands K-major.
__device__ __forceinline__ uint32_t idesc_f8(int n) {
    return 1u << 4 | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}

// Four rows of the tensor map, 128 bytes each, to 512 consecutive (swizzled) bytes.
__device__ __forceinline__ void tma_gather4(void *dst, const CUtensorMap *map, int c0, int4 r, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(smem_u32(bar))
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

struct Tile {
    int e, n0, r0, nrow, width;
};

// Tiles of this CTA in order: blockIdx.x, blockIdx.x + gridDim.x, ...; within an
// expert the weight tile runs fastest.
struct Walk {
    const int *lo, *cnt, *first;
    int E, nn, e;
    long long i;
    __device__ bool next(Tile &t) {
        while (e < E && i >= (long long)first[e + 1] * nn) ++e;
        if (e >= E) return false;
        const int local = (int)(i - (long long)first[e] * nn);
        const int nt = first[e + 1] - first[e], c = cnt[e];
        t.e = e;
        t.n0 = local % nn * 128;
        t.width = ((c + nt - 1) / nt + 15) / 16 * 16;
        const int j = local / nn * t.width;
        t.r0 = lo[e] + j;
        t.nrow = min(t.width, c - j);
        i += gridDim.x;
        return true;
    }
};

__device__ __forceinline__ bool twait(uint64_t *bar, uint32_t parity, volatile int *abort, long long limit) {
    if (*abort) return false;
    if (!wf_wait(bar, parity, &g_err, limit)) {
        *abort = 1;
        return false;
    }
    return true;
}
__device__ __forceinline__ float scale_at(const void *s, int f32, size_t i) {
    if (f32) return __ldg((const float *)s + i);
    const uint32_t b = __ldg((const uint8_t *)s + i);
    return b == 255 ? __uint_as_float(0x7fffffffu) : e8m0_to_f32(b);
}

__global__ void __launch_bounds__(THREADS, 1) k_grouped_f32(const __grid_constant__ Args p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bar = reinterpret_cast<uint64_t *>(base + OFF_BAR);
    uint64_t *full = bar, *empty = bar + STAGES, *acc_ready = empty + STAGES, *acc_free = acc_ready + NACC;
    uint64_t *sf_full = acc_free + NACC, *sf_empty = sf_full + 2, *fin = sf_empty + 2;
    uint32_t *tmem_base = reinterpret_cast<uint32_t *>(bar + NBAR);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_base + 1);
    float *sa = reinterpret_cast<float *>(base + OFF_SA);
    int *lo = reinterpret_cast<int *>(base + OFF_LO), *cnt = reinterpret_cast<int *>(base + OFF_CNT);
    int *first = reinterpret_cast<int *>(base + OFF_T);
    volatile uint32_t *mask = reinterpret_cast<volatile uint32_t *>(base + OFF_MASK);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nks = p.K / 128, nn = (p.N + 127) / 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
        for (int j = 0; j < NACC; ++j) { mbar_init(acc_ready + j, 1); mbar_init(acc_free + j, WORKERS); }
        for (int j = 0; j < 2; ++j) { mbar_init(sf_full + j, W_WORK0 - W_SCALE0); mbar_init(sf_empty + j, WORKERS); }
        mbar_init(fin, 1);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == W_MMA) { tmem_alloc(tmem_base, 512); tmem_relinquish(); }
    // every expert's rows, clamped to the R rows there are, and its first token tile
    for (int e = threadIdx.x; e < p.E; e += THREADS) {
        const int a = min(max(p.offsets[e], 0), p.R), b = min(max(p.offsets[e + 1], 0), p.R);
        lo[e] = a;
        cnt[e] = max(b - a, 0);
    }
    __syncthreads();
    if (warp == W_PROD) {
        int sum = 0, own[MAX_E / 32];
#pragma unroll
        for (int j = 0; j < MAX_E / 32; ++j) {
            const int e = lane * (MAX_E / 32) + j;
            own[j] = sum;
            if (e < p.E) sum += (cnt[e] + NT - 1) / NT;
        }
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
#pragma unroll
        for (int j = 0; j < MAX_E / 32; ++j) {
            const int e = lane * (MAX_E / 32) + j;
            if (e < p.E) first[e] = incl - sum + own[j];
        }
        if (lane == 31) first[p.E] = incl;
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tm = *tmem_base;
    Walk walk{lo, cnt, first, p.E, nn, 0, (long long)blockIdx.x};
    Tile t;

    if (warp == W_PROD) {
        int gs = 0;
        bool ok = true;
        while (ok && walk.next(t)) {
            int4 src = make_int4(0, 0, 0, 0);
            int *s4 = reinterpret_cast<int *>(&src);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = t.r0 + min(4 * lane + j, t.nrow - 1);
                s4[j] = min(max(p.rows ? __ldg(p.rows + r) : r, 0), p.M - 1);
            }
            for (int ks = 0; ks < nks; ++ks, ++gs) {
                const int st = gs % STAGES;
                if (gs >= STAGES) ok = twait(empty + st, (gs / STAGES - 1) & 1, abort, p.limit);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                uint8_t *dst = base + st * STAGE;
                if (lane == 0) {
                    mbar_arrive_expect_tx(full + st, ABYTES + t.width * 128);
                    tma_load_2d(dst, &p.tmW, ks * 128, t.e * p.N + t.n0, full + st);
                }
                __syncwarp();
                if (4 * lane < t.width) tma_gather4(dst + ABYTES + lane * 512, &p.tmA, ks * 128, src, full + st);
            }
        }
        if (*abort) {  // the copies issued must land before the CTA's memory goes
            for (int u = max(0, gs - STAGES); u < gs; ++u) wf_wait(full + u % STAGES, (u / STAGES) & 1, &g_err);
        }
    } else if (warp == W_MMA) {
        if (lane == 0) {
            int gs = 0;
            bool ok = true;
            while (ok && walk.next(t)) {
                const uint32_t id = idesc_f8(t.width);
                for (int ks = 0; ks < nks; ++ks, ++gs) {
                    const int st = gs % STAGES, ab = gs % NACC;
                    ok = gs < NACC || twait(acc_free + ab, (gs / NACC - 1) & 1, abort, p.limit);
                    ok = ok && twait(full + st, (gs / STAGES) & 1, abort, p.limit);
                    if (!ok) break;
                    fence_after_sync();
                    const uint64_t ad = smem_desc_sw128(base + st * STAGE), bd = smem_desc_sw128(base + st * STAGE + ABYTES);
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma_f8(tm + NT * ab, ad + 2 * j, bd + 2 * j, id, j != 0);
                    commit(empty + st);
                    commit(acc_ready + ab);
                }
            }
            commit(fin);  // TMEM goes only when every MMA is done
            wf_wait(fin, 0, &g_err);
        }
    } else if (warp < W_WORK0) {
        const int i = threadIdx.x - 32 * W_SCALE0;  // this thread: tokens i and i + 64 of the tile
        int sg = 0;
        bool ok = true;
        while (ok && walk.next(t)) {
            size_t ai[2];
            bool valid[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = t.r0 + min(i + 64 * h, t.nrow - 1);
                const int src = p.rows ? __ldg(p.rows + r) : r;
                valid[h] = src >= 0 && src < p.M;
                ai[h] = (size_t)(valid[h] ? src : 0) * nks;
            }
            const size_t wi = ((size_t)t.e * nn + t.n0 / 128) * nks;
            for (int k0 = 0; k0 < nks; k0 += SGRP, ++sg) {
                const int b = sg & 1;
                if (sg >= 2) ok = twait(sf_empty + b, (sg / 2 - 1) & 1, abort, p.limit);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
#pragma unroll
                for (int g = 0; g < SGRP; ++g)
                    if (k0 + g < nks) {
                        const float ws = scale_at(p.w_s, p.w_f32, wi + k0 + g);
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            sa[(b * SGRP + g) * NT + i + 64 * h] = scale_at(p.a_s, p.a_f32, ai[h] + k0 + g) * ws;
                    }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t m = __ballot_sync(0xffffffffu, valid[h]);
                    if (lane == 0) mask[4 * b + i / 32 + 2 * h] = m;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(sf_full + b);
            }
        }
    } else {
        const int q = warp & 3, half = (warp - W_WORK0) >> 2;
        const uint32_t col = tm + ((uint32_t)(32 * q) << 16) + 64 * half;
        int gs = 0, sg = 0;
        bool ok = true;
        while (ok && walk.next(t)) {
            float acc[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) acc[j] = 0.f;
            uint32_t m[2] = {0, 0};
            for (int ks = 0; ks < nks; ++ks, ++gs) {
                const int g = ks % SGRP, b = sg & 1, ab = gs % NACC;
                if (g == 0) {
                    ok = twait(sf_full + b, (sg / 2) & 1, abort, p.limit);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    m[0] = mask[4 * b + 2 * half];
                    m[1] = mask[4 * b + 2 * half + 1];
                }
                ok = twait(acc_ready + ab, (gs / NACC) & 1, abort, p.limit);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                fence_after_sync();
                const float *s = sa + (b * SGRP + g) * NT + 64 * half;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (64 * half + 32 * c < t.width) {
                        uint32_t v[32];
                        tmem_ld32(col + NT * ab + 32 * c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 f = *reinterpret_cast<const float4 *>(s + 32 * c + j);
                            acc[32 * c + j] += f.x * __uint_as_float(v[j]);
                            acc[32 * c + j + 1] += f.y * __uint_as_float(v[j + 1]);
                            acc[32 * c + j + 2] += f.z * __uint_as_float(v[j + 2]);
                            acc[32 * c + j + 3] += f.w * __uint_as_float(v[j + 3]);
                        }
                    }
                }
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_free + ab);
                if (g == SGRP - 1 || ks == nks - 1) {
                    if (lane == 0) mbar_arrive(sf_empty + b);
                    ++sg;
                }
            }
            if (!ok) break;
            const int n = t.n0 + 32 * q + lane;
            if (n < p.N) {
                __nv_bfloat16 *o = p.out + (size_t)(t.r0 + 64 * half) * p.N + n;
#pragma unroll
                for (int j = 0; j < 64; ++j)
                    if (64 * half + j < t.nrow)
                        o[(size_t)j * p.N] = __float2bfloat16_rn(m[j / 32] >> (j % 32) & 1 ? acc[j] : 0.f);
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

}  // namespace grp
}  // namespace wf

using wf::host::cuda_fail;
using wf::host::fail;

extern "C" {

int wf_grouped_fp8_gemm(const void *a, const void *a_s, int32_t a_scale_kind, const void *w, const void *w_s,
                        int32_t w_scale_kind, const int32_t *offsets, const int32_t *rows, int64_t M, int64_t R,
                        int32_t E, int64_t N, int64_t K, void *out, void *stream) {
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
    int rc = wf::grp::tensor_map(&p.tmW, w, (uint64_t)E * N, K, 128);
    if (!rc) rc = wf::grp::tensor_map(&p.tmA, a, M, K, 1);
    if (rc) return rc;
    p.a_s = a_s; p.w_s = w_s; p.offsets = offsets; p.rows = rows; p.out = (__nv_bfloat16 *)out;
    p.limit = wf::host::wait_limit();
    p.M = (int)M; p.R = (int)R; p.E = E; p.N = (int)N; p.K = (int)K;
    p.a_f32 = a_scale_kind == WF_SCALE_F32; p.w_f32 = w_scale_kind == WF_SCALE_F32;
    const int sms = wf::host::sm_count();
    if (sms <= 0) return fail(WF_E_CUDA, "no CUDA device");
    cudaError_t e = cudaFuncSetAttribute(wf::grp::k_grouped_f32, cudaFuncAttributeMaxDynamicSharedMemorySize, wf::grp::SMEM);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(grouped_fp8_gemm)");
    const int64_t tiles = (R / wf::grp::NT + (E < R ? E : R)) * ((N + 127) / 128);
    wf::grp::k_grouped_f32<<<(unsigned)(tiles < sms ? tiles : sms), wf::grp::THREADS, wf::grp::SMEM, (cudaStream_t)stream>>>(p);
    wf::host::counted();
    e = cudaGetLastError();
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
