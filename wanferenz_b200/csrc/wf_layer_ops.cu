// wf_layer_ops.cu - the operators between a layer's residual stream and its
// experts' products: RMS norm with the residual's addition and an E4M3 output,
// routing with groups, the expert dispatch lists, and the weighted combine.
//
// Each is bound by HBM for many tokens and by launch latency for few; none needs
// a workspace that outlives the call, and each writes the same bits for the same
// inputs (no floating-point atomics).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "../../include/wfb200.h"
#include "wf_host.h"
#include "wf_ptx.cuh"

namespace wf {
namespace lops {

using host::cuda_fail;
using host::fail;

__device__ __forceinline__ float2 bf2(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Two 32-bit operations in one instruction: (a0, a1) * (b0, b1) and + (c0, c1).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 r, a, b;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 r, a, b, c;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

// ---------------------------------------------------------------------------
// RMS norm + residual + E4M3 output
//   h = bf16(x + residual)          (the residual stream; x itself without one)
//   n = h * rsqrt(mean(h^2) + eps) * weight               (32 bits)
//   y = bf16(n)
//   per 128 columns: s = max(amax|n|, 1e-4) / 448, with ue8m0 rounded up to a
//   power of two; q = e4m3(n / s)
// The statistics are those of the rounded h, which is what the next layer reads
// back.  q is taken from the 32-bit n, not from y: one rounding fewer.
// A CTA walks over rows.  A thread copies its own 8-column chunks of the rows ahead into
// shared memory (cp.async, so no thread waits for another's copies), keeps a row in registers
// between the sum of squares and the output, and reads every input once.  A block of 128
// columns is 16 neighbouring lanes.
// Bound by HBM: 16384 x 4096 with residual and both outputs, 604 MB, takes 94 to 102 us, 6 TB/s
// (one CTA per row: 114 us; the next row in registers: 102 us, and 4.1 TB/s at D = 8192).  By
// instructions where q is the only output: 203 MB without residual take 60 us, 3.4 TB/s (e8m0
// scales 55 us, 3.7).
// ---------------------------------------------------------------------------
struct NormArgs {
    const uint4 *x, *res;
    const void *weight;
    uint4 *y, *h;
    uint2 *q;
    void *s;
    float eps, inv_d;
    int chunks;  // D / 8
    long long T;
    int weight_bf16, ue8m0, s_f32;
    int depth;   // rows of a CTA in flight, 2 or 3
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ void copy_ahead(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Waits until at most depth - 1 of this thread's groups of copies are in flight.
__device__ __forceinline__ void copies_left(int depth) {
    if (depth == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 2;" ::: "memory");
}

constexpr int NORM_THREADS = 512;  // at most

template <int CH>  // chunks per thread
__global__ void __launch_bounds__(NORM_THREADS, CH == 4 ? 1 : 2) k_rms_norm_quant(const __grid_constant__ NormArgs p) {
    extern __shared__ uint4 ahead[];  // [depth][x, residual][CH][threads]
    __shared__ __align__(16) float parts[2][NORM_THREADS / 32];
    const int nt = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slot_size = (p.res ? 2 : 1) * CH * nt;
    if (threadIdx.x < 2 * (NORM_THREADS / 32)) parts[0][threadIdx.x] = 0.f;  // warps that a narrow block does not have
    pdl_wait();
    float2 w[CH][4];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = threadIdx.x + i * nt;
        if (c >= p.chunks) continue;
        if (p.weight_bf16) {
            const uint4 a = __ldg((const uint4 *)p.weight + c);
            const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i][j] = bf2(u[j]);
        } else {
            const float4 a = __ldg((const float4 *)p.weight + 2 * c), b = __ldg((const float4 *)p.weight + 2 * c + 1);
            w[i][0] = make_float2(a.x, a.y); w[i][1] = make_float2(a.z, a.w);
            w[i][2] = make_float2(b.x, b.y); w[i][3] = make_float2(b.z, b.w);
        }
    }
    auto fetch = [&](long long t, int slot) {
        if (t < p.T) {
            uint4 *dst = ahead + slot * slot_size + threadIdx.x;
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int c = threadIdx.x + i * nt;
                if (c < p.chunks) {
                    copy_ahead(dst + i * nt, p.x + t * p.chunks + c);
                    if (p.res) copy_ahead(dst + (CH + i) * nt, p.res + t * p.chunks + c);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int d = 0; d + 1 < p.depth; ++d) fetch(blockIdx.x + (long long)d * gridDim.x, d);
    __syncthreads();
    int flip = 0, slot = 0;
    for (long long t = blockIdx.x; t < p.T; t += gridDim.x, flip ^= 1) {
        const size_t row = (size_t)t * p.chunks;
        float *part = parts[flip];
        const int last = slot == 0 ? p.depth - 1 : slot - 1;  // the slot that the row before this one left
        fetch(t + (long long)(p.depth - 1) * gridDim.x, last);
        copies_left(p.depth);
        const uint4 *src = ahead + slot * slot_size + threadIdx.x;
        if (++slot == p.depth) slot = 0;
        float2 v[CH][4], sq = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = threadIdx.x + i * nt;
            if (c < p.chunks) {
                const uint4 a = src[i * nt];
                const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = bf2(u[j]);
                if (p.res) {
                    const uint4 b = src[(CH + i) * nt];
                    const uint32_t r4[4] = {b.x, b.y, b.z, b.w};
                    uint32_t o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 f = bf2(r4[j]);
                        o[j] = pack_bf2(v[i][j].x + f.x, v[i][j].y + f.y);
                        v[i][j] = bf2(o[j]);
                    }
                    p.h[row + c] = make_uint4(o[0], o[1], o[2], o[3]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) sq = fma2(v[i][j], v[i][j], sq);
            }
        }
        float ss = sq.x + sq.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane == 0) part[warp] = ss;
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int j = 0; j < NORM_THREADS / 32; j += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(part + j);
            ss += (f.x + f.y) + (f.z + f.w);
        }
        const float rstd = rsqrtf(ss * p.inv_d + p.eps);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = threadIdx.x + i * nt;
            const bool on = c < p.chunks;  // whole groups of 16 lanes: chunks is a multiple of 16
            float amax = 0.f;
            if (on) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[i][j] = mul2(mul2(v[i][j], make_float2(rstd, rstd)), w[i][j]);
                    amax = max_nan(amax, max_nan(fabsf(v[i][j].x), fabsf(v[i][j].y)));
                }
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            if (!on) continue;
            // NaN passes through the maximum, so it reaches the scale as it does in n
            float s = max_nan(amax, 1e-4f) * (1.0f / 448.0f);
            uint32_t byte = 0;
            if (p.ue8m0) {
                const uint32_t b = __float_as_uint(s);
                byte = s < CUDART_INF_F ? (b + 0x7fffffu) >> 23 : 0xffu;
                s = byte < 0xffu ? __uint_as_float(byte << 23) : CUDART_NAN_F;
            }
            // n / s: exact by the reciprocal of a power of two (below 2^120, as n is finite).  Else
            // Markstein's division (IBM J. Res. Dev. 34, 1990): the product with the rounded reciprocal
            // plus the reciprocal times the remainder (0 for an infinite s) is the rounded quotient,
            // but for a significand of s that is all ones: a power of two over it comes out a step low.
            // That moves one q, n / s next above 2^-10 (to 0, not 2^-9); every other significand of s,
            // with the dividends nearest every e4m3 midpoint, was tried on the CPU.
            const float inv = !p.ue8m0 ? __frcp_rn(s) : byte < 0xffu ? __uint_as_float((254u - byte) << 23) : CUDART_NAN_F;
            float2 u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = mul2(v[i][j], make_float2(inv, inv));
            if (!p.ue8m0) {
                const float den = s < CUDART_INF_F ? -s : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    u[j] = fma2(fma2(u[j], make_float2(den, den), v[i][j]), make_float2(inv, inv), u[j]);
            }
            const uint32_t lo = f32x2_to_e4m3x2(u[0].x, u[0].y) | (uint32_t)f32x2_to_e4m3x2(u[1].x, u[1].y) << 16;
            const uint32_t hi = f32x2_to_e4m3x2(u[2].x, u[2].y) | (uint32_t)f32x2_to_e4m3x2(u[3].x, u[3].y) << 16;
            p.q[row + c] = make_uint2(lo, hi);
            if (p.y)
                p.y[row + c] = make_uint4(pack_bf2(v[i][0].x, v[i][0].y), pack_bf2(v[i][1].x, v[i][1].y),
                                          pack_bf2(v[i][2].x, v[i][2].y), pack_bf2(v[i][3].x, v[i][3].y));
            if ((lane & 15) == 0) {
                const size_t at = (row + c) >> 4;
                if (p.s_f32) ((float *)p.s)[at] = s;
                else ((uint8_t *)p.s)[at] = (uint8_t)byte;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Routing: scores, bias, groups, top-k, renormalised weights
//   s = f(logit), sel = s + bias; a group's value is the sum of its two largest
//   sel (or its largest); the topk_groups best groups stay; the k best sel of
//   theirs are the experts, in descending order; w = s / sum(s) * route_scale.
// Scores and sums are in 64 bits: the choice is discrete, and two experts whose
// 32-bit scores agree to the last bit must still come out in the order of their
// logits.  Equal values go to the lower index.  A logit (or biased score) of
// -infinity masks its expert: it is never chosen, and slots that find no expert
// get index -1 and weight 0.  NaN counts as the largest value, as in torch.topk,
// so it shows in the weights.
// One warp per token; a lane holds experts lane, lane + 32, ...  Scores of sigmoid and
// sqrt(softplus) are screened in 32 bits first (route32); rows whose choice 32 bits
// cannot settle, and softmax, take the 64-bit path (route64).  The chosen experts'
// weights are in 64 bits on both.
// Bound by instructions (1461 a token with 8 groups; the logits' bytes would take 1.4 us): 8191 x
// 256, k = 8, takes 16.3 us with 8 groups, 11.4 without; softmax, all in 64 bits, 24 us.  Sigmoid
// and 8 groups all in 64 bits took 43, with whole rows sent to route64 for one close call 28.
// ---------------------------------------------------------------------------
constexpr int ROUTE_MAX_E = 512, ROUTE_MAX_K = 16, ROUTE_MAX_G = 32;
constexpr int ROUTE_WARPS = 4;

struct RouteArgs {
    const void *logits;
    const float *bias;
    float *w;
    long long *idx;
    long long T;
    double scale;
    int E, k, G, keep, bf16, score, top2, renorm;
    int per, part;   // experts per group, log2 of the lanes that share a group
    uint32_t magic;  // e * magic >> 20 = e / per for e < 512
};

// doubles in an order that unsigned comparison keeps; 0 is below every value, NaN above
__device__ __forceinline__ unsigned long long order_key(double d) {
    if (d != d) return ~0ull;
    if (d == 0.0) d = 0.0;  // -0 is 0
    const long long b = __double_as_longlong(d);
    return (unsigned long long)b ^ (b < 0 ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value(unsigned long long k) {
    if (k == ~0ull) return CUDART_NAN;
    return __longlong_as_double((long long)(k & 0x8000000000000000ull ? k ^ 0x8000000000000000ull : ~k));
}
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return (unsigned long long)hi << 32 | lo;
}

// One score in 64 bits (sigmoid, sqrt(softplus); softmax needs the row).
__device__ __forceinline__ double score64(double z, int score) {
    if (score == WF_SCORE_SIGMOID) return 1.0 / (1.0 + exp(-z));
    return sqrt((z > 0 ? z : 0.0) + log1p(exp(-fabs(z))));
}

__device__ __forceinline__ float logit_at(const RouteArgs &p, long long i) {
    return p.bf16 ? __bfloat162float(((const __nv_bfloat16 *)p.logits)[i]) : __ldg((const float *)p.logits + i);
}

struct Pick {
    int expert;    // -1: none
    double score;
};

// The whole choice of token t in 64 bits: lane j < k returns slot j.  Out of line, and with the
// logits read anew, so that the common path keeps its registers.
template <int N>
__device__ __noinline__ Pick route64(const RouteArgs &p, long long t) {
    const int lane = threadIdx.x & 31;
    float zf[N];
#pragma unroll
    for (int i = 0; i < N; ++i) zf[i] = lane + 32 * i < p.E ? logit_at(p, t * p.E + lane + 32 * i) : -CUDART_INF_F;
    double s[N];
    unsigned long long key[N];
    double top = -CUDART_INF;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s[i] = zf[i];
        nan |= zf[i] != zf[i];
        top = fmax(top, s[i]);
    }
    if (p.score == WF_SCORE_SOFTMAX) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (__any_sync(0xffffffffu, nan)) top = CUDART_NAN;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            key[i] = s[i] != -CUDART_INF;
            s[i] = key[i] ? exp(s[i] - top) : 0.0;
            sum += s[i];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double inv = 1.0 / sum;
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = key[i] ? s[i] * inv : 0.0;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            key[i] = s[i] != -CUDART_INF;
            s[i] = score64(s[i], p.score);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = lane + 32 * i;
        if (key[i]) {
            const double sel = p.bias ? s[i] + (double)__ldg(p.bias + e) : s[i];
            key[i] = sel == -CUDART_INF ? 0ull : order_key(sel);
        }
    }
    if (p.G > 1) {
        // lane g ends with group g's value
        const int per = p.E / p.G;
        unsigned long long mine = 0;
        for (int g = 0; g < p.G; ++g) {
            unsigned long long a = 0, b = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = lane + 32 * i;
                if (e >= g * per && e < (g + 1) * per) {
                    if (key[i] > a) { b = a; a = key[i]; }
                    else if (key[i] > b) b = key[i];
                }
            }
            const unsigned long long m1 = warp_max(a);
            unsigned long long gv = m1;
            if (p.top2 && m1) {
                const int who = __ffs(__ballot_sync(0xffffffffu, a == m1)) - 1;
                const unsigned long long m2 = warp_max(lane == who ? b : a);
                if (m2) gv = order_key(key_value(m1) + key_value(m2));
            }
            if (lane == g) mine = gv;
        }
        uint32_t kept = 0;  // one bit per group
        for (int j = 0; j < p.keep; ++j) {
            const unsigned long long m = warp_max(mine);
            if (!m) break;
            const int who = __ffs(__ballot_sync(0xffffffffu, mine == m)) - 1;
            kept |= 1u << who;
            if (lane == who) mine = 0;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = lane + 32 * i;
            if (e < p.E && !(kept >> (e / per) & 1)) key[i] = 0;
        }
    }
    Pick mine = {-1, 0.0};
    for (int j = 0; j < p.k; ++j) {
        unsigned long long a = 0;
        double sa = 0.0;
        int e = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (key[i] > a) { a = key[i]; sa = s[i]; e = lane + 32 * i; }
        const unsigned long long m = warp_max(a);
        if (!m) break;
        const uint32_t best = __reduce_min_sync(0xffffffffu, a == m ? (uint32_t)e : 0xffffffffu);
        const double sb = __shfl_sync(0xffffffffu, sa, best & 31);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((uint32_t)(lane + 32 * i) == best) key[i] = 0;
        if (lane == j) mine = {(int)best, sb};
    }
    return mine;
}

// sel of expert e of token t in 64 bits
__device__ __noinline__ double sel64(const RouteArgs &p, long long t, int e) {
    const double s = score64((double)logit_at(p, t * p.E + e), p.score);
    return p.bias ? s + (double)__ldg(p.bias + e) : s;
}

// 32-bit keys: order kept under unsigned comparison, 0 below every value
__device__ __forceinline__ uint32_t key32(float f) {
    const uint32_t b = __float_as_uint(f);
    return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value32(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The groups kept, one bit each, by 64-bit values of their best experts (32-bit keys a and b of
// group grp in its leader lane); 0 where a third expert is too near to tell which two are best.
__device__ __noinline__ uint32_t groups64(const RouteArgs &p, long long t, const uint32_t *sm, uint32_t a, uint32_t b, int grp,
                                          bool leader, float gap0) {
    const int lane = threadIdx.x & 31;
    int ea = -1, eb = -1;
    uint32_t c = 0;
    if (leader) {
        for (int j = 0; j < p.per; ++j) {
            const uint32_t v = sm[grp * p.per + j];
            if (v == a && ea < 0) ea = grp * p.per + j;
            else if (v == b && eb < 0) eb = grp * p.per + j;
            else c = max(c, v);
        }
    }
    const float edge = p.top2 ? value32(b) : value32(a);
    if (__any_sync(0xffffffffu, leader && c && !(edge - value32(c) > gap0 + fmaxf(fabsf(edge), fabsf(value32(c))) * 0x1p-17f)))
        return 0;
    const double xa = sel64(p, t, max(ea, 0)), xb = sel64(p, t, max(eb, 0));
    unsigned long long mine = 0;
    if (leader && a) mine = order_key(!b ? xa : p.top2 ? xa + xb : fmax(xa, xb));
    uint32_t kept = 0;
    for (int j = 0; j < p.keep; ++j) {
        const unsigned long long m = warp_max(mine);
        if (!m) break;
        const int who = __ffs(__ballot_sync(0xffffffffu, mine == m)) - 1;
        kept |= 1u << __shfl_sync(0xffffffffu, grp, who);
        if (lane == who) mine = 0;
    }
    return kept;
}

// The choice screened in 32 bits.  A 32-bit score is off by less than 2^-21 of itself (expf and
// log1pf to 2 ulp, an addition, a reciprocal or a square root) and sel by half an ulp more; its key
// gives up its 4 lowest bits (2^-19 of sel) to the place of the expert in its lane, so one
// reduction finds a winner and where it sits.  Two values further apart than `gap` are in the
// right order; a winner closer than that to the one before it (1.2 % of rows of 256 normal logits)
// is put in its place by the 64-bit values of the winners so far, one evaluation in all lanes at
// once, and so is a choice of groups (0.1 % of rows of 8 groups).  Rows with NaN, +infinity or too
// few experts and long runs of equal values are left to route64, which takes several times as
// long, and a launch takes as long as its slowest row.  Returns whether the row was settled;
// lane j < k has the expert of slot j.
template <int N>
__device__ __forceinline__ bool route32(const RouteArgs &p, long long t, const float (&z)[N], const float (&bias)[N],
                                        uint32_t *sm, int &my_idx) {
    static_assert(N <= 16, "4 bits for the place in the lane");
    const int lane = threadIdx.x & 31;
    uint32_t key[N];
    float smax = 0.f, all = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float sc;
        if (p.score == WF_SCORE_SIGMOID) {
            const float d = 1.0f + expf(-z[i]);
            asm("rcp.approx.f32 %0, %1;" : "=f"(sc) : "f"(d));
        } else {
            sc = __fsqrt_rn(fmaxf(z[i], 0.f) + log1pf(expf(-fabsf(z[i]))));
        }
        const float sel = sc + bias[i];
        smax = fmaxf(smax, sc);
        all = max_nan(all, max_nan(z[i], sel));
        key[i] = z[i] == -CUDART_INF_F || sel == -CUDART_INF_F ? 0u : (key32(sel) & ~15u) | i;
    }
    if (__any_sync(0xffffffffu, !(all < CUDART_INF_F))) return false;
    smax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(smax)));  // scores are not negative
    if (smax < 0x1p-40f) return false;  // subnormal steps of expf: the bound above does not hold
    const float gap0 = smax * 0x1p-18f;
    if (p.G > 1) {
        // 2^w lanes per group: each takes every 2^w-th expert of it, then their best two are merged
        const int per = p.per, w = p.part, sub = lane & ((1 << w) - 1), grp = lane >> w;
#pragma unroll
        for (int i = 0; i < N; ++i) sm[lane + 32 * i] = key[i];
        __syncwarp();
        uint32_t a = 0, b = 0;
        if (grp < p.G) {
            const int n = (per - sub + (1 << w) - 1) >> w;
            const uint32_t *g = sm + grp * per + sub;
            int q = grp < n ? grp : 0;  // groups start apart: their lanes read other banks
            for (int j = 0; j < n; ++j) {
                const uint32_t v = g[q << w];
                b = max(b, min(a, v));
                a = max(a, v);
                if (++q == n) q = 0;
            }
        }
        for (int o = 1; o < 1 << w; o <<= 1) {
            const uint32_t a2 = __shfl_xor_sync(0xffffffffu, a, o), b2 = __shfl_xor_sync(0xffffffffu, b, o);
            b = max(min(a, a2), max(b, b2));
            a = max(a, a2);
        }
        // a sum's error goes with its terms, which may cancel
        const float mag = __uint_as_float(__reduce_max_sync(
            0xffffffffu, max(a ? __float_as_uint(fabsf(value32(a))) : 0u, b ? __float_as_uint(fabsf(value32(b))) : 0u)));
        uint32_t mine = a;
        if (p.top2 && b) {
            const float v = value32(a) + value32(b);
            mine = v > -CUDART_INF_F ? key32(v) : 0u;
        }
        if (sub) mine = 0;
        uint32_t kept = 0, m = 0;
        for (int j = 0; j < p.keep; ++j) {
            m = __reduce_max_sync(0xffffffffu, mine);
            if (!m) return false;
            const int who = __ffs(__ballot_sync(0xffffffffu, mine == m)) - 1;
            kept |= 1u << (who >> w);
            if (lane == who) mine = 0;
        }
        const uint32_t next = __reduce_max_sync(0xffffffffu, mine);
        if (next && !(value32(m) - value32(next) > 2 * gap0 + mag * 0x1p-16f)) {
            kept = groups64(p, t, sm, a, b, grp, sub == 0 && grp < p.G, gap0);
            if (!kept) return false;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!(kept >> ((lane + 32 * i) * p.magic >> 20) & 1)) key[i] = 0;  // (past E: 0 already)
    }
    // each lane's keys in descending order (a bitonic network): a winner is the head of its lane
#pragma unroll
    for (int size = 2; size <= N; size <<= 1)
#pragma unroll
        for (int st = size >> 1; st > 0; st >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if ((i & st) == 0) {
                    const uint32_t hi = max(key[i], key[i | st]), lo = min(key[i], key[i | st]);
                    key[i] = (i & size) == 0 ? hi : lo;
                    key[i | st] = (i & size) == 0 ? lo : hi;
                }
    my_idx = -1;
    float last = 0.f, kth = 0.f;
    for (int j = 0; j < p.k + 8; ++j) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, key[0]);
        if (!m) return j >= p.k;
        const float v = value32(m);
        // the slots hold the k best so far: what is left cannot pass the k-th by its error
        if (j >= p.k && kth - v > gap0 + fmaxf(fabsf(kth), fabsf(v)) * 0x1p-17f) return true;
        const int who = __ffs(__ballot_sync(0xffffffffu, key[0] == m)) - 1;
        const int e = who + 32 * (int)(m & 15);
        if (lane == who) {
#pragma unroll
            for (int i = 0; i + 1 < N; ++i) key[i] = key[i + 1];
            key[N - 1] = 0;
        }
        if (j == 0 || last - v > gap0 + fmaxf(fabsf(last), fabsf(v)) * 0x1p-17f) {
            if (lane == j) my_idx = e;
        } else {
            const int have = min(j, p.k), mine = lane < have ? my_idx : e;
            const double x = sel64(p, t, mine), xe = __shfl_sync(0xffffffffu, x, 31);
            const int rank = __popc(__ballot_sync(0xffffffffu, lane < have && (x > xe || (x == xe && mine < e))));
            const int below = __shfl_up_sync(0xffffffffu, my_idx, 1);
            if (lane < p.k) my_idx = lane == rank ? e : lane > rank && lane <= have ? below : my_idx;
        }
        last = v;
        if (j == p.k - 1) kth = v;
    }
    return false;
}

template <int N>  // experts per lane
__global__ void __launch_bounds__(32 * ROUTE_WARPS, N <= 8 ? 10 : 4) k_route_topk(const __grid_constant__ RouteArgs p) {
    __shared__ uint32_t sm[ROUTE_WARPS][32 * N];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long t = (long long)blockIdx.x * ROUTE_WARPS + warp;
    pdl_wait();
    if (t >= p.T) return;
    float z[N], bias[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        z[i] = lane + 32 * i < p.E ? logit_at(p, t * p.E + lane + 32 * i) : -CUDART_INF_F;
        bias[i] = p.bias && lane + 32 * i < p.E ? __ldg(p.bias + lane + 32 * i) : 0.f;
    }
    Pick pick;
    // softmax weights need the row's sum in 64 bits anyway
    if (p.score != WF_SCORE_SOFTMAX && route32<N>(p, t, z, bias, sm[warp], pick.expert))
        pick.score = pick.expert < 0 ? 0.0 : score64((double)logit_at(p, t * p.E + pick.expert), p.score);
    else
        pick = route64<N>(p, t);
    if (p.renorm) {
        double sum = 0.0;  // the same order in every lane
        for (int j = 0; j < p.k; ++j) sum += __shfl_sync(0xffffffffu, pick.score, j);
        pick.score = sum == 0.0 ? 0.0 : pick.score / sum;
    }
    if (lane < p.k) {
        p.w[t * p.k + lane] = (float)(pick.expert < 0 ? 0.0 : pick.score * p.scale);
        p.idx[t * p.k + lane] = pick.expert;
    }
}

// ---------------------------------------------------------------------------
// Dispatch: a stable counting sort of the (token, slot) pairs by expert
//   offsets[e] = first row of expert e, tokens[r] = token of row r,
//   slots[t, j] = row of pair (t, j), or -1 for an expert outside the range.
// A row's place is its expert's start plus the number of earlier pairs of that
// expert, so the order is (expert, token, slot) whatever the schedule.  The pairs
// are cut into chunks, one CTA each, and a chunk into one run per warp; every
// warp counts its run per expert (lanes that hold the same expert find one
// another with match_any), the counts are summed over warps and chunks, and a
// second walk over the run hands out the places.  One launch where one chunk
// holds all pairs; else a counting launch before it, under which this one starts
// (programmatic launch) and reads and counts its own run.
// Latency-bound at every size (16384 x 8 pairs are 2 MB): a warp's pairs sit in
// registers, 4 loads in flight, and the two walks read no memory.
// ---------------------------------------------------------------------------
constexpr int DISP_MAX_E = 512, DISP_WARPS = 16, DISP_LANE = 4, DISP_STEP = 32 * DISP_LANE;  // pairs of a warp's step
constexpr int DISP_CHUNK = DISP_WARPS * DISP_STEP, DISP_MAX_CHUNKS = 512;

struct DispArgs {
    const void *indices;
    int idx64;
    int pairs, k, E, base;
    int run, nchunks;  // pairs per warp (a multiple of 32), chunks of DISP_WARPS runs
    int row;           // E rounded up to a multiple of 4
    int *hist;         // [nchunks, row] when nchunks > 1
    int *offsets, *tokens, *slots;
};

// The local experts of DISP_LANE x 32 consecutive pairs from i0 on (-1: none), pair i0 + 32 j + lane in e[j].
__device__ __forceinline__ void disp_load(const DispArgs &p, int i0, int hi, int (&e)[DISP_LANE]) {
    const int lane = threadIdx.x & 31;
    long long v[DISP_LANE];
#pragma unroll
    for (int j = 0; j < DISP_LANE; ++j) {
        const int i = i0 + 32 * j + lane;
        v[j] = -1;
        if (i < hi) v[j] = p.idx64 ? __ldg((const long long *)p.indices + i) : (long long)__ldg((const int *)p.indices + i);
    }
#pragma unroll
    for (int j = 0; j < DISP_LANE; ++j) {
        const int i = i0 + 32 * j + lane;
        e[j] = i < hi && v[j] >= p.base && v[j] < (long long)p.base + p.E ? (int)(v[j] - p.base) : -1;
    }
}

__global__ void __launch_bounds__(32 * DISP_WARPS) k_dispatch_count(const __grid_constant__ DispArgs p) {
    __shared__ int cnt[DISP_MAX_E];
    pdl_wait();
    pdl_launch_dependents();  // behind the wait: k_dispatch_place reads the indices without one of its own
    const int warp = threadIdx.x >> 5;
    const int lo = min(p.pairs, (blockIdx.x * DISP_WARPS + warp) * p.run), hi = min(p.pairs, lo + p.run);
    int e[DISP_LANE];
    disp_load(p, lo, hi, e);
    for (int x = threadIdx.x; x < p.E; x += blockDim.x) cnt[x] = 0;
    __syncthreads();
    for (int i0 = lo; i0 < hi;) {
#pragma unroll
        for (int j = 0; j < DISP_LANE; ++j)
            if (e[j] >= 0) atomicAdd(&cnt[e[j]], 1);
        i0 += DISP_STEP;
        if (i0 < hi) disp_load(p, i0, hi, e);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < p.row; x += blockDim.x) p.hist[(size_t)blockIdx.x * p.row + x] = x < p.E ? cnt[x] : 0;
}

__global__ void __launch_bounds__(32 * DISP_WARPS) k_dispatch_place(const __grid_constant__ DispArgs p) {
    __shared__ int cnt[DISP_WARPS][DISP_MAX_E];
    __shared__ int total[DISP_MAX_E + 1], before[DISP_MAX_E], scan[DISP_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int lo = min(p.pairs, (blockIdx.x * DISP_WARPS + warp) * p.run), hi = min(p.pairs, lo + p.run);
    const bool whole = hi - lo <= DISP_STEP;  // the run stays in registers
    int e[DISP_LANE], ahead[DISP_LANE];
    // After the counting kernel, which lets this one start only when everything before it is done,
    // the indices can be read at once.
    if (p.nchunks == 1) pdl_wait();
    disp_load(p, lo, hi, e);
    for (int x = lane; x < p.E; x += 32) cnt[warp][x] = 0;
    for (int x = threadIdx.x; x < p.E; x += blockDim.x) total[x] = before[x] = 0;
    __syncwarp();
    for (int i0 = lo; i0 < hi;) {
#pragma unroll
        for (int j = 0; j < DISP_LANE; ++j) {
            // pairs of the same expert earlier in the run: this warp's so far, then lower lanes
            const uint32_t same = __match_any_sync(0xffffffffu, e[j]);
            const int at = e[j] >= 0 ? cnt[warp][e[j]] : 0;
            ahead[j] = at + __popc(same & ((1u << lane) - 1));
            __syncwarp();
            if (e[j] >= 0 && lane == __ffs(same) - 1) cnt[warp][e[j]] = at + __popc(same);
            __syncwarp();
        }
        i0 += DISP_STEP;
        if (i0 < hi) disp_load(p, i0, hi, e);
    }
    if (p.nchunks > 1) {
        __syncthreads();
        pdl_wait();
        // four experts a thread, the chunks dealt out over the groups of threads that cover a row
        const int quads = p.row / 4, g = threadIdx.x / quads, groups = blockDim.x / quads, x = threadIdx.x % quads * 4;
        if (g < groups) {
            int4 pre = make_int4(0, 0, 0, 0), all = pre;
#pragma unroll 8
            for (int c = g; c < p.nchunks; c += groups) {
                const int4 n = __ldcg(reinterpret_cast<const int4 *>(p.hist + (size_t)c * p.row + x));
                const int m = c < (int)blockIdx.x ? -1 : 0;
                all.x += n.x; all.y += n.y; all.z += n.z; all.w += n.w;
                pre.x += n.x & m; pre.y += n.y & m; pre.z += n.z & m; pre.w += n.w & m;
            }
            const int va[4] = {all.x, all.y, all.z, all.w}, vp[4] = {pre.x, pre.y, pre.z, pre.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (va[j]) atomicAdd(&total[x + j], va[j]);
                if (vp[j]) atomicAdd(&before[x + j], vp[j]);
            }
        }
    }
    __syncthreads();
    // expert x (one thread each): where each warp's pairs of it start, and where the expert starts
    {
        const int x = threadIdx.x;
        int at = 0, all = 0;
        if (x < p.E) {
            at = before[x];
#pragma unroll
            for (int w = 0; w < DISP_WARPS; ++w) {
                const int n = cnt[w][x];
                cnt[w][x] = at;
                at += n;
            }
            all = p.nchunks > 1 ? total[x] : at;
        }
        int incl = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        int start = incl - all;
        for (int w = 0; w < warp; ++w) start += scan[w];
        if (x <= p.E) total[x] = start;
        if (x == DISP_MAX_E - 1 && p.E == DISP_MAX_E) total[DISP_MAX_E] = start + all;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int x = threadIdx.x; x <= p.E; x += blockDim.x) p.offsets[x] = total[x];
    for (int i0 = lo; i0 < hi; i0 += DISP_STEP) {
        if (!whole) disp_load(p, i0, hi, e);
#pragma unroll
        for (int j = 0; j < DISP_LANE; ++j) {
            const int i = i0 + 32 * j + lane;
            int r = -1;
            if (whole) {
                if (e[j] >= 0) r = total[e[j]] + cnt[warp][e[j]] + ahead[j];
            } else {
                const uint32_t same = __match_any_sync(0xffffffffu, e[j]);
                const int at = e[j] >= 0 ? cnt[warp][e[j]] : 0;
                __syncwarp();
                if (e[j] >= 0 && lane == __ffs(same) - 1) cnt[warp][e[j]] = at + __popc(same);
                __syncwarp();
                if (e[j] >= 0) r = total[e[j]] + at + __popc(same & ((1u << lane) - 1));
            }
            if (i < hi) {
                if (r >= 0) p.tokens[r] = i / p.k;
                p.slots[i] = r;
            }
        }
    }
    // rows that no pair of the range fills
    for (int r = total[p.E] + blockIdx.x * blockDim.x + threadIdx.x; r < p.pairs; r += gridDim.x * blockDim.x)
        p.tokens[r] = -1;
}

// ---------------------------------------------------------------------------
// Combine: y[t] = sum over the token's rows of weight * rows[slot] (+ shared[t])
// in ascending row order (ascending expert, the layer's own order), in 32 bits.
// A slot outside [0, R) adds nothing.  One CTA per token and 2048 columns, 8
// columns per thread; the token's slots are sorted once per CTA.
// Bound by HBM: 8192 tokens x 8 rows of 4096 with the shared rows, 671 MB, take 104 to 107 us,
// 6.4 TB/s (one row's load at a time: 117 us; eight, with fewer CTAs on an SM: 112 us).
// ---------------------------------------------------------------------------
constexpr int COMB_MAX_K = 16;

struct CombArgs {
    const uint4 *rows, *shared;
    const int *slots;
    const float *weights;
    void *y;
    int R, k, chunks, y_f32;
};

__global__ void __launch_bounds__(256) k_combine(const __grid_constant__ CombArgs p) {
    __shared__ int slot[COMB_MAX_K];
    __shared__ float weight[COMB_MAX_K];
    const size_t t = blockIdx.x;
    const int lane = threadIdx.x & 31;
    pdl_wait();
    if (threadIdx.x < 32) {
        const int s = lane < p.k ? p.slots[t * p.k + lane] : -1;
        const float w = lane < p.k && p.weights ? p.weights[t * p.k + lane] : 1.0f;
        int rank = 0;
        for (int j = 0; j < p.k; ++j) {
            const int o = __shfl_sync(0xffffffffu, s, j);
            rank += o < s || (o == s && j < lane);
        }
        if (lane < p.k) {
            slot[rank] = s;
            weight[rank] = w;
        }
    }
    __syncthreads();
    const int c = blockIdx.y * blockDim.x + threadIdx.x;
    if (c >= p.chunks) return;
    float acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
    for (int i0 = 0; i0 < p.k; i0 += 4) {  // four rows' loads in flight
        uint4 a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = i0 + i < p.k ? slot[i0 + i] : -1;
            if (s >= 0 && s < p.R) a[i] = __ldg(p.rows + (size_t)s * p.chunks + c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = i0 + i < p.k ? slot[i0 + i] : -1;
            if (s < 0 || s >= p.R) continue;
            const float w = weight[i0 + i];
            const uint32_t u[4] = {a[i].x, a[i].y, a[i].z, a[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = bf2(u[j]);
                acc[2 * j] += w * f.x;
                acc[2 * j + 1] += w * f.y;
            }
        }
    }
    const size_t at = t * p.chunks + c;
    if (p.shared) {
        const uint4 a = __ldg(p.shared + at);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = bf2(u[j]);
            acc[2 * j] += f.x;
            acc[2 * j + 1] += f.y;
        }
    }
    if (p.y_f32) {
        float4 *y = (float4 *)p.y + 2 * at;
        y[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        y[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    } else {
        ((uint4 *)p.y)[at] = make_uint4(pack_bf2(acc[0], acc[1]), pack_bf2(acc[2], acc[3]), pack_bf2(acc[4], acc[5]),
                                        pack_bf2(acc[6], acc[7]));
    }
}

std::atomic<uint64_t> norm_ready[64];  // devices on which a variant may use its shared memory

int launched(cudaError_t e, const char *what) { return e == cudaSuccess ? WF_OK : cuda_fail(e, what); }

bool misaligned(const void *p, uintptr_t to) { return (uintptr_t)p % to != 0; }

}  // namespace lops
}  // namespace wf

using namespace wf::lops;

extern "C" {

int wf_rms_norm_quant(const void *x, const void *residual, const void *weight, int32_t weight_bf16, int64_t T,
                      int64_t D, float eps, int32_t ue8m0, void *q, void *s, int32_t scale_kind, void *y, void *h,
                      void *stream) {
    if (!x || !weight || !q || !s) return fail(WF_E_ARG, "null pointer");
    if (!residual != !h) return fail(WF_E_ARG, "residual and h go together");
    if (T <= 0 || T > 0x7fffffff) return fail(WF_E_SHAPE, "T outside 1..2^31-1");
    if (D <= 0 || D % 128 || D > 16384) return fail(WF_E_SHAPE, "D must be a positive multiple of 128, at most 16384");
    if (scale_kind != WF_SCALE_F32 && scale_kind != WF_SCALE_E8M0) return fail(WF_E_DTYPE, "bad scale kind");
    if (scale_kind == WF_SCALE_E8M0 && !ue8m0) return fail(WF_E_DTYPE, "e8m0 scales need ue8m0 rounding");
    if (misaligned(x, 16) || misaligned(residual, 16) || misaligned(weight, 16) || misaligned(y, 16) ||
        misaligned(h, 16) || misaligned(q, 8) || misaligned(s, 4))
        return fail(WF_E_ARG, "x, residual, weight, y and h must be 16-byte aligned, q 8-byte, s 4-byte");
    NormArgs p;
    p.x = (const uint4 *)x; p.res = (const uint4 *)residual; p.weight = weight;
    p.y = (uint4 *)y; p.h = (uint4 *)h; p.q = (uint2 *)q; p.s = s;
    p.eps = eps; p.inv_d = 1.0f / (float)D; p.chunks = (int)(D / 8); p.T = T;
    p.weight_bf16 = weight_bf16 != 0; p.ue8m0 = ue8m0 != 0; p.s_f32 = scale_kind == WF_SCALE_F32;
    const int sms = wf::host::sm_count();
    if (sms <= 0) return fail(WF_E_CUDA, "no CUDA device");
    // Threads: one, two or four chunks each, the fewest that hold a row in a block.  CTAs: reads and
    // writes together run best with few rows open at a time (with residual and both outputs, 2, 3 and
    // 4 CTAs on an SM: D = 4096 6.4, 5.3 and 5.2 TB/s; D = 2048 5.3, 6.2 and 5.8); without the
    // residual the instructions count and more threads help (D = 4096 4.2, 5.0 and 5.3 TB/s).
    const int ch = p.chunks <= 256 ? 1 : p.chunks <= 1024 ? 2 : 4;
    const int nt = ((p.chunks + ch - 1) / ch + 31) / 32 * 32;
    const int threads = ch == 4 ? 512 : !residual ? 1024 : ch == 2 ? 704 : 768;
    const int ctas = threads / nt < 32 ? threads / nt : 32;
    const int64_t most = (int64_t)sms * ctas;
    const dim3 g((unsigned)(T < most ? T : most));
    p.depth = T <= most || ch == 4 || (residual && ch == 1) ? 2 : 3;
    const int room = 128 << 10;  // two rows of 16384 with their residuals
    const size_t smem = (size_t)p.depth * (residual ? 2 : 1) * ch * nt * 16;
    auto k = ch == 1 ? k_rms_norm_quant<1> : ch == 2 ? k_rms_norm_quant<2> : k_rms_norm_quant<4>;
    if (smem > 47 << 10) {  // (the static arrays count too)
        const cudaError_t e = wf::host::allow_smem((const void *)k, ch, room, norm_ready);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(rms_norm_quant)");
    }
    return launched(wf::host::launch_pdl(k, g, nt, smem, (cudaStream_t)stream, p), "rms_norm_quant launch");
}

int wf_route_topk(const void *logits, int32_t logits_bf16, const float *bias, int64_t T, int32_t E, int32_t topk,
                  int32_t score_func, int32_t n_groups, int32_t topk_groups, int32_t group_top2, int32_t renorm,
                  float route_scale, float *out_weights, int64_t *out_indices, void *stream) {
    if (!logits || !out_weights || !out_indices) return fail(WF_E_ARG, "null pointer");
    if (T <= 0 || T > 0x7fffffff) return fail(WF_E_SHAPE, "T outside 1..2^31-1");
    if (E <= 0 || E > ROUTE_MAX_E) return fail(WF_E_SHAPE, "n_experts must be in 1..512");
    if (topk <= 0 || topk > ROUTE_MAX_K || topk > E) return fail(WF_E_SHAPE, "topk must be in 1..min(16, n_experts)");
    if (score_func < 0 || score_func > 2) return fail(WF_E_DTYPE, "bad score_func");
    if (n_groups <= 0 || n_groups > ROUTE_MAX_G || E % n_groups)
        return fail(WF_E_SHAPE, "n_groups must be in 1..32 and divide n_experts");
    if (topk_groups <= 0 || topk_groups > n_groups) return fail(WF_E_SHAPE, "topk_groups must be in 1..n_groups");
    if (topk > (int64_t)topk_groups * (E / n_groups))
        return fail(WF_E_SHAPE, "topk exceeds the experts of topk_groups groups");
    if (misaligned(logits, logits_bf16 ? 2 : 4) || misaligned(bias, 4) || misaligned(out_weights, 4) ||
        misaligned(out_indices, 8))
        return fail(WF_E_ARG, "misaligned pointer");
    RouteArgs p;
    p.logits = logits; p.bias = bias; p.w = out_weights; p.idx = (long long *)out_indices;
    p.T = T; p.scale = route_scale; p.E = E; p.k = topk; p.G = n_groups == topk_groups ? 1 : n_groups;
    p.keep = topk_groups; p.bf16 = logits_bf16 != 0; p.score = score_func; p.top2 = group_top2 != 0;
    p.renorm = renorm != 0;
    p.per = E / n_groups;
    p.magic = ((1u << 20) + p.per - 1) / p.per;
    p.part = 0;
    while (2 << p.part <= 32 / n_groups) ++p.part;
    const dim3 g((unsigned)((T + ROUTE_WARPS - 1) / ROUTE_WARPS));
    const int per = (E + 31) / 32;
    auto k = per <= 2 ? k_route_topk<2> : per <= 4 ? k_route_topk<4> : per <= 8 ? k_route_topk<8> : k_route_topk<16>;
    return launched(wf::host::launch_pdl(k, g, 32 * ROUTE_WARPS, 0, (cudaStream_t)stream, p), "route_topk launch");
}

// Chunks of `pairs` pairs, and the pairs of a warp's run: short runs for few pairs, so that the
// warps of the one CTA share them, longer than a step only past DISP_MAX_CHUNKS full chunks.
static int disp_chunks(int64_t pairs, int *run) {
    int64_t r = DISP_STEP;
    if (pairs <= DISP_CHUNK) {
        r = (pairs + DISP_WARPS - 1) / DISP_WARPS;
        r = (r + 31) / 32 * 32;
    } else if (pairs > (int64_t)DISP_CHUNK * DISP_MAX_CHUNKS) {
        r = (pairs + (int64_t)DISP_MAX_CHUNKS * DISP_WARPS - 1) / (DISP_MAX_CHUNKS * DISP_WARPS);
        r = (r + DISP_STEP - 1) / DISP_STEP * DISP_STEP;
    }
    *run = (int)r;
    return (int)((pairs + r * DISP_WARPS - 1) / (r * DISP_WARPS));
}

static bool disp_ok(int64_t T, int32_t topk, int32_t n_experts) {
    return T > 0 && topk > 0 && topk <= ROUTE_MAX_K && T <= 1 << 30 && T * topk <= 1 << 30 && n_experts > 0 &&
           n_experts <= DISP_MAX_E;
}

size_t wf_expert_dispatch_workspace_bytes(int64_t T, int32_t topk, int32_t n_experts) {
    if (!disp_ok(T, topk, n_experts)) return 0;
    int run;
    const int n = disp_chunks(T * topk, &run);
    return n > 1 ? (size_t)n * ((n_experts + 3) / 4 * 4) * 4 : 0;
}

int wf_expert_dispatch(const void *indices, int32_t indices_64, int64_t T, int32_t topk, int32_t n_experts,
                       int64_t expert_offset, int32_t *offsets, int32_t *tokens, int32_t *slots, void *workspace,
                       size_t workspace_bytes, void *stream) {
    if (!indices || !offsets || !tokens || !slots) return fail(WF_E_ARG, "null pointer");
    if (!disp_ok(T, topk, n_experts))
        return fail(WF_E_SHAPE, "need topk in 1..16, T * topk in 1..2^30 and n_experts in 1..512");
    if (expert_offset < 0 || expert_offset > 0x7fffffff - DISP_MAX_E) return fail(WF_E_SHAPE, "expert_offset out of range");
    const size_t need = wf_expert_dispatch_workspace_bytes(T, topk, n_experts);
    if (need && (!workspace || workspace_bytes < need))
        return fail(WF_E_ARG, "workspace too small (see wf_expert_dispatch_workspace_bytes)");
    if (misaligned(indices, indices_64 ? 8 : 4) || misaligned(offsets, 4) || misaligned(tokens, 4) ||
        misaligned(slots, 4) || misaligned(workspace, 16))
        return fail(WF_E_ARG, "misaligned pointer (indices to their size, the workspace to 16 bytes, the rest to 4)");
    DispArgs p;
    p.indices = indices; p.idx64 = indices_64 != 0; p.pairs = (int)(T * topk); p.k = topk; p.E = n_experts;
    p.row = (n_experts + 3) / 4 * 4; p.base = (int)expert_offset; p.hist = (int *)workspace; p.offsets = offsets; p.tokens = tokens; p.slots = slots;
    p.nchunks = disp_chunks(p.pairs, &p.run);
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = cudaSuccess;
    if (p.nchunks > 1) e = wf::host::launch_pdl(k_dispatch_count, dim3(p.nchunks), 32 * DISP_WARPS, 0, st, p);
    if (e == cudaSuccess) e = wf::host::launch_pdl(k_dispatch_place, dim3(p.nchunks), 32 * DISP_WARPS, 0, st, p);
    return launched(e, "expert_dispatch launch");
}

int wf_expert_combine(const void *rows, int64_t R, const int32_t *slots, const float *weights, const void *shared,
                      int64_t T, int32_t topk, int64_t D, void *y, int32_t y_f32, void *stream) {
    if ((!rows && R) || !slots || !y) return fail(WF_E_ARG, "null pointer");
    if (R < 0 || R > 0x7fffffff) return fail(WF_E_SHAPE, "R outside 0..2^31-1");
    if (T <= 0 || T > 0x7fffffff) return fail(WF_E_SHAPE, "T outside 1..2^31-1");
    if (topk <= 0 || topk > COMB_MAX_K) return fail(WF_E_SHAPE, "topk must be in 1..16");
    if (D <= 0 || D % 8 || D > (1 << 20)) return fail(WF_E_SHAPE, "D must be a positive multiple of 8, at most 2^20");
    if (misaligned(rows, 16) || misaligned(shared, 16) || misaligned(y, 16) || misaligned(slots, 4) ||
        misaligned(weights, 4))
        return fail(WF_E_ARG, "rows, shared and y must be 16-byte aligned");
    CombArgs p;
    p.rows = (const uint4 *)rows; p.shared = (const uint4 *)shared; p.slots = slots; p.weights = weights; p.y = y;
    p.R = (int)R; p.k = topk; p.chunks = (int)(D / 8); p.y_f32 = y_f32 != 0;
    const int nt = p.chunks >= 256 ? 256 : (p.chunks + 31) / 32 * 32;
    const dim3 g((unsigned)T, (unsigned)((p.chunks + nt - 1) / nt));
    return launched(wf::host::launch_pdl(k_combine, g, nt, 0, (cudaStream_t)stream, p), "expert_combine launch");
}

}  // extern "C"
