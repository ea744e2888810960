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

// ---------------------------------------------------------------------------
// RMS norm + residual + E4M3 output
//   h = bf16(x + residual)          (the residual stream; x itself without one)
//   n = h * rsqrt(mean(h^2) + eps) * weight               (32 bits)
//   y = bf16(n)
//   per 128 columns: s = max(amax|n|, 1e-4) / 448, with ue8m0 rounded up to a
//   power of two; q = e4m3(n / s)
// The statistics are those of the rounded h, which is what the next layer reads
// back.  q is taken from the 32-bit n, not from y: one rounding fewer.
// One CTA per row; a thread keeps its 8-column chunks in registers between the
// sum of squares and the output, so every input is read once.  A block of 128
// columns is 16 neighbouring lanes.
// ---------------------------------------------------------------------------
struct NormArgs {
    const uint4 *x, *res;
    const void *weight;
    uint4 *y, *h;
    uint2 *q;
    void *s;
    float eps, inv_d;
    int chunks;  // D / 8
    int weight_bf16, ue8m0, s_f32;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <int CH>
__global__ void __launch_bounds__(256) k_rms_norm_quant(const __grid_constant__ NormArgs p) {
    __shared__ float part[8];
    const int nt = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t row = (size_t)blockIdx.x * p.chunks;
    float v[CH][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = threadIdx.x + i * nt;
        if (c < p.chunks) {
            const uint4 a = __ldg(p.x + row + c);
            const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = bf2(u[j]);
                v[i][2 * j] = f.x;
                v[i][2 * j + 1] = f.y;
            }
            if (p.res) {
                const uint4 b = __ldg(p.res + row + c);
                const uint32_t w[4] = {b.x, b.y, b.z, b.w};
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = bf2(w[j]);
                    o[j] = pack_bf2(v[i][2 * j] + f.x, v[i][2 * j + 1] + f.y);
                    const float2 r = bf2(o[j]);
                    v[i][2 * j] = r.x;
                    v[i][2 * j + 1] = r.y;
                }
                p.h[row + c] = make_uint4(o[0], o[1], o[2], o[3]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    ss = 0.f;
    for (int w = 0; w < nt / 32; ++w) ss += part[w];
    const float rstd = rsqrtf(ss * p.inv_d + p.eps);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = threadIdx.x + i * nt;
        const bool on = c < p.chunks;  // whole groups of 16 lanes: chunks is a multiple of 16
        float amax = 0.f;
        if (on) {
            float w[8];
            if (p.weight_bf16) {
                const uint4 a = __ldg((const uint4 *)p.weight + c);
                const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = bf2(u[j]);
                    w[2 * j] = f.x;
                    w[2 * j + 1] = f.y;
                }
            } else {
                const float4 a = __ldg((const float4 *)p.weight + 2 * c), b = __ldg((const float4 *)p.weight + 2 * c + 1);
                w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
                w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[i][j] = v[i][j] * rstd * w[j];
                amax = max_nan(amax, fabsf(v[i][j]));
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
        uint32_t lo, hi;
        if (p.ue8m0) {
            const float inv = 1.0f / s;  // exact
            lo = f32x2_to_e4m3x2(v[i][0] * inv, v[i][1] * inv) | (uint32_t)f32x2_to_e4m3x2(v[i][2] * inv, v[i][3] * inv) << 16;
            hi = f32x2_to_e4m3x2(v[i][4] * inv, v[i][5] * inv) | (uint32_t)f32x2_to_e4m3x2(v[i][6] * inv, v[i][7] * inv) << 16;
        } else {
            lo = f32x2_to_e4m3x2(v[i][0] / s, v[i][1] / s) | (uint32_t)f32x2_to_e4m3x2(v[i][2] / s, v[i][3] / s) << 16;
            hi = f32x2_to_e4m3x2(v[i][4] / s, v[i][5] / s) | (uint32_t)f32x2_to_e4m3x2(v[i][6] / s, v[i][7] / s) << 16;
        }
        p.q[row + c] = make_uint2(lo, hi);
        if (p.y)
            p.y[row + c] = make_uint4(pack_bf2(v[i][0], v[i][1]), pack_bf2(v[i][2], v[i][3]),
                                      pack_bf2(v[i][4], v[i][5]), pack_bf2(v[i][6], v[i][7]));
        if ((lane & 15) == 0) {
            const size_t at = (row + c) >> 4;
            if (p.s_f32) ((float *)p.s)[at] = s;
            else ((uint8_t *)p.s)[at] = (uint8_t)byte;
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
// One warp per token; a lane holds experts lane, lane + 32, ...
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

template <int N>  // experts per lane
__global__ void __launch_bounds__(32 * ROUTE_WARPS) k_route_topk(const __grid_constant__ RouteArgs p) {
    __shared__ double picked[ROUTE_WARPS][ROUTE_MAX_K];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long t = (long long)blockIdx.x * ROUTE_WARPS + warp;
    if (t >= p.T) return;
    double s[N];
    unsigned long long key[N];
    double top = -CUDART_INF;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = lane + 32 * i;
        float z = -CUDART_INF_F;
        if (e < p.E)
            z = p.bf16 ? __bfloat162float(((const __nv_bfloat16 *)p.logits)[t * p.E + e])
                       : ((const float *)p.logits)[t * p.E + e];
        s[i] = z;
        nan |= z != z;
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
            const double z = s[i];
            key[i] = z != -CUDART_INF;
            if (p.score == WF_SCORE_SIGMOID) s[i] = 1.0 / (1.0 + exp(-z));
            else s[i] = sqrt((z > 0 ? z : 0.0) + log1p(exp(-fabs(z))));
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
        // keep the best groups: one flag bit each
        uint32_t kept = 0;
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
    int my_idx = -1;
    for (int j = 0; j < p.k; ++j) {
        unsigned long long a = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (key[i] > a) { a = key[i]; at = i; }
        const unsigned long long m = warp_max(a);
        if (!m) {
            if (lane >= j && lane < p.k) picked[warp][lane] = 0.0;
            break;
        }
        const int e = lane + 32 * at;
        const uint32_t best = __reduce_min_sync(0xffffffffu, a == m ? (uint32_t)e : 0xffffffffu);
        if (a == m && (uint32_t)e == best) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i == at) {
                    key[i] = 0;
                    picked[warp][j] = s[i];
                }
        }
        if (lane == j) my_idx = (int)best;
    }
    __syncwarp();
    if (lane < p.k) {
        double w = picked[warp][lane];
        if (p.renorm) {
            double sum = 0.0;
            for (int j = 0; j < p.k; ++j) sum += picked[warp][j];
            w = sum == 0.0 ? 0.0 : w / sum;
        }
        p.w[t * p.k + lane] = (float)(my_idx < 0 ? 0.0 : w * p.scale);
        p.idx[t * p.k + lane] = my_idx;
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
// holds all pairs, else a counting launch before it.
// ---------------------------------------------------------------------------
constexpr int DISP_MAX_E = 512, DISP_WARPS = 8, DISP_MAX_CHUNKS = 256, DISP_CHUNK = 2048;

struct DispArgs {
    const void *indices;
    int idx64;
    int pairs, k, E, base;
    int chunk, nchunks;
    int *hist;  // [nchunks, E] when nchunks > 1
    int *offsets, *tokens, *slots;
};

__device__ __forceinline__ int disp_expert(const DispArgs &p, int i) {
    const long long e = (p.idx64 ? ((const long long *)p.indices)[i] : (long long)((const int *)p.indices)[i]) - p.base;
    return e >= 0 && e < p.E ? (int)e : -1;
}

// per-warp counts of a chunk into cnt[warp][E]
__device__ __forceinline__ void disp_count(const DispArgs &p, int lo, int hi, int *cnt) {
    const int lane = threadIdx.x & 31;
    for (int e = lane; e < p.E; e += 32) cnt[e] = 0;
    __syncwarp();
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        const int e = i < hi ? disp_expert(p, i) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && lane == __ffs(same) - 1) cnt[e] += __popc(same);
        __syncwarp();
    }
}

__global__ void __launch_bounds__(32 * DISP_WARPS) k_dispatch_count(const __grid_constant__ DispArgs p) {
    __shared__ int cnt[DISP_WARPS][DISP_MAX_E];
    const int warp = threadIdx.x >> 5;
    const int run = p.chunk / DISP_WARPS;
    const int lo = min(p.pairs, blockIdx.x * p.chunk + warp * run), hi = min(p.pairs, lo + run);
    disp_count(p, lo, hi, cnt[warp]);
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
        int n = 0;
#pragma unroll
        for (int w = 0; w < DISP_WARPS; ++w) n += cnt[w][e];
        p.hist[(size_t)blockIdx.x * p.E + e] = n;
    }
}

__global__ void __launch_bounds__(32 * DISP_WARPS) k_dispatch_place(const __grid_constant__ DispArgs p) {
    __shared__ int cnt[DISP_WARPS][DISP_MAX_E];
    __shared__ int total[DISP_MAX_E + 1], scan[DISP_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int run = p.chunk / DISP_WARPS;
    const int lo = min(p.pairs, blockIdx.x * p.chunk + warp * run), hi = min(p.pairs, lo + run);
    disp_count(p, lo, hi, cnt[warp]);
    __syncthreads();
    // each warp's start within the expert, relative to the expert's first row
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
        int before = 0, all = 0;
        if (p.nchunks > 1) {
            for (int c = 0; c < p.nchunks; ++c) {
                const int n = p.hist[(size_t)c * p.E + e];
                if (c < (int)blockIdx.x) before += n;
                all += n;
            }
        }
#pragma unroll
        for (int w = 0; w < DISP_WARPS; ++w) {
            const int n = cnt[w][e];
            cnt[w][e] = before;
            before += n;
        }
        total[e] = p.nchunks > 1 ? all : before;
    }
    __syncthreads();
    // exclusive scan of the experts' totals: two neighbouring experts per thread
    {
        const int e0 = 2 * threadIdx.x;
        const int a = e0 < p.E ? total[e0] : 0, b = e0 + 1 < p.E ? total[e0 + 1] : 0;
        int incl = a + b;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        int at = incl - a - b;
        for (int w = 0; w < warp; ++w) at += scan[w];
        if (e0 <= p.E) total[e0] = at;
        if (e0 + 1 <= p.E) total[e0 + 1] = at + a;
        if (threadIdx.x == blockDim.x - 1 && p.E == DISP_MAX_E) total[p.E] = at + a + b;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= p.E; e += blockDim.x) p.offsets[e] = total[e];
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        const int e = i < hi ? disp_expert(p, i) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        int at = 0;
        if (e >= 0) at = cnt[warp][e];
        __syncwarp();
        if (e >= 0 && lane == __ffs(same) - 1) cnt[warp][e] = at + __popc(same);
        __syncwarp();
        if (i < hi) {
            int r = -1;
            if (e >= 0) {
                r = total[e] + at + __popc(same & ((1u << lane) - 1));
                p.tokens[r] = i / p.k;
            }
            p.slots[i] = r;
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
    for (int i = 0; i < p.k; ++i) {
        const int s = slot[i];
        if (s < 0 || s >= p.R) continue;
        const uint4 a = __ldg(p.rows + (size_t)s * p.chunks + c);
        const float w = weight[i];
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = bf2(u[j]);
            acc[2 * j] += w * f.x;
            acc[2 * j + 1] += w * f.y;
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

int launched(const char *what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? WF_OK : cuda_fail(e, what);
}

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
    p.eps = eps; p.inv_d = 1.0f / (float)D; p.chunks = (int)(D / 8);
    p.weight_bf16 = weight_bf16 != 0; p.ue8m0 = ue8m0 != 0; p.s_f32 = scale_kind == WF_SCALE_F32;
    const int ch = (p.chunks + 255) / 256;
    const int nt = ch > 1 ? 256 : (p.chunks + 31) / 32 * 32;
    const unsigned g = (unsigned)T;
    cudaStream_t st = (cudaStream_t)stream;
    switch (ch) {
        case 1: k_rms_norm_quant<1><<<g, nt, 0, st>>>(p); break;
        case 2: k_rms_norm_quant<2><<<g, nt, 0, st>>>(p); break;
        case 3: case 4: k_rms_norm_quant<4><<<g, nt, 0, st>>>(p); break;
        default: k_rms_norm_quant<8><<<g, nt, 0, st>>>(p); break;
    }
    wf::host::counted();
    return launched("rms_norm_quant launch");
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
    const unsigned g = (unsigned)((T + ROUTE_WARPS - 1) / ROUTE_WARPS);
    cudaStream_t st = (cudaStream_t)stream;
    const int per = (E + 31) / 32;
    if (per <= 2) k_route_topk<2><<<g, 32 * ROUTE_WARPS, 0, st>>>(p);
    else if (per <= 4) k_route_topk<4><<<g, 32 * ROUTE_WARPS, 0, st>>>(p);
    else if (per <= 8) k_route_topk<8><<<g, 32 * ROUTE_WARPS, 0, st>>>(p);
    else k_route_topk<16><<<g, 32 * ROUTE_WARPS, 0, st>>>(p);
    wf::host::counted();
    return launched("route_topk launch");
}

static int disp_chunks(int64_t pairs, int *chunk) {
    int64_t c = DISP_CHUNK;
    if (pairs > c * DISP_MAX_CHUNKS) {
        c = (pairs + DISP_MAX_CHUNKS - 1) / DISP_MAX_CHUNKS;
        c = (c + 32 * DISP_WARPS - 1) / (32 * DISP_WARPS) * (32 * DISP_WARPS);
    }
    *chunk = (int)c;
    return (int)((pairs + c - 1) / c);
}

size_t wf_expert_dispatch_workspace_bytes(int64_t T, int32_t topk, int32_t n_experts) {
    if (T <= 0 || topk <= 0 || topk > ROUTE_MAX_K || T > (1 << 30) || T * topk > (1 << 30) || n_experts <= 0 ||
        n_experts > DISP_MAX_E) {
        fail(WF_E_SHAPE, "need topk in 1..16, T * topk in 1..2^30 and n_experts in 1..512");
        return 0;
    }
    int chunk;
    const int n = disp_chunks(T * topk, &chunk);
    return n > 1 ? (size_t)n * n_experts * 4 : 16;
}

int wf_expert_dispatch(const void *indices, int32_t indices_64, int64_t T, int32_t topk, int32_t n_experts,
                       int64_t expert_offset, int32_t *offsets, int32_t *tokens, int32_t *slots, void *workspace,
                       size_t workspace_bytes, void *stream) {
    if (!indices || !offsets || !tokens || !slots || !workspace) return fail(WF_E_ARG, "null pointer");
    const size_t need = wf_expert_dispatch_workspace_bytes(T, topk, n_experts);
    if (!need) return WF_E_SHAPE;
    if (expert_offset < 0 || expert_offset > 0x7fffffff - DISP_MAX_E) return fail(WF_E_SHAPE, "expert_offset out of range");
    if (workspace_bytes < need)
        return fail(WF_E_ARG, "workspace too small (see wf_expert_dispatch_workspace_bytes)");
    if (misaligned(indices, indices_64 ? 8 : 4) || misaligned(offsets, 4) || misaligned(tokens, 4) ||
        misaligned(slots, 4) || misaligned(workspace, 4))
        return fail(WF_E_ARG, "misaligned pointer");
    DispArgs p;
    p.indices = indices; p.idx64 = indices_64 != 0; p.pairs = (int)(T * topk); p.k = topk; p.E = n_experts;
    p.base = (int)expert_offset; p.hist = (int *)workspace; p.offsets = offsets; p.tokens = tokens; p.slots = slots;
    p.nchunks = disp_chunks(p.pairs, &p.chunk);
    cudaStream_t st = (cudaStream_t)stream;
    if (p.nchunks > 1) {
        k_dispatch_count<<<p.nchunks, 32 * DISP_WARPS, 0, st>>>(p);
        wf::host::counted();
    }
    k_dispatch_place<<<p.nchunks, 32 * DISP_WARPS, 0, st>>>(p);
    wf::host::counted();
    return launched("expert_dispatch launch");
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
    k_combine<<<g, nt, 0, (cudaStream_t)stream>>>(p);
    wf::host::counted();
    return launched("expert_combine launch");
}

}  // extern "C"
