// wf_tcgen05.cuh - tcgen05 (5th-generation tensor core) building blocks for sm_100a:
// TMEM allocation, block-scaled MMA (kind::mxf8f6f4.block_scale), tensor-memory
// loads/stores, commit-to-mbarrier, 2D tiled TMA loads, and the shared-memory
// matrix / instruction descriptors.
//
// Operand conventions used by the kernels:
//   A = weight rows (M = 128 per MMA), K-major, 128-byte swizzled rows in
//       shared memory, loaded by TMA: E2M1 through the unpacking tensor-map
//       type 16U4_ALIGN16B (16 packed nibbles + 8 zero bytes per 16-byte
//       chunk, 1 byte per element on average), E4M3 as plain bytes;
//   B = tokens (N = 16 or 32 per MMA), E4M3, K-major, same swizzle, written by
//       the worker warps after quantizing activations;
//   D = f32 accumulator in TMEM: lane = weight row, column = token;
//   scale factors (UE8M0, one per 32 K) in TMEM, 4 consecutive K-blocks of one
//       row packed in one 32-bit column word; for 128 rows the word of row
//       r = r0 + 32*r1 sits at lane r0 (replicated in all 4 lane quadrants),
//       column base + r1.  The MMA picks the byte with the descriptor's sf_id.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "wf_ptx.cuh"

namespace wf {
namespace tc {

// ---- TMEM allocation (one warp) -----------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t *dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(dst_smem)),
                 "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
                 : "memory");
}

// ---- ordering of tcgen05 operations around thread synchronization ------
__device__ __forceinline__ void fence_before_sync() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after_sync() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// ---- block-scaled MMA: D[tmem] (+)= A[smem] x B[smem], scales in TMEM ----
__device__ __forceinline__ void mma_mxf8f6f4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t sfa_tmem, uint32_t sfb_tmem,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
        : "memory");
}

// Arrive on `bar` once every tcgen05 operation this thread issued so far is complete.
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
            smem_u32(bar))
        : "memory");
}

// ---- TMEM <-> registers (a warp accesses the 32 lanes of its quadrant) --
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
          "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c,
                                         uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr),
                 "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// ---- 2D tiled TMA load, completion on an mbarrier -----------------------
__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, int c0, int c1,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
        : "memory");
}

// 3D tiled TMA load, completion on an mbarrier.
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int c0, int c1, int c2,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

// L2 policy for streamed weights: evict first, so a layer step's ~1 GB of weights
// passing through the 126 MB L2 does not displace the kernels' instructions, the
// routing tables and the activations, which are read again.
__device__ __forceinline__ uint64_t policy_evict_first() {
    uint64_t pol;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
    return pol;
}

// tma_load_2d / tma_load_3d with an L2 cache policy.
__device__ __forceinline__ void tma_load_2d_hint(void *dst, const CUtensorMap *map, int c0, int c1, uint64_t *bar,
                                                 uint64_t pol) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar)), "l"(pol)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d_hint(void *dst, const CUtensorMap *map, int c0, int c1, int c2,
                                                 uint64_t *bar, uint64_t pol) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar)), "l"(pol)
        : "memory");
}

// Prefetch one 2D box of the tensor map into L2 (no shared memory, no completion).
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap *map, int c0, int c1) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(c0), "r"(c1)
                 : "memory");
}

// ---- descriptors -------------------------------------------------------------
// Shared-memory matrix descriptor: K-major, 128-byte swizzle, 8-row atoms of
// 1024 bytes (SBO), start address in 16-byte units, descriptor version 1.
__device__ __forceinline__ uint64_t smem_desc_sw128(const void *p) {
    const uint64_t addr = (smem_u32(p) & 0x3ffffu) >> 4;
    uint64_t d = 0;
    d |= addr;                       // [0,14) start address
    d |= (uint64_t)1 << 16;          // [16,30) leading byte offset (16 B, unused for SW128 K-major)
    d |= (uint64_t)(1024 >> 4) << 32;  // [32,46) stride byte offset: 8 rows x 128 B
    d |= (uint64_t)1 << 46;          // [46,48) version
    d |= (uint64_t)2 << 61;          // [61,64) layout: 128-byte swizzle
    return d;
}

// Instruction descriptor of kind::mxf8f6f4.block_scale with UE8M0 scales,
// M = 128, dense, both operands K-major.
//   a_fmt / b_fmt: 0 = E4M3, 5 = E2M1.
__device__ __forceinline__ uint32_t idesc_mxf8f6f4(int a_fmt, int b_fmt, int n, int sf_id) {
    uint32_t d = 0;
    d |= (uint32_t)(sf_id & 3) << 4;   // B scale-factor byte
    d |= (uint32_t)(a_fmt & 7) << 7;
    d |= (uint32_t)(b_fmt & 7) << 10;
    d |= (uint32_t)((n >> 3) & 63) << 17;
    d |= 1u << 23;                     // scale format UE8M0
    d |= (uint32_t)((128 >> 4) & 31) << 24;
    d |= (uint32_t)(sf_id & 3) << 29;  // A scale-factor byte
    return d;
}

// Byte offset inside a 128-byte-swizzled K-major tile of the 16-byte chunk
// `chunk` (0..7) of row `row`.
__device__ __forceinline__ uint32_t sw128_offset(int row, int chunk) {
    return (uint32_t)row * 128u + (uint32_t)((chunk ^ (row & 7)) << 4);
}

}  // namespace tc
}  // namespace wf
