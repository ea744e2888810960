// wf_host.h - host-side services of the library shared by its translation units
// (defined in wf_moe.cu, which holds the error message and the launch counter).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace wf {
namespace host {

// Records `msg` as the calling thread's last error and returns `code`.
int fail(int code, const char *msg) noexcept;
int cuda_fail(cudaError_t e, const char *what) noexcept;
// Adds n to the count of launched kernels.
void counted(int n = 1) noexcept;
// SMs of the current device (0 without one).
int sm_count() noexcept;
// Bound of the kernels' waits on another role's progress (wf_set_wait_limit).
long long wait_limit() noexcept;

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                  const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// cuTensorMapEncodeTiled through the runtime's driver entry point (NULL when unavailable).
EncodeTiledFn encode_fn() noexcept;

// Lets `kernel` use `bytes` of dynamic shared memory on the current device: set once per device and
// `which` (0..63, the caller's own number for the kernel; the attribute is the function's, whichever
// thread sets it).
inline cudaError_t allow_smem(const void *kernel, int which, size_t bytes, std::atomic<uint64_t> (&done)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << which;
    if (dev < 64 && (done[dev].load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) done[dev].fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Launches `kernel` so that it may start while the kernel before it on the stream drains
// (programmatic dependent launch).  Every CTA of `kernel` executes griddepcontrol.wait before it
// touches global memory, so the order of the stream holds for what it reads and writes.  One
// exception: k_dispatch_place behind k_dispatch_count reads the indices before its wait.  Only the
// first kernel of an operator's two lets the next start early (griddepcontrol.launch_dependents),
// and it must do so behind its own wait, when all before it is done: that exception rests on it.
// The framework's products read their weights ahead of their wait, so no kernel whose output a
// caller may pass on lets the next start early.
template <class... P, class... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    counted();
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace host
}  // namespace wf
