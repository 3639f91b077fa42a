// What the operators over a key/value cache share: lengths, launches with an early start, warp sums.
#pragma once

#include "../../include/bittorch_b200_cache.h"
#include "common.cuh"

namespace bt {

// Per-sequence filled slots, int32 or int64, possibly one value for the whole batch (stride 0).
struct Lengths {
    const void* ptr;
    int64_t stride;
    int i64;
    // clamped to [0, limit]
    __device__ __forceinline__ int at(int b, int limit) const {
        const int64_t n = i64 ? static_cast<const int64_t*>(ptr)[b * stride] : static_cast<const int32_t*>(ptr)[b * stride];
        return static_cast<int>(n < 0 ? 0 : n > limit ? limit : n);
    }
};

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over a warp of a value per lane; every lane gets it.
__device__ __forceinline__ int warp_add(int v) {
#ifdef BT_SIMT_HOST
    return warp_sum(v);
#else
    return __reduce_add_sync(0xffffffffu, v);
#endif
}
// Threads that share a row of `units` pieces when a row is copied: a power of two, at most a warp.
inline int row_lanes_log2(int units) {
    int lg = 0;
    while (lg < 5 && (1 << lg) < units) ++lg;
    return lg;
}

__device__ __forceinline__ float exp2_fast(float x) {              // 2 ulp; -infinity gives 0
#ifdef BT_SIMT_HOST
    return exp2f(x);
#else
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
#endif
}

// Launch that may start while its predecessor on the stream drains; the kernel calls pdl_wait() before it touches
// global memory, so the call is stream-ordered like any other.
template <typename Kern, typename Params>
static int launch_early(Kern kern, const char* name, dim3 grid, int threads, size_t smem, void* stream, const Params& p) {
#ifdef BT_SIMT_HOST
    (void)stream;
    const int rc = ::simt::launch(kern, grid, dim3(threads), smem, p);
    if (rc != BT_OK) set_error("%s: %s", name, ::simt::error_text());
    return rc;
#else
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("launch of %s failed: %s", name, cudaGetErrorString(e));
        return BT_ERR_CUDA;
    }
    return BT_OK;
#endif
}

}  // namespace bt
