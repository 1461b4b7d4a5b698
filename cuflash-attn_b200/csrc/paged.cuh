#pragma once

// Shared by the paged-cache serving kernels (append, ragged attention,
// shared-prefix decode): the sequence a token belongs to.

#include <cuda_runtime.h>

namespace cuflash {
namespace detail {

// A length read from device memory, clamped to [0, most].
__host__ __device__ __forceinline__ int clamp_len(int n, int most) {
    return n < 0 ? 0 : (n < most ? n : most);
}

// Keys of a sequence of `len` that a token sees, the from_end-th from its end: at
// most len, also where offsets that do not ascend put a token behind the end (its
// keys would lie behind the table).
__host__ __device__ __forceinline__ int visible_keys(int len, int from_end, int causal) {
    return causal && from_end > 1 ? len - (from_end - 1) : len;
}

#ifdef __CUDACC__
// Launches `kern` so that its blocks may be scheduled while the kernel before
// it on the stream still runs: every thread calls stream_wait() before it
// touches global memory, and none returns without.  Between calls of a serving
// step this hides the launch and the set-up of a kernel.
template <typename... Params, typename... Args>
inline cudaError_t launch_behind(void (*kern)(Params...), dim3 grid, int threads, size_t smem,
                                 cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}
__device__ __forceinline__ void stream_wait() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
// the next kernel's blocks may start; it waits for this one's end by itself
__device__ __forceinline__ void stream_release() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Sequence of token t among cu[0..B] (ascending, cu[b] = first token of
// sequence b): the last b with cu[b] <= t < cu[b + 1], or -1 for a token
// outside [cu[0], cu[B]).  Each round the 32 lanes probe 32 evenly spaced
// entries at once, so a batch of up to 1024 sequences takes two dependent
// loads instead of the ten of a binary search.  Every index read lies in
// [0, B] whatever the array holds.  Warp-uniform t and result.
__device__ __forceinline__ int sequence_of_token(const int* __restrict__ cu, int B, int t) {
    const int lane = threadIdx.x & 31;
    const int edge = cu[lane == 0 ? 0 : B];
    const bool outside = lane == 0 ? t < edge : t >= edge;
    if (__any_sync(0xffffffffu, outside)) return -1;
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int idx = lo + (lane + 1) * step;
        const bool below = idx < hi && cu[idx] <= t;
        const int n = __popc(__ballot_sync(0xffffffffu, below));
        lo += n * step;
        hi = min(hi, lo + step);
    }
    return lo;
}
#endif

}  // namespace detail
}  // namespace cuflash
