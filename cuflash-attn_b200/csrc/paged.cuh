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

#ifdef __CUDACC__
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
