// The requests of a serving step, as the operators that work request by request look them up.
#pragma once

#include "common.hpp"

namespace slhip {

// The request of row t: the last one of [0, B) that begins at or before it (which is the one with rows there, where some have
// none). By a whole wave, 64 requests a look: up to 64 take one memory latency, 4096 two. Wave-uniform.
__device__ __forceinline__ int32_t row_request(const int32_t* starts, int32_t B, int64_t t)
{
    int32_t lo = 0, n = B;
    const int lane = threadIdx.x & 63;
    while (n > 64) {
        const int32_t step = (n + 63) / 64, i = lo + lane * step;
        const int32_t k = __popcll(__ballot(i < lo + n && starts[i < lo + n ? i : lo] <= t));
        if (k > 0) {
            lo += (k - 1) * step;
            n -= (k - 1) * step;
        }
        n = min(n, step);
    }
    const int32_t k = __popcll(__ballot(lane < n && starts[lo + (lane < n ? lane : 0)] <= t));
    return __builtin_amdgcn_readfirstlane(lo + max(k - 1, 0));
}

// A 16-byte load from any address: global memory takes it at any alignment.
__device__ __forceinline__ uint4 load_any(const void* p)
{
    uint4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

}  // namespace slhip
