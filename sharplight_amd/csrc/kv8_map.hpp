// Which work item belongs to which request of a serving step (slhip_kv8_batch), on host and device.
//
// The lengths live on the device, so a launch is sized from what the host knows -- T rows, B requests -- and each item
// finds its request from the step's `starts`. Request i with n rows from starts[i] is cut into pieces of `tile` rows; its
// first item is item_base = starts[i] / tile + extra * i, which leaves at least n / tile + extra items before the next
// request's first one. With extra = 1 that holds its ceil(n / tile) pieces from row 0; with extra = 2 also the
// blocks of `tile` positions that n tokens can touch when they begin inside a block. Items behind a request's last piece
// have nothing to do.
#pragma once

#include <stdint.h>

#if defined(__HIP__) || defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define SLHIP_HD __host__ __device__ __forceinline__
#else
#define SLHIP_HD inline
#endif

namespace slhip {

SLHIP_HD int64_t item_base(int64_t start, int64_t i, int64_t tile, int64_t extra) { return start / tile + extra * i; }

// Items of a launch over T rows of B requests: no base + pieces goes past it.
SLHIP_HD int64_t item_count(int64_t T, int64_t B, int64_t tile, int64_t extra) { return T / tile + extra * B; }

// Whether a request of the step is one the kernels may work on: rows [s0, s1) of T, `past` cached tokens, slot `slot` of
// page_slots table rows that hold `row_tokens` tokens each.
SLHIP_HD bool request_fits(int64_t s0, int64_t s1, int64_t T, int64_t past, int64_t slot, int64_t page_slots, int64_t row_tokens)
{
    return s0 >= 0 && s1 >= s0 && s1 <= T && past >= 0 && past + (s1 - s0) <= row_tokens && slot >= 0 && slot < page_slots;
}

// The largest request i of [0, B) whose first item is at or below `item` (0 if none is), by halving.
template <class Starts>
SLHIP_HD int64_t item_request(const Starts& starts, int64_t B, int64_t item, int64_t tile, int64_t extra)
{
    int64_t lo = 0, n = B;
    while (n > 1) {
        const int64_t half = n / 2;
        if (item_base(starts(lo + half), lo + half, tile, extra) <= item) {
            lo += half;
            n -= half;
        } else {
            n = half;
        }
    }
    return lo;
}

}  // namespace slhip
