// The 8-bit paged KV cache as its kernels take it: requests of a step, blocks, codes.
#pragma once

#include "common.hpp"
#include "kv8_map.hpp"

namespace slhip {

struct Kv8Dev {
    uint8_t *k, *v;
    float *ks, *vs;
    int32_t blocks, shift, heads, D;  // shift: log2(block_size)
    int32_t B;
    int64_t T;
    const int32_t *starts, *past, *slots, *pages;
    int64_t page_slots, bps;
    uint32_t* err;
};

// Checks what the host can see of a cache and a batch (kv8_write.hip) and fills `out`.
int make_kv8(const char* op, const slhip_kv8_cache* c, const slhip_kv8_batch* b, Kv8Dev* out);

// A request of the step. n = 0 where it has no rows or does not fit (bad).
struct Kv8Request {
    int32_t first, n, past, slot;
    bool bad;
    const int32_t* table;
};

__device__ __forceinline__ Kv8Request kv8_request(const Kv8Dev& d, int32_t i)
{
    Kv8Request r;
    const int32_t s0 = d.starts[i], s1 = d.starts[i + 1];
    r.past = d.past[i];
    r.slot = d.slots ? d.slots[i] : i;
    r.bad = !request_fits(s0, s1, d.T, r.past, r.slot, d.page_slots, d.bps << d.shift);
    r.first = s0;
    r.n = r.bad ? 0 : s1 - s0;
    r.table = d.pages + (r.bad ? 0 : r.slot * d.bps);
    return r;
}

__device__ __forceinline__ void raise_request(const Kv8Dev& d, int32_t i, const Kv8Request& r)
{
    const int64_t n = static_cast<int64_t>(d.starts[i + 1]) - d.starts[i];
    raise_error(d.err, kErrKvRequest, i, r.slot, r.past, static_cast<uint32_t>(n), static_cast<uint32_t>(static_cast<uint64_t>(n) >> 32), 0);
}

__device__ __forceinline__ void raise_block(const Kv8Dev& d, int32_t row, int32_t slot, int32_t pos, int32_t block)
{
    const int64_t v = block;
    raise_error(d.err, kErrCacheBlock, row, slot, pos, static_cast<uint32_t>(v), static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32),
                static_cast<uint32_t>(static_cast<int64_t>(d.blocks) << d.shift));
}

// The request of an item, and which of its items that is.
struct Kv8Item {
    int32_t i;
    int64_t piece;  // below 0 or past the request's pieces where there is nothing to do
    Kv8Request r;
};

// item_request by a whole wave: 64 requests are looked at a step, and the last step brings the request itself, so up to 64
// take one memory latency and 4096 two. Wave-uniform.
__device__ __forceinline__ Kv8Item kv8_find(const Kv8Dev& d, int64_t item, int64_t tile, int64_t extra)
{
    int32_t lo = 0, n = d.B;
    const int lane = threadIdx.x & 63;
    while (n > 64) {
        const int32_t step = (n + 63) / 64, i = lo + lane * step;
        const bool under = i < lo + n && item_base(d.starts[i < lo + n ? i : lo], i, tile, extra) <= item;
        const int32_t k = __popcll(__ballot(under));
        if (k > 0) {
            lo += (k - 1) * step;
            n -= (k - 1) * step;
        }
        n = min(n, step);
    }
    const int32_t i = lo + (lane < n ? lane : 0);
    const Kv8Request mine = kv8_request(d, i);
    const int32_t start = d.starts[i];
    const int32_t k = max(__popcll(__ballot(lane < n && item_base(start, i, tile, extra) <= item)) - 1, 0);
    Kv8Item f;
    f.i = __builtin_amdgcn_readfirstlane(lo) + k;
    f.piece = item - item_base(__builtin_amdgcn_readlane(start, k), f.i, tile, extra);
    f.r.first = __builtin_amdgcn_readlane(mine.first, k);
    f.r.n = __builtin_amdgcn_readlane(mine.n, k);
    f.r.past = __builtin_amdgcn_readlane(mine.past, k);
    f.r.slot = __builtin_amdgcn_readlane(mine.slot, k);
    f.r.bad = __builtin_amdgcn_readlane(static_cast<int>(mine.bad), k) != 0;
    f.r.table = d.pages + (f.r.bad ? 0 : f.r.slot * d.bps);
    return f;
}

}  // namespace slhip
