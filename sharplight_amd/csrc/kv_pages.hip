// Block tables and slot maps of a serving step, from request lengths on the device (slhip_kv_pages_advance / _trim / _release).
//
// Mathematics: two prefix sums over the requests -- of their new tokens (starts) and of the blocks those need (which ids
// of the free list are theirs) -- then one write per taken block and one row per token. Nothing here moves enough bytes to
// matter (20 a token); what a call costs is its launch and the chain load lengths -> scan -> load table -> store. So a
// thread block of 1024 does it all, with the sums and the slots seen (a bit each, for the duplicate check) in LDS, and
// decides over the whole step before it writes anything: all or nothing needs no second pass. Steps of more rows than it
// writes in the time of a launch (kBlockRows) take more thread blocks, each of which scans the lengths again and takes its
// share of the rows; the first one alone writes the tables. A new block's id comes from the free list, an old one's from the
// table, so no thread block waits for another's stores. Only the free list's count can be written where it is read (in
// place); a step of many rows then has its rows in a second launch.
// Measured: 64 requests of a token 4.4 us, 333 requests of 1 to 200 tokens (some 33000 rows) 6.2 us; an empty launch takes 2.5.
// With kBlockRows = 4096 the latter took 10.4 us, and with the rows in a second launch 10.0. A release is one thread block's too: 64
// requests of 256 blocks 7.5 us, of 8192 412.
// A trim is a release that leaves each request's first blocks, and it fills the stack from the other end, so that it undoes an
// advance. Its few blocks' chain is the release's: lengths -> scan -> table entries -> stores. 64 requests with up to 4 refused drafts each 3.3 us,
// 333 that give back 10400 blocks 7.9 (with a search of each block's request in the sums, of ten steps, 10.2).
#include <type_traits>

#include "common.hpp"
#include "kv8_map.hpp"

namespace slhip {

constexpr int kPagesThreads = 1024;
constexpr int kMaxRequests = 4096;
constexpr int kMaxSlots = 131072;
constexpr int64_t kBlockRows = 1024;
constexpr int kListed = 16 * kPagesThreads;  // blocks that a release looks up at once

struct KvPagesArgs {
    int32_t B;
    const int32_t *past, *count, *slots;
    int32_t* pages;
    int64_t page_slots, bps;
    int32_t shift;  // log2(block_size)
    int32_t* free_blocks;
    int64_t capacity;
    const int32_t* n_free;
    int32_t* n_free_out;
    int64_t tokens;
    int32_t *starts, *seq, *pos;
    int64_t block_rows;  // rows of a thread block (0: none here)
    uint32_t* err;
};

enum : uint32_t { kBadLength = 1, kBadSlot = 2, kBadRows = 3, kBadFree = 4, kBadEntry = 5 };

__device__ __forceinline__ int64_t blocks_of(int64_t tokens, int shift) { return (tokens + (int64_t{1} << shift) - 1) >> shift; }

__device__ __forceinline__ void store_row(const KvPagesArgs& a, int64_t t, int32_t slot, int32_t pos, int32_t i, int32_t block)
{
    if (a.seq) {
        int32_t* s = a.seq + t * 4;
        if ((reinterpret_cast<uintptr_t>(a.seq) & 15u) == 0) {
            *reinterpret_cast<int4*>(s) = make_int4(slot, pos, i, block);
        } else {
            s[0] = slot;
            s[1] = pos;
            s[2] = i;
            s[3] = block;
        }
    }
    if (a.pos) a.pos[t] = max(pos, 0);
}

// Inclusive sums over the wave of numbers below 2^32, in 64 bits: the halves of 16 bits apart.
__device__ __forceinline__ int64_t wave_scan_wide(uint32_t v)
{
    return (static_cast<int64_t>(wave_scan(v >> 16)) << 16) + wave_scan(v & 0xFFFF);
}

enum { kAdvance = 0, kRelease = 1, kTrim = 2 };

template <int OP>
__global__ __launch_bounds__(kPagesThreads) void kv_pages_tables(KvPagesArgs a)
{
    constexpr bool RELEASE = OP != kAdvance, COUNTS = OP != kRelease;  // blocks go back; requests have a count
    __shared__ int32_t s_start[kMaxRequests + 1], s_off[kMaxRequests + 1];
    __shared__ uint32_t s_seen[kMaxSlots / 32];  // (of as many words as there are requests at most)
    static_assert(kMaxSlots / 32 >= kMaxRequests);
    __shared__ uint32_t s_bits[RELEASE ? kListed / 32 : 1];  // of blocks that go back: a request's first one
    __shared__ int32_t s_base[RELEASE ? kListed / 32 : 1];   // bits in the words before
    __shared__ uint16_t s_list[RELEASE ? kMaxRequests : 1];  // the requests of the bits
    __shared__ int64_t s_wave[2][kPagesThreads / 64];
    __shared__ uint32_t s_bad;  // the first bad request * 8 + what is wrong with it
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int64_t n_free = *a.n_free;
    const int per = (a.B + kPagesThreads - 1) / kPagesThreads;
    const int i0 = min(tid * per, a.B), i1 = min(i0 + per, a.B);
    const int64_t row_tokens = a.bps << a.shift;
    const auto slot_of = [&](int i) { return a.slots ? a.slots[i] : i; };
    // the thread's first request: most steps have no more than one a thread
    const int32_t past0 = i0 < i1 ? a.past[i0] : 0, count0 = i0 < i1 && COUNTS ? a.count[i0] : 0, slot0 = i0 < i1 ? slot_of(i0) : 0;
    for (int64_t w = tid; w < (a.page_slots + 31) / 32; w += kPagesThreads) s_seen[w] = 0;
    if (RELEASE && tid < kListed / 32) s_bits[tid] = 0;
    if (tid == 0) s_bad = 0xFFFFFFFFu;
    __syncthreads();

    // the blocks that a request takes or gives back
    const auto moved = [&](int64_t past, int64_t count) {
        return OP == kRelease ? blocks_of(past, a.shift) : blocks_of(past + count, a.shift) - blocks_of(past, a.shift);
    };
    // sums of the thread's requests: four of below 2^31 each at most, cut off below at 2^32 - 1, which no step takes
    int64_t tokens = 0, blocks = 0;
    for (int i = i0; i < i1; i++) {
        const int64_t past = i == i0 ? past0 : a.past[i], count = !COUNTS ? 0 : i == i0 ? count0 : a.count[i], slot = i == i0 ? slot0 : slot_of(i);
        uint32_t bad = 0;
        if (slot < 0 || slot >= a.page_slots || (atomicOr(&s_seen[slot >> 5], 1u << (slot & 31)) >> (slot & 31) & 1u)) bad = kBadSlot;
        if (past < 0 || count < 0 || past + count > row_tokens) bad = kBadLength;
        if (bad) {
            atomicMin(&s_bad, static_cast<uint32_t>(i) * 8 + bad);
        } else {
            tokens += count;
            blocks += moved(past, count);
        }
    }
    const int64_t most = 0xFFFFFFFF;  // more than any step has rows or any list has room for
    const int64_t ct = min(tokens, most), co = min(blocks, most);
    int64_t st = wave_scan_wide(static_cast<uint32_t>(ct)), so = wave_scan_wide(static_cast<uint32_t>(co));
    if (lane == 63) {
        s_wave[0][wave] = st;
        s_wave[1][wave] = so;
    }
    __syncthreads();
    st -= ct;
    so -= co;
    int64_t all_tokens = 0, all_blocks = 0;
    for (int w = 0; w < kPagesThreads / 64; w++) {
        if (w == wave) {
            st += all_tokens;
            so += all_blocks;
        }
        all_tokens += s_wave[0][w];
        all_blocks += s_wave[1][w];
    }
    uint32_t bad = s_bad;
    if (bad == 0xFFFFFFFFu) {
        const bool room = n_free >= 0 && n_free <= a.capacity && (RELEASE ? n_free + all_blocks <= a.capacity : all_blocks <= n_free);
        if (!RELEASE && all_tokens > a.tokens) bad = kBadRows;
        else if (!room) bad = kBadFree;
    }
    const bool first = blockIdx.x == 0;
    bool ok = bad == 0xFFFFFFFFu;
    if (!ok) all_tokens = all_blocks = 0;
    for (int i = i0; i < i1; i++) {
        s_off[i] = static_cast<int32_t>(so);
        if (RELEASE) {  // block k of all is request i's entry k + s_seen[i] of table row s_start[i]
            s_start[i] = i == i0 ? slot0 : slot_of(i);
            s_seen[i] = static_cast<uint32_t>((OP == kTrim ? blocks_of(i == i0 ? past0 : a.past[i], a.shift) : 0) - so);
        } else {
            s_start[i] = static_cast<int32_t>(st);
        }
        if (!RELEASE && first) a.starts[i] = ok ? static_cast<int32_t>(st) : 0;
        if (!ok) continue;
        const int64_t past = i == i0 ? past0 : a.past[i], count = !COUNTS ? 0 : i == i0 ? count0 : a.count[i];
        const int64_t blocks_here = moved(past, count);
        if (RELEASE && blocks_here > 0 && all_blocks <= kListed) atomicOr(&s_bits[so >> 5], 1u << (so & 31));
        st += count;
        so += blocks_here;
    }
    if (!RELEASE && first && tid == 0) a.starts[a.B] = static_cast<int32_t>(all_tokens);
    __syncthreads();
    const auto request_of = [&](const int32_t* sums, int64_t k) {
        return static_cast<int32_t>(item_request([&](int64_t r) { return sums[r]; }, a.B, k, 1, 0));
    };
    const auto entry_at = [&](int32_t i, int64_t k) { return a.pages + s_start[i] * a.bps + (k + static_cast<int32_t>(s_seen[i])); };
    // where block k of all goes on the stack
    const auto place = [&](int64_t k) { return n_free + (OP == kTrim ? all_blocks - 1 - k : k); };
    // What goes back has to be there (a request that was released before has no entries), so all entries are looked at before one is
    // moved: none, if the thread's first block that is not there (none of all: all_blocks) is below.
    const auto decide = [&](int64_t none) {
        if (none < all_blocks) atomicMin(&s_bad, static_cast<uint32_t>(request_of(s_off, none)) * 8 + kBadEntry);
        __syncthreads();
        bad = s_bad;
        ok = bad == 0xFFFFFFFFu;
    };
    const auto report = [&]() {
        if (!first || tid != 0) return;
        if (!ok) {
            const int i = min(static_cast<int>(bad >> 3), a.B - 1);
            const int64_t count = !COUNTS || i < 0 ? 0 : a.count[i];
            raise_error(a.err, kErrKvPages, max(i, 0), i < 0 ? 0 : slot_of(i), i < 0 ? 0 : a.past[i], static_cast<uint32_t>(count),
                        static_cast<uint32_t>(static_cast<uint64_t>(count) >> 32), bad & 7);
        }
        *a.n_free_out = static_cast<int32_t>(!ok ? n_free : RELEASE ? n_free + all_blocks : n_free - all_blocks);
    };
    // Up to 16 blocks a thread are looked up once, all searches and loads on their way together (those behind the last look at it again).
    const auto give_back = [&](auto each) __attribute__((always_inline)) {
        constexpr int U = decltype(each)::value;
        int32_t *at[U], entry[U], k[U], i[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            k[u] = static_cast<int32_t>(min(static_cast<int64_t>(tid + u * kPagesThreads), all_blocks - 1));
            i[u] = 0;
        }
        if (U == 1) {
            for (int32_t n = a.B; n > 1; n -= n / 2) i[0] += s_off[i[0] + n / 2] <= k[0] ? n / 2 : 0;  // request_of
        } else {  // a block's request is the one of the last bit up to it: three reads of neighbours, where a search is ten of any
            const int32_t ones = tid < kListed / 32 ? __popc(s_bits[tid]) : 0;
            int32_t up = wave_scan(ones);
            if (lane == 63) s_wave[0][wave] = up;
            __syncthreads();
            for (int w = 0; w < wave && w < kListed / 32 / 64; w++) up += static_cast<int32_t>(s_wave[0][w]);
            if (tid < kListed / 32) s_base[tid] = up - ones;
            __syncthreads();
            const auto bit_of = [&](int32_t at) { return s_base[at >> 5] + __popc(s_bits[at >> 5] & (0xFFFFFFFFu >> (31 - (at & 31)))) - 1; };
            for (int j = i0; j < i1; j++)
                if ((j + 1 < a.B ? s_off[j + 1] : all_blocks) > s_off[j]) s_list[bit_of(s_off[j])] = static_cast<uint16_t>(j);
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; u++) i[u] = s_list[bit_of(k[u])];
        }
#pragma unroll
        for (int u = 0; u < U; u++) at[u] = entry_at(i[u], k[u]);
#pragma unroll
        for (int u = 0; u < U; u++) entry[u] = *at[u];
        int64_t none = all_blocks;
#pragma unroll
        for (int u = U - 1; u >= 0; u--)
            if (tid + u * kPagesThreads < all_blocks && entry[u] < 0) none = tid + u * kPagesThreads;
        decide(none);
        report();
        if (!ok) return;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (tid + u * kPagesThreads >= all_blocks) break;
            a.free_blocks[place(tid + u * kPagesThreads)] = entry[u];
            *at[u] = -1;
        }
    };
    if (RELEASE && ok && all_blocks > 0) {
        if (all_blocks <= kPagesThreads) return give_back(std::integral_constant<int, 1>{});
        if (all_blocks <= 4 * kPagesThreads) return give_back(std::integral_constant<int, 4>{});
        if (all_blocks <= kListed) return give_back(std::integral_constant<int, 16>{});
        // of more, a request is searched for only where the last one's blocks end
        const auto entry_of = [&](int64_t k, int32_t& i) {
            if (i + 1 < a.B && k >= s_off[i + 1]) i = request_of(s_off, k);
            return entry_at(i, k);
        };
        int64_t none = all_blocks;
        int32_t i = 0;
        for (int64_t k = tid; k < all_blocks; k += kPagesThreads)
            if (*entry_of(k, i) < 0) none = min(none, k);
        decide(none);
        report();
        if (!ok) return;
        i = 0;
        for (int64_t k = tid; k < all_blocks; k += kPagesThreads) {
            int32_t* e = entry_of(k, i);
            a.free_blocks[place(k)] = *e;
            *e = -1;
        }
        return;
    }
    report();
    if (RELEASE) return;
    if (first) {
        for (int64_t k = tid; k < all_blocks; k += kPagesThreads) {
            const int32_t i = request_of(s_off, k);
            a.pages[slot_of(i) * a.bps + blocks_of(a.past[i], a.shift) + (k - s_off[i])] = a.free_blocks[n_free - 1 - k];
        }
    }
    const int64_t t1 = min((static_cast<int64_t>(blockIdx.x) + 1) * a.block_rows, a.tokens);
    for (int64_t t = blockIdx.x * a.block_rows + tid; t < t1; t += kPagesThreads) {
        if (t >= all_tokens) {
            store_row(a, t, -1, -1, -1, -1);
            continue;
        }
        const int32_t i = request_of(s_start, t);
        const int32_t past = a.past[i], slot = slot_of(i), pos = past + static_cast<int32_t>(t - s_start[i]);
        const int64_t j = pos >> a.shift, taken = j - blocks_of(past, a.shift);  // a new block's number among the request's
        const int32_t block = taken < 0 ? a.pages[slot * a.bps + j] : a.free_blocks[n_free - 1 - (s_off[i] + taken)];
        store_row(a, t, slot, pos, i, block);
    }
}

// The rows after the tables: a step of many rows whose free list counts in place.
__global__ __launch_bounds__(256) void kv_pages_rows(KvPagesArgs a)
{
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (t >= a.tokens) return;
    if (t >= a.starts[a.B]) {
        store_row(a, t, -1, -1, -1, -1);
        return;
    }
    const int32_t i = static_cast<int32_t>(item_request([&](int64_t r) { return a.starts[r]; }, a.B, t, 1, 0));
    const int32_t slot = a.slots ? a.slots[i] : i, pos = a.past[i] + static_cast<int32_t>(t - a.starts[i]);
    store_row(a, t, slot, pos, i, a.pages[slot * a.bps + (pos >> a.shift)]);
}

// Checks what the host can see of the arguments.
static int make_args(const char* op, int kind, const slhip_kv_pages* p, KvPagesArgs* a)
{
    if (!p) return fail(SLHIP_ERR_INVALID, "%s: arguments are null", op);
    if (p->requests < 0 || p->page_slots < 0 || p->blocks_per_slot < 0 || p->free_capacity < 0 || p->tokens < 0)
        return fail(SLHIP_ERR_INVALID, "%s: negative size", op);
    if (p->requests > kMaxRequests) return fail(SLHIP_ERR_UNSUPPORTED, "%s: more than %d requests", op, kMaxRequests);
    if (p->page_slots > kMaxSlots) return fail(SLHIP_ERR_UNSUPPORTED, "%s: more than %d table rows", op, kMaxSlots);
    if (p->block_size < 1 || p->block_size > (1 << 20) || (p->block_size & (p->block_size - 1)))
        return fail(SLHIP_ERR_INVALID, "%s: block size %lld is not a power of two up to 2^20", op, static_cast<long long>(p->block_size));
    if (p->blocks_per_slot > 0x7FFFFFFF / p->block_size)
        return fail(SLHIP_ERR_UNSUPPORTED, "%s: table rows of 2^31 tokens or more", op);
    if (p->tokens > 0x7FFFFFFF || p->free_capacity > 0x7FFFFFFF) return fail(SLHIP_ERR_UNSUPPORTED, "%s: 2^31 tokens or blocks or more", op);
    if (!p->n_free || !p->n_free_out) return fail(SLHIP_ERR_INVALID, "%s: n_free and n_free_out are required", op);
    if (p->free_capacity > 0 && !p->free_blocks) return fail(SLHIP_ERR_INVALID, "%s: the free list is null", op);
    if (p->requests > 0 && (!p->past || !p->pages || (kind != kRelease && !p->count)))
        return fail(SLHIP_ERR_INVALID, "%s: past, count and pages are required", op);
    if (kind == kAdvance && !p->starts) return fail(SLHIP_ERR_INVALID, "%s: starts is required", op);
    int shift = 0;
    while ((int64_t{1} << shift) < p->block_size) shift++;
    *a = KvPagesArgs{static_cast<int32_t>(p->requests), p->past, p->count, p->slots, p->pages, p->page_slots, p->blocks_per_slot,
                     shift, p->free_blocks, p->free_capacity, p->n_free, p->n_free_out, p->tokens, p->starts, p->seq, p->pos,
                     0, nullptr};
    return error_word(&a->err);
}

}  // namespace slhip

using namespace slhip;

extern "C" SLHIP_API int slhip_kv_pages_advance(const slhip_kv_pages* p, slhip_stream stream)
{
    KvPagesArgs a;
    const int e = make_args("kv_pages_advance", kAdvance, p, &a);
    if (e) return e;
    const bool rows = a.tokens > 0 && (a.seq || a.pos), apart = rows && a.tokens > kBlockRows && a.n_free == a.n_free_out;
    a.block_rows = rows && !apart ? kBlockRows : 0;
    const int64_t grid = a.block_rows ? (a.tokens + kBlockRows - 1) / kBlockRows : 1;
    kv_pages_tables<kAdvance><<<static_cast<unsigned>(grid), kPagesThreads, 0, to_stream(stream)>>>(a);
    const int s = check_launch("kv_pages_tables");
    if (s || !apart) return s;
    kv_pages_rows<<<static_cast<unsigned>((a.tokens + 255) / 256), 256, 0, to_stream(stream)>>>(a);
    return check_launch("kv_pages_rows");
}

extern "C" SLHIP_API int slhip_kv_pages_release(const slhip_kv_pages* p, slhip_stream stream)
{
    KvPagesArgs a;
    const int e = make_args("kv_pages_release", kRelease, p, &a);
    if (e) return e;
    kv_pages_tables<kRelease><<<1, kPagesThreads, 0, to_stream(stream)>>>(a);
    return check_launch("kv_pages_tables");
}

extern "C" SLHIP_API int slhip_kv_pages_trim(const slhip_kv_pages* p, slhip_stream stream)
{
    KvPagesArgs a;
    const int e = make_args("kv_pages_trim", kTrim, p, &a);
    if (e) return e;
    kv_pages_tables<kTrim><<<1, kPagesThreads, 0, to_stream(stream)>>>(a);
    return check_launch("kv_pages_tables");
}
