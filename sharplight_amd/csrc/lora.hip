// Low-rank adapters of many requests beside a shared projection (slhip_lora).
//
// Mathematics. y = add + s_a B_a (A_a x) for each row x of a request with adapter a. Two launches: h = A_a x (shrink, sums over K cut
// into ranges that later add up) and y = add + s_a B_a h (expand). HBM bounds both: a prompt's rows are read and written once,
// a decode step reads every adapter that it uses once.
//
// Layout. Rows that share an adapter are taken together whatever requests they are of: the rows of an adapter, in the requests'
// order, are one list, which is cut into tiles of TM rows. Request i works on the tiles that begin in its part of the list
// (no more than its rows alone would make), so a launch is sized from rows and requests (item_base). Up to 64
// requests a wave looks at all of them at once, a lane each, and every thread block finds its rows so; of more, a launch before (lora_plan)
// lists the tiles, and the others share out what there is: 256 requests that share 8 adapters are 17 tiles, of 272 that there might be.
// With mfma 16x16x32 (A[m][8g+j], B[8g+j][n], C[4g+r][n] in lane (n or m) + 16 g) the first product has adapters as the first operand and rows
// as the second one, so that a lane's sums are four neighbours of one row of h; the second product has rows first (lora_expand).
//
// Measured, in us: one row of 16 ranks, [4096, 4096] in bf16: 4.6 + 6.0 (latencies: lengths -> adapter -> weights, twice); 64 requests with
// an adapter each into 14336 outputs: 6.4 + 13.4 (38 MB of adapters), with f32 adapters 8.3 + 21.7 (75 MB); 256 requests that share 8 of 64 ranks, f32
// [4096, 14336]: 4.8 for the list, 12.2 + 8.8; 23 requests' 2194 rows, f32 with f16 adapters of 24 ranks [4104, 2880]: 11.7 + 23.8 (25 and 70 MB); a prompt
// of 8192 into 14336 outputs in bf16: 16.2 (69 MB) + 96.8 (470 MB, 4.9 TB/s; a kernel that only copies rows in pieces as short as these takes 81 to 95).
// Made in one launch, each thread block its own h, a row takes 10.5 and the 64 requests 22. One thread block writes the list, and one lane of it the keys of an
// adapter's tiles: of long requests that share an adapter it takes more than products of [64, 64] (100 requests of 184 rows 20 us, the products 12; 300 of 3700
// 916 and 345).
//
// Numbers. All products are of bf16 numbers on the matrix cores, with f32 sums. A number of another type is the sum of bf16 ones, exactly:
// f16 of two, f32 of three, each the last one's remainder cut to 8 bits; a product takes all pairs. h is f32 and goes on in three
// parts. Two parts of 16 ranks fill the two halves of one instruction's 32 products.
#include <type_traits>

#include "kv8_map.hpp"
#include "step.hpp"

namespace slhip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kMaxRank = 256;
constexpr int kMaxRequests = 4096;
constexpr int64_t kMaxRows = 0x7FFFFFFF - 32 * kMaxRequests;  // the places of their tiles are 32 bits
constexpr int kUnit = 64;          // inputs that a wave takes together: a line of 16-bit rows
constexpr int kMostSplits = 16;
constexpr int64_t kSplitRows = 65536;  // rows times ranges are at most so many, or the rows

struct Plan {
    int32_t tiles, splits, col_blocks, reserved;
};

struct LoraArgs {
    const void *x, *add;
    void* y;
    int64_t xs, as, ys;
    const void *a, *b;
    int64_t sa, sb;
    int32_t adapters, R, R16, K, N;
    const int32_t* rank;
    const float* scale;
    int32_t B;
    int64_t T;
    const int32_t *starts, *adapter;
    float* h;  // [splits][T][R16]
    int32_t splits, rank_blocks, col_blocks;  // ranges of K, of the ranks; thread blocks that share a tile's columns
    int32_t cols;                             // that there could be
    Plan* plan;                               // of more than 64 requests
    int32_t *plan_key, *plan_rows;            // [tiles], [tiles][TM]
    int32_t spare;  // columns that the load of a column's last ranks may reach into
    uint32_t* err;
};

// How many thread blocks share out the columns of all tiles. A tile's beginning (its rows, h) costs a thread block as much as some of its
// steps. Thread blocks that all run at once are few, with even shares of steps: 32-row tiles' 640 (a prompt of 2048 into 14336 outputs, 16
// ranks: 520 thread blocks 36 us with the first product, 910 39.7, 3640 43.5; 64 ranks: 520 54 us, 715 with uneven shares 66), 16-row
// tiles' 512 (64 requests of an adapter each: 512 18.7 us, 2048 22.5). Many steps end more evenly in several rounds of up to 16 ranks (a prompt of 8192
// into 14336: 514 125 us, 3855 110; into 8192: 79 and 73; 4096 into 14336, 7224 steps: 69.5 and 69.8; into 8192: 43 and 52; with 64 ranks
// 8192 into 14336 take 514 179 us, 4096 192).
SLHIP_HD int64_t expand_blocks(int64_t tiles, int64_t cols, int mt, int32_t r16) { return mt == 1 ? 512 : r16 <= 16 && tiles * cols > 6144 ? 4096 : 640; }
SLHIP_HD int32_t columns_shared(int64_t tiles, int64_t cols, int mt, int32_t r16)
{
    const int64_t blocks = expand_blocks(tiles, cols, mt, r16);
    int64_t most = blocks / tiles;
    most = most < 1 ? 1 : most > cols ? cols : most;
    if (blocks != 4096) {
        const int64_t steps = (cols + most - 1) / most;
        most = (cols + steps - 1) / steps;
    }
    return static_cast<int32_t>(most);
}

// ---- rows ----------------------------------------------------------------------------------------------------------

constexpr int32_t kNoTile = -2;

// A request's adapter; one that is none of the set's counts as none.
__device__ __forceinline__ int32_t adapter_of(const LoraArgs& a, int32_t i)
{
    const int32_t v = a.adapter[i];
    return v >= 0 && v < a.adapters ? v : -1;
}

__device__ __forceinline__ int32_t rows_of(const LoraArgs& a, int32_t i)
{
    const int32_t s0 = a.starts[i], s1 = a.starts[i + 1];
    return s0 >= 0 && s1 >= s0 && s1 <= a.T ? s1 - s0 : 0;
}

// A tile of up to 64 requests, a lane each: one memory latency, and nothing but the rows goes through LDS.
template <int TM> __device__ __forceinline__ int32_t find_tile_64(const LoraArgs& a, int64_t item, int32_t* s_rows)
{
    const int lane = threadIdx.x & 63, j = min(lane, a.B - 1);
    const int32_t s0 = a.starts[j], mine = lane < a.B ? rows_of(a, j) : 0, own = adapter_of(a, j);
    const int k = max(__popcll(__ballot(lane < a.B && item_base(s0, j, TM, 1) <= item)) - 1, 0);
    const int32_t n = __builtin_amdgcn_readlane(mine, k), key = __builtin_amdgcn_readlane(own, k), at = __builtin_amdgcn_readlane(s0, k);
    const int64_t piece = item - item_base(at, k, TM, 1);
    if (piece < 0 || piece * TM >= n) return kNoTile;
    const int32_t match = own == key ? mine : 0, up = wave_scan(match) - match, before = __builtin_amdgcn_readlane(up, k);
    const int64_t first = ((static_cast<int64_t>(before) + TM - 1) / TM + piece) * TM, off = first - before;
    if (off < 0 || off >= n) return kNoTile;  // (below 0 where requests overlap, which none may)
    if (threadIdx.x < 64) {
        const int32_t have = static_cast<int32_t>(min(static_cast<int64_t>(TM), n - off));
        if (lane < TM) s_rows[lane] = lane < have ? at + static_cast<int32_t>(off) + lane : -1;
        if (lane > k && up >= static_cast<int64_t>(before) + n) {
            for (int32_t r = 0; r < match && up + r - first < TM; r++) s_rows[up + r - first] = s0 + r;
        }
    }
    __syncthreads();
    return key;
}

// Lists the tiles of more than 64 requests, by one thread block: the rows of each adapter in a hash table of adapters, in any
// order (no row's result depends on the others of its tile), then the adapters' first tiles by a sum over the table.
constexpr int kPlanThreads = 1024, kSlots = 2 * kMaxRequests, kEach = kMaxRequests / kPlanThreads;
constexpr int32_t kEmpty = -0x7FFFFFFF;
constexpr int kPlanLds = (2 * kSlots + kPlanThreads / 64) * 4;

template <int TM> __global__ __launch_bounds__(kPlanThreads) void lora_plan(LoraArgs a, int32_t blocks1)
{
    extern __shared__ int32_t s_slots[];
    int32_t *s_key = s_slots, *s_count = s_slots + kSlots, *s_wave = s_slots + 2 * kSlots;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    int slots = 256;
    while (slots < 2 * a.B) slots *= 2;  // a power of two, at most kSlots
    for (int i = tid; i < slots; i += kPlanThreads) {
        s_key[i] = kEmpty;
        s_count[i] = 0;
    }
    __shared__ unsigned long long s_all;
    if (tid == 0) s_all = 0;
    __syncthreads();
    int32_t s0[kEach], n[kEach], slot[kEach], at[kEach];
    unsigned long long rows_mine = 0;
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const int32_t j = lane * (kPlanThreads / 64) + wave + e * kPlanThreads;  // few requests, too, are shared out over the waves
        const bool in = j < a.B;
        s0[e] = in ? a.starts[j] : 0;
        n[e] = in ? rows_of(a, j) : 0;
        rows_mine += n[e];
        const int32_t key = in ? adapter_of(a, j) : -1;
        if (n[e] == 0) continue;
        int32_t h = static_cast<uint32_t>(key) * 2654435761u >> 16 & (slots - 1);
        for (;;) {  // there are fewer keys than slots
            const int32_t was = atomicCAS(&s_key[h], kEmpty, key);
            if (was == kEmpty || was == key) break;
            h = (h + 1) & (slots - 1);
        }
        slot[e] = h;
        at[e] = atomicAdd(&s_count[h], n[e]);
    }
    if (rows_mine > 0) atomicAdd(&s_all, rows_mine);
    __syncthreads();
    if (s_all > static_cast<unsigned long long>(a.T)) {  // requests overlap, so starts falls, which is reported: there is no list for that
        if (tid == 0) *a.plan = Plan{0, 1, 1, 0};
        return;
    }
    const int each = slots <= kPlanThreads ? 1 : slots / kPlanThreads;
    int32_t mine = 0;
    for (int i = tid * each; i < min((tid + 1) * each, slots); i++) mine += (s_count[i] + TM - 1) / TM;
    int32_t up = wave_scan(mine);
    if (lane == 63) s_wave[wave] = up;
    up -= mine;
    __syncthreads();
    int32_t tiles = 0;
    for (int w = 0; w < kPlanThreads / 64; w++) {
        if (w == wave) up += tiles;
        tiles += s_wave[w];
    }
    for (int i = tid * each; i < min((tid + 1) * each, slots); i++) {
        const int32_t rows = s_count[i], some = (rows + TM - 1) / TM;
        for (int32_t t = 0; t < some; t++) a.plan_key[up + t] = s_key[i];
        for (int32_t r = rows; r < some * TM; r++) a.plan_rows[up * TM + r] = -1;
        s_count[i] = up;
        up += some;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const int32_t to = n[e] > 0 ? s_count[slot[e]] * TM + at[e] : 0;
        if (n[e] <= 4) {
            for (int32_t r = 0; r < n[e]; r++) a.plan_rows[to + r] = s0[e] + r;
        }
        for (uint64_t many = __ballot(n[e] > 4); many; many &= many - 1) {  // by the whole wave
            const int k = __ffsll(static_cast<long long>(many)) - 1;
            const int32_t rows = __builtin_amdgcn_readlane(n[e], k), p = __builtin_amdgcn_readlane(to, k), s = __builtin_amdgcn_readlane(s0[e], k);
            for (int32_t r = lane; r < rows; r += 64) a.plan_rows[p + r] = s + r;
        }
    }
    if (tid == 0) {  // the tiles share out the thread blocks that there are
        const int32_t some = max(tiles, 1);
        *a.plan = Plan{tiles, max(min(a.splits, blocks1 / (some * a.rank_blocks)), 1), columns_shared(some, a.cols, TM / 16, a.R16), 0};
    }
}

// The rows of tile `item` into s_rows (-1 behind the last), and their adapter; kNoTile where there is none.
template <int TM> __device__ __forceinline__ int32_t find_tile(const LoraArgs& a, int64_t item, int32_t* s_rows)
{
    if (!a.plan) return find_tile_64<TM>(a, item, s_rows);
    const int32_t key = a.plan_key[item];
    if (threadIdx.x < TM) s_rows[threadIdx.x] = a.plan_rows[item * TM + threadIdx.x];
    __syncthreads();
    return key;
}

__device__ __forceinline__ int32_t rank_of(const LoraArgs& a, int32_t adapter)
{
    return a.rank ? min(max(a.rank[adapter], 0), a.R) : a.R;
}

// ---- loads ---------------------------------------------------------------------------------------------------------

template <int DT> constexpr int kParts = DT == SLHIP_BF16 ? 1 : DT == SLHIP_F16 ? 2 : 3;

// v as P bf16 numbers that add up to it (all of its bits are in them). An infinity leaves a NaN behind.
template <int P> __device__ __forceinline__ void cut(const float (&v)[8], bf16x8 (&p)[P])
{
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; e++) r[e] = v[e];
#pragma unroll
    for (int i = 0; i < P; i++) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = __builtin_amdgcn_perm(__float_as_uint(r[2 * e + 1]), __float_as_uint(r[2 * e]), 0x07060302u);  // upper halves
        p[i] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int e = 0; e < 8; e++) r[e] -= __uint_as_float(__float_as_uint(r[e]) & 0xFFFF0000u);
    }
}

// v's bytes from `bytes` (0 .. 16, even) on, zeros behind them.
__device__ __forceinline__ uint4 shift_down(uint4 v, int32_t bytes)
{
    if (bytes & 16) v = make_uint4(0, 0, 0, 0);
    if (bytes & 8) v = make_uint4(v.z, v.w, 0, 0);
    if (bytes & 4) v = make_uint4(v.y, v.z, v.w, 0);
    const uint32_t s = (bytes & 2) * 8;
    return make_uint4(__builtin_amdgcn_alignbit(v.y, v.x, s), __builtin_amdgcn_alignbit(v.z, v.y, s), __builtin_amdgcn_alignbit(v.w, v.z, s), v.w >> s);
}

// 16 bytes from element `at` of a row of n (16 bytes or more): zeros behind its end.
template <int DT> __device__ __forceinline__ uint4 load_end(const char* row, int32_t at, int32_t n)
{
    constexpr int E = Vec<DT>::N;
    const int32_t in = min(at, n - E);
    return shift_down(load_any(row + static_cast<uint32_t>(in) * Vec<DT>::BYTES), min(at - in, E) * Vec<DT>::BYTES);
}

// v's bytes moved up by `bytes` (0 .. 16, even), zeros below them.
__device__ __forceinline__ uint4 shift_up(uint4 v, int32_t bytes)
{
    if (bytes & 16) v = make_uint4(0, 0, 0, 0);
    if (bytes & 8) v = make_uint4(0, 0, v.x, v.y);
    if (bytes & 4) v = make_uint4(0, v.x, v.y, v.z);
    if (bytes & 2) v = make_uint4(v.x << 16, __builtin_amdgcn_alignbit(v.y, v.x, 16), __builtin_amdgcn_alignbit(v.z, v.y, 16), __builtin_amdgcn_alignbit(v.w, v.z, 16));
    return v;
}

// The first n elements of v; the others become 0.
template <int DT> __device__ __forceinline__ uint4 keep(const uint4& v, int32_t n)
{
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if constexpr (DT == SLHIP_F32) w[j] = n > j ? w[j] : 0;
        else w[j] = n > 2 * j + 1 ? w[j] : n > 2 * j ? w[j] & 0xFFFF : 0;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// N neighbours (8 or 16).
template <int DT, int N> struct Run {
    static constexpr int kVecs = N * Vec<DT>::BYTES / 16, kPer = Vec<DT>::N;
    uint4 w[kVecs];
    __device__ __forceinline__ void load(const char* p)
    {
#pragma unroll
        for (int i = 0; i < kVecs; i++) w[i] = load_any(p + 16 * i);
    }
    __device__ __forceinline__ void load_end(const char* row, int32_t at, int32_t n)
    {
#pragma unroll
        for (int i = 0; i < kVecs; i++) w[i] = slhip::load_end<DT>(row, at + i * kPer, n);
    }
    // The elements from the k-th on, zeros behind them.
    __device__ __forceinline__ void shift(int32_t k)
    {
#pragma unroll
        for (int i = 0; i < kVecs; i++) {  // (of two vectors the second one's first come behind the first one's last)
            const int32_t by = min(k, kPer) * Vec<DT>::BYTES;
            if (kVecs == 2 && i == 0 && k > 0) {
                const uint4 a = shift_down(w[0], by), b = w[1];
                const uint4 up = shift_up(b, 16 - by);
                w[0] = k >= kPer ? shift_down(b, min(k - kPer, kPer) * Vec<DT>::BYTES) : make_uint4(a.x | up.x, a.y | up.y, a.z | up.z, a.w | up.w);
            } else if (kVecs == 2 && i == 1) {
                w[1] = shift_down(w[1], by);
            } else {
                w[i] = shift_down(w[i], by);
            }
        }
    }
    __device__ __forceinline__ void keep(int32_t n)
    {
#pragma unroll
        for (int i = 0; i < kVecs; i++) w[i] = slhip::keep<DT>(w[i], n - i * kPer);
    }
    // Eight of them as bf16 parts.
    template <int P> __device__ __forceinline__ void parts(int half, bf16x8 (&p)[P]) const
    {
        if constexpr (DT == SLHIP_BF16) {
            p[0] = __builtin_bit_cast(bf16x8, w[half]);
        } else {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8 / kPer; i++) Vec<DT>::unpack(w[half * (8 / kPer) + i], &f[i * kPer]);
            cut(f, p);
        }
    }
};

// ---- h = A x -------------------------------------------------------------------------------------------------------

template <int XT, int WT, int MT, int RB> __global__ __launch_bounds__(kThreads) void lora_shrink(LoraArgs a, int32_t pieces)
{
    constexpr int TM = 16 * MT, PX = kParts<XT>, PW = kParts<WT>;
    constexpr int U = MT * RB == 1 ? 4 : MT * RB == 8 && WT == SLHIP_F32 ? 1 : MT == 1 || XT == SLHIP_BF16 ? 2 : 1;  // units whose loads are on their way together
    __shared__ int32_t s_rows[TM];
    __shared__ f32x4 s_acc[kWaves / 2][MT * RB][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), c = lane & 15, g = lane >> 4;
    if (blockIdx.x == 0) {
        for (int32_t i = tid; i < a.B; i += kThreads) {
            const int64_t s0 = a.starts[i], n = a.starts[i + 1] - s0;
            if (s0 < 0 || n < 0 || s0 + n > a.T)
                raise_error(a.err, kErrKvRequest, static_cast<uint32_t>(i), static_cast<uint32_t>(i), 0, static_cast<uint32_t>(n), static_cast<uint32_t>(static_cast<uint64_t>(n) >> 32), 0);
            else if (n > 0 && a.adapter[i] != adapter_of(a, i))
                raise_error(a.err, kErrAdapter, static_cast<uint32_t>(i), static_cast<uint32_t>(a.adapter[i]), static_cast<uint32_t>(a.adapters), 0, 0, 0);
        }
    }
    const int32_t splits = a.plan ? a.plan->splits : a.splits, work = a.plan ? a.plan->tiles * splits * a.rank_blocks : pieces;
    const auto piece = [&](int32_t item) __attribute__((always_inline)) {
    const int32_t rb = item % a.rank_blocks, rest = item / a.rank_blocks, split = rest % splits;
    const int32_t key = find_tile<TM>(a, rest / splits, s_rows);
    if (key < 0) return;
    const int32_t rank = rank_of(a, key), r0 = rb * RB * 16;
    if (r0 >= rank) return;
    const int32_t units = (a.K + kUnit - 1) / kUnit, each = (units + splits - 1) / splits;
    const int32_t u0 = split * each, u1 = min(u0 + each, units);
    // rows and ranks that are not there: others, whose sums nothing takes
    const char* xp[MT];
    uint32_t ap[RB];
    const char* const ad = static_cast<const char*>(a.a) + key * a.sa * Vec<WT>::BYTES;
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int32_t row = s_rows[16 * m + c];
        xp[m] = static_cast<const char*>(a.x) + ((row >= 0 ? row : s_rows[0]) * a.xs + 16 * g) * Vec<XT>::BYTES;
    }
#pragma unroll
    for (int q = 0; q < RB; q++) ap[q] = static_cast<uint32_t>(min(r0 + 16 * q + c, rank - 1) * a.K + 16 * g) * Vec<WT>::BYTES;
    f32x4 acc[MT][RB];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int q = 0; q < RB; q++) acc[m][q] = f32x4{0, 0, 0, 0};
    const int32_t ranks = (min(rank - r0, RB * 16) + 15) / 16;
    const auto multiply = [&](const Run<XT, 16> (&x)[MT], const Run<WT, 16> (&w)[RB]) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            bf16x8 px[MT][PX];
#pragma unroll
            for (int m = 0; m < MT; m++) x[m].parts(s, px[m]);
#pragma unroll
            for (int q = 0; q < RB; q++) {
                if (q > 0 && q >= ranks) break;
                bf16x8 pw[PW];
                w[q].parts(s, pw);
#pragma unroll
                for (int i = PX - 1; i >= 0; i--)  // small ones first
#pragma unroll
                    for (int j = PW - 1; j >= 0; j--)
#pragma unroll
                        for (int m = 0; m < MT; m++) acc[m][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pw[j], px[m][i], acc[m][q], 0, 0, 0);
            }
        }
    };
    int32_t u = u0 + wave;
    const int32_t whole = min(u1, a.K / kUnit);  // (the last unit may not be)
    for (; u + (U - 1) * kWaves < whole; u += kWaves * U) {
        Run<XT, 16> x[U][MT];
        Run<WT, 16> w[U][RB];
#pragma unroll
        for (int v = 0; v < U; v++) {
            const uint32_t k = static_cast<uint32_t>(u + v * kWaves) * kUnit;
#pragma unroll
            for (int q = 0; q < RB; q++)
                if (q == 0 || q < ranks) w[v][q].load(ad + (ap[q] + k * Vec<WT>::BYTES));
#pragma unroll
            for (int m = 0; m < MT; m++) x[v][m].load(xp[m] + k * Vec<XT>::BYTES);
        }
#pragma unroll
        for (int v = 0; v < U; v++) multiply(x[v], w[v]);
    }
    for (; u < u1; u += kWaves) {
        Run<XT, 16> x[MT];
        Run<WT, 16> w[RB];
        const int32_t k = u * kUnit + 16 * g;
#pragma unroll
        for (int q = 0; q < RB; q++) w[q].load_end(ad + (ap[q] - 16 * g * Vec<WT>::BYTES), k, a.K);
#pragma unroll
        for (int m = 0; m < MT; m++) x[m].load_end(xp[m] - 16 * g * Vec<XT>::BYTES, k, a.K);
        multiply(x, w);
    }
    // the sums of waves 2 and 3 into 0 and 1, and 1 into 0
    for (int half = kWaves / 2; half > 0; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int q = 0; q < RB; q++) s_acc[wave - half][m * RB + q][lane] = acc[m][q];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int q = 0; q < RB; q++) acc[m][q] += s_acc[wave][m * RB + q][lane];
        }
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int32_t row = s_rows[16 * m + c];
        if (row < 0) continue;
        float* h = a.h + (static_cast<int64_t>(split) * a.T + row) * a.R16 + r0 + 4 * g;
#pragma unroll
        for (int q = 0; q < RB; q++)
            if (r0 + 16 * q < rank) *reinterpret_cast<f32x4*>(h + 16 * q) = acc[m][q];
    }
    };
    for (int32_t item = blockIdx.x; item < work; item += gridDim.x) {
        piece(item);
        if (item + gridDim.x < work) __syncthreads();  // the next piece's rows
    }
}

// ---- y = add + s B h -----------------------------------------------------------------------------------------------

// E neighbours of a row of add or y, 8 or 16 bytes.
template <int DT, int E> struct Piece {
    static constexpr int kWords = E * Vec<DT>::BYTES / 4;
    typedef uint32_t words __attribute__((ext_vector_type(kWords)));
    typedef words words_any __attribute__((aligned(2)));
    words w;
    __device__ __forceinline__ void load(const char* p) { w = __builtin_nontemporal_load(reinterpret_cast<const words_any*>(p)); }
    __device__ __forceinline__ void store(char* p) const { __builtin_nontemporal_store(w, reinterpret_cast<words_any*>(p)); }
    __device__ __forceinline__ void floats(float (&f)[E]) const
    {
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            if constexpr (DT == SLHIP_F32) {
                f[i] = __uint_as_float(w[i]);
            } else {
                f[2 * i] = bf16_lo(w[i]);
                f[2 * i + 1] = bf16_hi(w[i]);
            }
        }
    }
    __device__ __forceinline__ void pack(const float (&f)[E])
    {
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            if constexpr (DT == SLHIP_F32) w[i] = __float_as_uint(f[i]);
            else w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
        }
    }
};

constexpr int kLane = 4;  // columns of a lane: 8 of bf16 take 256 registers with their sums, and two waves a SIMD are too few

// Rows are the first operand here and columns the second. A wave has 64 columns of its rows: product u the columns 4 c + u, so that a
// lane's sums of the four products are neighbours in a row, and 16 lanes load and store whole lines of it. Row 4 r + g of 16 stands in the operand's
// place 4 g + r: lane (c, g) has it in element r, and of up to four rows (a decode step's, most often one) all lie in element 0.
template <int YT, int WT, int MT, bool WIDE> __global__ __launch_bounds__(kThreads) void lora_expand(LoraArgs a, int32_t pieces)
{
    constexpr int TM = 16 * MT, PW = kParts<WT>, E = kLane, kColumns = 16 * E;
    // h's three parts of RC ranks are the first operands of H instructions: up to 16 ranks two of them share one, more have one each
    constexpr int H = WIDE ? kParts<SLHIP_F32> : 2, RC = WIDE ? 32 : 16;
    __shared__ int32_t s_rows[TM];
    extern __shared__ uint4 s_h[];  // [MT][all][H][64]
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), c = lane & 15, g = lane >> 4;
    const int32_t col_blocks = a.plan ? a.plan->col_blocks : a.col_blocks, work = a.plan ? a.plan->tiles * col_blocks : pieces;
    const auto piece = [&](int32_t item) __attribute__((always_inline)) {
    const int32_t cb = item % col_blocks;
    const int32_t key = find_tile<TM>(a, item / col_blocks, s_rows);
    if (key == kNoTile || (key < 0 && a.add == a.y)) return;
    const char* const ad = static_cast<const char*>(a.b) + (key < 0 ? 0 : key * a.sb * Vec<WT>::BYTES);
    const uint32_t as = static_cast<uint32_t>(a.as * Vec<YT>::BYTES), ys = static_cast<uint32_t>(a.ys * Vec<YT>::BYTES);
    uint32_t row[MT][4];
    bool there[MT][4];
    int most = 0;  // rows' elements that hold one
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int32_t v = s_rows[16 * m + 4 * r + g];
            there[m][r] = v >= 0;
            row[m][r] = v >= 0 ? v : s_rows[0];
            if (__any(v >= 0)) most = 4 * m + r + 1;
        }
    Piece<YT, E> add[MT][4];
    Run<WT, 8> w[E];
    const int rl = 8 * (WIDE ? g : g & 1);  // the lane's ranks of RC
    // The lane's columns from n0 on: of lanes behind the last column those before it once more. Of a column's last ranks the loads reach into the
    // next one's; those that would leave the adapter begin before, and what they brought is moved down (fix).
    const auto column = [&](int32_t n0) { return min(n0 + E * c, a.N - E); };
    const auto whole = [&](int32_t n0) { return n0 + kColumns + a.spare <= a.N; };
    const auto fetch_w = [&](int32_t n0, int q) __attribute__((always_inline)) {
        const int32_t at = column(n0) * a.R + RC * q + rl, last = a.N * a.R - 8;
#pragma unroll
        for (int u = 0; u < E; u++) w[u].load(ad + static_cast<uint32_t>(min(at + u * a.R, last)) * Vec<WT>::BYTES);
    };
    const auto fix = [&](int32_t n0, int q) __attribute__((always_inline)) {
        const int32_t at = column(n0) * a.R + RC * q + rl, last = a.N * a.R - 8;
#pragma unroll
        for (int u = 0; u < E; u++) w[u].shift(max(at + u * a.R - last, 0));
    };
    const auto fetch_add = [&](int32_t n0) __attribute__((always_inline)) {
        const char* const at = static_cast<const char*>(a.add) + static_cast<uint32_t>(column(n0)) * Vec<YT>::BYTES;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (m + r > 0 && 4 * m + r >= most) break;
                if (a.add) add[m][r].load(at + static_cast<uint64_t>(row[m][r]) * as);
                else add[m][r].w = 0;
            }
    };
    // thread blocks that run together take neighbouring columns: the same columns of many rows lie in few memory channels
    const int32_t first = (cb * kWaves + wave) * kColumns, step = col_blocks * kWaves * kColumns;
    const int32_t rank = key < 0 ? 0 : rank_of(a, key), tiles = (rank + RC - 1) / RC, all = (a.R + RC - 1) / RC;
    const auto finish = [&](int32_t n0) __attribute__((always_inline)) {
        f32x4 acc[MT][E];
        const auto multiply = [&](int q, auto begins) __attribute__((always_inline)) {
            if (!whole(n0)) fix(n0, q);
            if (RC * q + RC > rank) {  // ranks behind the last may hold anything
#pragma unroll
                for (int u = 0; u < E; u++) w[u].keep(rank - RC * q - rl);
            }
            bf16x8 pw[E][PW];
#pragma unroll
            for (int u = 0; u < E; u++) w[u].parts(0, pw[u]);
            if (WIDE && q + 1 < tiles) fetch_w(n0, q + 1);
            else if (WIDE && n0 + step < a.N) fetch_w(n0 + step, 0);
            bf16x8 x[MT][H];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int h = 0; h < H; h++) x[m][h] = __builtin_bit_cast(bf16x8, s_h[((m * all + q) * H + h) * 64 + lane]);
#pragma unroll
            for (int u = 0; u < E; u++)
#pragma unroll
                for (int h = H - 1; h >= 0; h--)
#pragma unroll
                    for (int i = PW - 1; i >= 0; i--)
#pragma unroll
                        for (int m = 0; m < MT; m++)
                            acc[m][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[m][h], pw[u][i], begins && h == H - 1 && i == PW - 1 ? f32x4{0, 0, 0, 0} : acc[m][u], 0, 0, 0);
        };
        if (tiles > 0) {
            multiply(0, std::true_type{});
            for (int q = 1; WIDE && q < tiles; q++) multiply(q, std::false_type{});
        } else {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int u = 0; u < E; u++) acc[m][u] = f32x4{0, 0, 0, 0};
        }
        const int32_t n = column(n0), mine = n0 + E * c;  // a lane's columns from `mine` on are its own
        char* const to = static_cast<char*>(a.y) + static_cast<uint32_t>(n) * Vec<YT>::BYTES;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (m + r > 0 && 4 * m + r >= most) break;
                float f[E];
                add[m][r].floats(f);
#pragma unroll
                for (int u = 0; u < E; u++) f[u] += acc[m][u][r];
                char* const p = to + static_cast<uint64_t>(row[m][r]) * ys;
                if (n == mine) {
                    add[m][r].pack(f);
                    if (there[m][r]) add[m][r].store(p);
                } else if (there[m][r] && mine < a.N) {
#pragma unroll
                    for (int u = 1; u < E; u++)
                        if (n + u >= mine) Vec<YT>::store1(p, u, f[u]);
                }
            }
    };
    if (first < a.N) {
        if (key >= 0) fetch_w(first, 0);
        fetch_add(first);
    }
    const float scale = key < 0 || !a.scale ? 1.0f : a.scale[key];
    const int32_t splits = a.plan ? a.plan->splits : a.splits;
    // h, ranges of K added up: `parts` lanes share eight ranks of a row
    const int32_t units = key < 0 ? 0 : MT * all * 2 * RC, parts = units <= 32 ? 8 : units <= 64 ? 4 : units <= 128 ? 2 : 1;
    for (int t = tid; t < units * parts; t += kThreads) {
        const int part = t & (parts - 1), unit = t / parts, m = unit / (all * 2 * RC), q = unit / (2 * RC) - m * all, l = unit & (2 * RC - 1);
        const int32_t at = s_rows[16 * m + 4 * (l & 3) + (l >> 2 & 3)], r = RC * q + 8 * (l >> 4);
        float f[8] = {};
        if (at >= 0 && r < rank) {
            const float* h = a.h + static_cast<int64_t>(at) * a.R16 + r;
            const int64_t range = a.T * a.R16;
            for (int s = part; s < splits; s += 2 * parts) {
                f32x4 x[2][2];
#pragma unroll
                for (int v = 0; v < 2; v++)
#pragma unroll
                    for (int e = 0; e < 2; e++) x[v][e] = reinterpret_cast<const f32x4*>(h + min(s + v * parts, splits - 1) * range)[e];
#pragma unroll
                for (int v = 0; v < 2; v++)
#pragma unroll
                    for (int e = 0; e < 8; e++) f[e] += s + v * parts < splits ? x[v][e >> 2][e & 3] : 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (parts > 1) f[e] += dpp_f32<0xB1>(f[e]);
            if (parts > 2) f[e] += dpp_f32<0x4E>(f[e]);
            if (parts > 4) f[e] += dpp_f32<0x141>(f[e]);
            f[e] = r + e < rank ? f[e] * scale : 0.0f;
        }
        if (part > 0) continue;
        uint4* const put = s_h + ((m * all + q) * H) * 64 + l;  // WIDE: an operand a part, else lanes l and l + 32 of one
        constexpr int kNext = WIDE ? 64 : 32;
        bf16x8 p[kParts<SLHIP_F32>];
        cut(f, p);
#pragma unroll
        for (int i = 0; i < kParts<SLHIP_F32>; i++) put[kNext * i] = __builtin_bit_cast(uint4, p[i]);
        if (!WIDE) put[kNext * kParts<SLHIP_F32>] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    for (int32_t n0 = first; n0 < a.N; n0 += step) {
        if (n0 > first) {
            if (!WIDE && key >= 0) fetch_w(n0, 0);
            fetch_add(n0);
        }
        finish(n0);
    }
    };
    for (int32_t item = blockIdx.x; item < work; item += gridDim.x) {
        piece(item);
        if (item + gridDim.x < work) __syncthreads();  // the next piece's rows and h
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------

static int64_t round16(int64_t n) { return (n + 15) & ~int64_t{15}; }

// Tiles that T rows can make, and what their list takes: key and rows each.
static int64_t most_tiles(int64_t T, int64_t tile) { return T / tile + (T < kMaxRequests ? T : kMaxRequests); }
static int64_t plan_of(int64_t T) { return 16 + round16(4 * 33 * most_tiles(T, 16)); }

static int64_t work_of(int64_t T, int64_t R)
{
    const int64_t most = T > kSplitRows ? T : kSplitRows;
    return (T * kMostSplits < most ? T * kMostSplits : most) * round16(R) * 4 + plan_of(T);
}

// A launch has less than 2^32 threads: beyond that thread blocks take turns. (Pieces are 2^28 at most: 2^31 rows in tiles of 32, by four ranges of ranks.)
static unsigned blocks_of(int64_t pieces) { return static_cast<unsigned>(pieces < 0xFFFFFF ? pieces : 0xFFFFFF); }

template <int XT, int WT, int MT> static int shrink(const LoraArgs& a, int64_t pieces, hipStream_t st)
{
    const auto kernel = a.R16 <= 16 ? lora_shrink<XT, WT, MT, 1> : a.R16 <= 32 ? lora_shrink<XT, WT, MT, 2> : lora_shrink<XT, WT, MT, 4>;
    kernel<<<blocks_of(pieces), kThreads, 0, st>>>(a, static_cast<int32_t>(pieces));
    return check_launch("lora_shrink");
}

template <int YT, int WT, int MT> static int expand(const LoraArgs& a, int64_t pieces, hipStream_t st)
{
    const int lds = MT * 1024 * (a.R16 <= 16 ? 2 : (a.R + 31) / 32 * kParts<SLHIP_F32>);  // at most 48 KB
    const auto kernel = a.R16 <= 16 ? lora_expand<YT, WT, MT, false> : lora_expand<YT, WT, MT, true>;
    kernel<<<blocks_of(pieces), kThreads, lds, st>>>(a, static_cast<int32_t>(pieces));
    return check_launch("lora_expand");
}

template <int MT> static int plan(const LoraArgs& a, int64_t blocks1, hipStream_t st)
{
    SLHIP_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&lora_plan<16 * MT>), hipFuncAttributeMaxDynamicSharedMemorySize, kPlanLds));
    lora_plan<16 * MT><<<1, kPlanThreads, kPlanLds, st>>>(a, static_cast<int32_t>(blocks1));
    return check_launch("lora_plan");
}

template <int WT, int MT> static int launch(int dtype_x, int dtype_y, LoraArgs& a, hipStream_t st)
{
    const bool planned = a.B > 64;
    const int64_t tiles = planned ? most_tiles(a.T, 16 * MT) : item_count(a.T, a.B, 16 * MT, 1);
    constexpr int64_t wide = kWaves * 16 * kLane;
    a.rank_blocks = a.R16 <= 32 ? 1 : (a.R16 + 63) / 64;
    a.cols = static_cast<int32_t>((a.N + wide - 1) / wide);
    // ranges of K of 512 inputs at least, as far as they give the machine work; of 32-row tiles, whose h is more, beyond 8 only for 256 thread blocks
    // (a prompt of 1500 rows, 64 ranks, 14336 inputs, 13312 outputs: 8 ranges 67.8 us, 16 73.7)
    int64_t splits = a.K / 512;
    if (splits > kMostSplits) splits = kMostSplits;
    if (splits > kSplitRows / a.T) splits = kSplitRows / a.T;
    if (!planned && splits > 1024 / (tiles * a.rank_blocks)) splits = 1024 / (tiles * a.rank_blocks);
    if (!planned && MT == 2 && splits > 8 && splits * tiles > 256) splits = 256 / tiles > 8 ? 256 / tiles : 8;
    a.splits = splits < 1 ? 1 : static_cast<int32_t>(splits);
    a.col_blocks = columns_shared(tiles, a.cols, MT, a.R16);
    int64_t first = tiles * a.splits * a.rank_blocks, second = tiles * a.col_blocks;
    if (planned) {
        if (first > 1024) first = 1024;
        second = tiles * a.cols;  // the most that there could be
        if (second > expand_blocks(tiles, a.cols, MT, a.R16)) second = expand_blocks(tiles, a.cols, MT, a.R16);
        const int e = plan<MT>(a, first, st);
        if (e) return e;
    } else {
        a.plan = nullptr;
    }
    const int e = dtype_x == SLHIP_F32 ? shrink<SLHIP_F32, WT, MT>(a, first, st) : shrink<SLHIP_BF16, WT, MT>(a, first, st);
    if (e) return e;
    return dtype_y == SLHIP_F32 ? expand<SLHIP_F32, WT, MT>(a, second, st) : expand<SLHIP_BF16, WT, MT>(a, second, st);
}

// Tiles of 16 rows where requests have few (a decode step), of 32 where they have many.
template <int WT> static int launch(int dtype_x, int dtype_y, LoraArgs& a, hipStream_t st)
{
    return a.T <= 32 * static_cast<int64_t>(a.B) ? launch<WT, 1>(dtype_x, dtype_y, a, st) : launch<WT, 2>(dtype_x, dtype_y, a, st);
}

}  // namespace slhip

using namespace slhip;

extern "C" SLHIP_API int64_t slhip_lora_work_bytes(int64_t tokens, int64_t max_rank)
{
    if (tokens < 0 || tokens > kMaxRows || max_rank < 1 || max_rank > kMaxRank) {
        fail(SLHIP_ERR_INVALID, "lora: bad size");
        return -1;
    }
    return work_of(tokens, max_rank);
}

extern "C" SLHIP_API int slhip_lora(int dtype_x, int dtype_y, const void* x, int64_t x_stride, const void* add, int64_t add_stride,
                                    void* y, int64_t y_stride, const slhip_lora_set* set, const slhip_lora_rows* rows, void* work,
                                    int64_t work_bytes, slhip_stream stream)
{
    if (!set || !rows) return fail(SLHIP_ERR_INVALID, "lora: set and rows are required");
    if ((dtype_x != SLHIP_F32 && dtype_x != SLHIP_BF16) || (dtype_y != SLHIP_F32 && dtype_y != SLHIP_BF16))
        return fail(SLHIP_ERR_UNSUPPORTED, "lora: dtypes %d, %d not supported", dtype_x, dtype_y);
    if (set->dtype != SLHIP_F32 && set->dtype != SLHIP_F16 && set->dtype != SLHIP_BF16)
        return fail(SLHIP_ERR_UNSUPPORTED, "lora: adapters of dtype %d not supported", set->dtype);
    if (set->adapters < 0 || set->max_rank < 1 || set->K < 1 || set->N < 1 || rows->requests < 0 || rows->tokens < 0)
        return fail(SLHIP_ERR_INVALID, "lora: bad size");
    if (set->K < 8 || set->N < 8) return fail(SLHIP_ERR_UNSUPPORTED, "lora: less than 8 inputs or outputs");  // a 16-byte load of bf16
    if (set->max_rank > kMaxRank) return fail(SLHIP_ERR_UNSUPPORTED, "lora: more than %d ranks", kMaxRank);
    if (rows->requests > kMaxRequests) return fail(SLHIP_ERR_UNSUPPORTED, "lora: more than %d requests", kMaxRequests);
    const int64_t widest = (set->K > set->N ? set->K : set->N) * set->max_rank * (set->dtype == SLHIP_F32 ? 4 : 2);
    if (set->adapters > 0x7FFFFFFF || widest > 0x7FFFFFFF || set->K > (1 << 24) || set->N > (1 << 24) || rows->tokens > kMaxRows)
        return fail(SLHIP_ERR_UNSUPPORTED, "lora: too many adapters, inputs, outputs or rows (a matrix of an adapter has less than 2^31 bytes)");
    if (x_stride < set->K || y_stride < set->N || (add && add_stride < set->N))
        return fail(SLHIP_ERR_INVALID, "lora: a row stride is smaller than the row");
    if (y_stride >= int64_t{1} << 30 || (add && add_stride >= int64_t{1} << 30)) return fail(SLHIP_ERR_UNSUPPORTED, "lora: rows 2^30 values apart or more");
    if (set->a_stride < set->max_rank * set->K || set->b_stride < set->max_rank * set->N)
        return fail(SLHIP_ERR_INVALID, "lora: an adapter stride is smaller than the adapter");
    if (rows->requests == 0 || rows->tokens == 0) return SLHIP_OK;
    if (!rows->starts || !rows->adapter) return fail(SLHIP_ERR_INVALID, "lora: starts and adapter are required");
    if (!x || !y || (set->adapters > 0 && (!set->a || !set->b))) return fail(SLHIP_ERR_INVALID, "lora: x, y, a and b are required");
    if (add == y && add_stride != y_stride) return fail(SLHIP_ERR_INVALID, "lora: add is y with another stride");
    const int64_t need = work_of(rows->tokens, set->max_rank);
    if (!work || !aligned16(work) || work_bytes < need)
        return fail(SLHIP_ERR_INVALID, "lora: the workspace has %lld bytes, %lld are needed (16-byte aligned)",
                    static_cast<long long>(work ? work_bytes : 0), static_cast<long long>(need));
    LoraArgs a{};
    a.x = x;
    a.add = add;
    a.y = y;
    a.xs = x_stride;
    a.as = add_stride;
    a.ys = y_stride;
    a.a = set->a;
    a.b = set->b;
    a.sa = set->a_stride;
    a.sb = set->b_stride;
    a.adapters = static_cast<int32_t>(set->adapters);
    a.R = static_cast<int32_t>(set->max_rank);
    a.R16 = static_cast<int32_t>(round16(set->max_rank));
    a.spare = a.R <= 16 ? 15 / a.R : ((a.R + 31) / 32 * 32 - 1) / a.R;
    a.K = static_cast<int32_t>(set->K);
    a.N = static_cast<int32_t>(set->N);
    a.rank = set->rank;
    a.scale = set->scale;
    a.B = static_cast<int32_t>(rows->requests);
    a.T = rows->tokens;
    a.starts = rows->starts;
    a.adapter = rows->adapter;
    a.plan = static_cast<Plan*>(work);
    a.plan_key = reinterpret_cast<int32_t*>(a.plan + 1);
    a.plan_rows = a.plan_key + most_tiles(a.T, 16);
    a.h = reinterpret_cast<float*>(static_cast<char*>(work) + plan_of(a.T));
    int e = error_word(&a.err);
    if (e) return e;
    hipStream_t st = to_stream(stream);
    if (set->dtype == SLHIP_F32) return launch<SLHIP_F32>(dtype_x, dtype_y, a, st);
    if (set->dtype == SLHIP_F16) return launch<SLHIP_F16>(dtype_x, dtype_y, a, st);
    return launch<SLHIP_BF16>(dtype_x, dtype_y, a, st);
}
