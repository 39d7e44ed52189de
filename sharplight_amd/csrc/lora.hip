// Low-rank adapters of many requests beside a shared projection (slhip_lora).
//
// Mathematics. y = add + s_a B_a (A_a x) for each row x of a request with adapter a. Two launches: h = A_a x (shrink, sums over K cut
// into ranges that later add up) and y = add + s_a B_a h (expand). HBM bounds both: a prompt's rows are read and written once,
// a decode step reads every adapter that it uses once.
//
// Layout. Rows that share an adapter are taken together whatever requests they are of: the rows of an adapter, in the requests'
// order, are one list, which is cut into tiles of TM rows. Request i works on the tiles that begin in its part of the list
// (no more than its rows alone would make), so a launch is sized from rows and requests (item_base), and a thread block finds its
// rows by one look at all requests.
// With mfma 16x16x32 (A[m][8g+j], B[8g+j][n], C[4g+r][n] in lane (n or m) + 16 g) adapters are the first operand and rows the
// second one, so that a lane's sums are four neighbours of one row: h is stored and y made without an exchange.
//
// Numbers. All products are of bf16 numbers on the matrix cores, with f32 sums. A number of another type is the sum of bf16 ones, exactly:
// f16 of two, f32 of three, each the last one's remainder cut to 8 bits; a product takes all pairs. h stays f32; for f32
// results it goes on in three parts, for bf16 ones in two (2^-17 of itself, against the result's 2^-8). Two parts of 16 ranks fill the two
// halves of one instruction's 32 products.
#include <type_traits>

#include "kv8_map.hpp"
#include "step.hpp"

namespace slhip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kMaxRank = 256;
constexpr int kMaxRequests = 4096;
constexpr int kUnit = 64;          // inputs that a wave takes together: a line of 16-bit rows
constexpr int kMostSplits = 16;
constexpr int64_t kSplitRows = 65536;  // rows times ranges are at most so many, or the rows

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
    int32_t splits, rank_blocks, col_blocks;
    int32_t spare;  // columns that the last 16 ranks of one may reach into
    uint32_t* err;
};

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

__device__ __forceinline__ int32_t block_scan(int32_t v, int32_t* lds, int32_t& total)
{
    v = wave_scan(v);
    if ((threadIdx.x & 63) == 63) lds[wave_id()] = v;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kWaves; w++) {
        if (w == wave_id()) v += total;
        total += lds[w];
    }
    __syncthreads();
    return v;
}

// The same for up to 64 requests, a lane each: one memory latency, and nothing but the rows goes through LDS.
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

// The same for up to kHeld * 256 requests: a thread holds kHeld of them, so there is one memory latency.
constexpr int kHeld = 4;

template <int TM> __device__ __forceinline__ int32_t find_tile_held(const LoraArgs& a, int64_t item, int32_t* s_rows)
{
    __shared__ int32_t s_at[kWaves], s_one[3], s_before[kWaves], s_sum[kHeld][kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    int32_t s0[kHeld], n[kHeld], key[kHeld], begun = 0;
#pragma unroll
    for (int e = 0; e < kHeld; e++) {
        const int32_t j = tid + e * kThreads, at = min(j, a.B - 1);
        s0[e] = a.starts[at];
        n[e] = j < a.B ? rows_of(a, at) : 0;
        key[e] = adapter_of(a, at);
    }
#pragma unroll
    for (int e = 0; e < kHeld; e++) {
        const int32_t j = tid + e * kThreads;
        begun += __popcll(__ballot(j < a.B && item_base(s0[e], j, TM, 1) <= item));
    }
    if (lane == 0) s_at[wave] = begun;
    if (tid < TM) s_rows[tid] = -1;
    __syncthreads();
    const int32_t i = max((s_at[0] + s_at[1]) + (s_at[2] + s_at[3]) - 1, 0);
#pragma unroll
    for (int e = 0; e < kHeld; e++)
        if (tid + e * kThreads == i) {
            s_one[0] = s0[e];
            s_one[1] = n[e];
            s_one[2] = key[e];
        }
    __syncthreads();
    const int32_t at = s_one[0], rows = s_one[1], mine = s_one[2];
    const int64_t piece = item - item_base(at, i, TM, 1);
    if (piece < 0 || piece * TM >= rows) return kNoTile;
    int32_t up[kHeld], before = 0;
#pragma unroll
    for (int e = 0; e < kHeld; e++) {
        if (key[e] != mine) n[e] = 0;
        up[e] = wave_scan(n[e]);
        if (lane == 63) s_sum[e][wave] = up[e];
        up[e] -= n[e];
        before += tid + e * kThreads < i ? n[e] : 0;
    }
    before = wave_scan(before);
    if (lane == 63) s_before[wave] = before;
    __syncthreads();
    before = (s_before[0] + s_before[1]) + (s_before[2] + s_before[3]);
    const int64_t first = ((static_cast<int64_t>(before) + TM - 1) / TM + piece) * TM, off = first - before;
    if (off < 0 || off >= rows) return kNoTile;  // (below 0 where requests overlap, which none may)
    if (tid < min(static_cast<int64_t>(TM), rows - off)) s_rows[tid] = at + static_cast<int32_t>(off) + tid;
    int64_t base = -first;  // of the wave's requests
#pragma unroll
    for (int e = 0; e < kHeld; e++) {
        int64_t to = base + up[e];
        for (int w = 0; w < kWaves; w++) {
            to += w < wave ? s_sum[e][w] : 0;
            base += s_sum[e][w];
        }
        if (tid + e * kThreads > i && to >= 1) {
            for (int32_t r = 0; r < n[e] && to + r < TM; r++) s_rows[to + r] = s0[e] + r;
        }
    }
    __syncthreads();
    return mine;
}

// The rows of tile `item` into s_rows (-1 behind the last), and their adapter; kNoTile where there is none.
template <int TM> __device__ __forceinline__ int32_t find_tile(const LoraArgs& a, int64_t item, int32_t* s_rows, int32_t* lds)
{
    const int lane = threadIdx.x & 63, tid = threadIdx.x;
    if (a.B <= 64) return find_tile_64<TM>(a, item, s_rows);
    if (a.B <= kHeld * kThreads) return find_tile_held<TM>(a, item, s_rows);
    int32_t i = 0;
    {   // as row_request, by the requests' first items
        int32_t lo = 0, n = a.B;
        while (n > 64) {
            const int32_t step = (n + 63) / 64, j = lo + lane * step;
            const int32_t k = __popcll(__ballot(j < lo + n && item_base(a.starts[j < lo + n ? j : lo], j, TM, 1) <= item));
            if (k > 0) {
                lo += (k - 1) * step;
                n -= (k - 1) * step;
            }
            n = min(n, step);
        }
        const int32_t j = lo + (lane < n ? lane : 0);
        const int32_t k = __popcll(__ballot(lane < n && item_base(a.starts[j], j, TM, 1) <= item));
        i = __builtin_amdgcn_readfirstlane(lo + max(k - 1, 0));
    }
    const int32_t s0 = a.starts[i], n = rows_of(a, i), key = adapter_of(a, i);
    const int64_t piece = item - item_base(s0, i, TM, 1);
    if (piece < 0 || piece * TM >= n) return kNoTile;
    int32_t before = 0;
    for (int32_t j = tid; j < i; j += kThreads)
        if (adapter_of(a, j) == key) before += rows_of(a, j);
    block_scan(before, lds, before);
    const int64_t off = ((static_cast<int64_t>(before) + TM - 1) / TM + piece) * TM - before;
    if (off < 0 || off >= n) return kNoTile;  // (below 0 where requests overlap, which none may)
    int32_t have = static_cast<int32_t>(min(static_cast<int64_t>(TM), n - off));
    if (tid < have) s_rows[tid] = s0 + static_cast<int32_t>(off) + tid;
    for (int32_t w = i + 1; have < TM && w < a.B; w += kThreads) {
        const int32_t j = w + tid;
        const int32_t count = j < a.B && adapter_of(a, j) == key ? min(rows_of(a, j), TM) : 0;
        int32_t total;
        const int32_t at = have + block_scan(count, lds, total) - count;
        for (int32_t r = 0; r < count && at + r < TM; r++) s_rows[at + r] = a.starts[j] + r;
        have = min(have + total, TM);
    }
    if (tid >= have && tid < TM) s_rows[tid] = -1;
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

// 16 bytes of an array that ends at element `end` (and has 16 bytes at least): zeros behind its end.
template <int DT> __device__ __forceinline__ uint4 load_end(const void* p, int64_t at, int64_t end)
{
    constexpr int E = Vec<DT>::N;
    const int64_t in = min(at, end - E);
    return shift_down(load_any(static_cast<const char*>(p) + in * Vec<DT>::BYTES), static_cast<int32_t>(min(at - in, static_cast<int64_t>(E))) * Vec<DT>::BYTES);
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
    // Of an array that ends at `end`.
    __device__ __forceinline__ void load_end(const void* p, int64_t at, int64_t end)
    {
#pragma unroll
        for (int i = 0; i < kVecs; i++) w[i] = slhip::load_end<DT>(p, at + i * kPer, end);
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

template <int XT, int WT, int MT, int RB> __global__ __launch_bounds__(kThreads) void lora_shrink(LoraArgs a)
{
    constexpr int TM = 16 * MT, PX = kParts<XT>, PW = kParts<WT>;
    constexpr int U = MT * RB == 1 ? 4 : MT == 1 || XT == SLHIP_BF16 ? 2 : 1;  // units whose loads are on their way together
    __shared__ int32_t s_rows[TM], lds[kWaves];
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
    const int32_t rb = blockIdx.x % a.rank_blocks, rest = blockIdx.x / a.rank_blocks, split = rest % a.splits;
    const int32_t key = find_tile<TM>(a, rest / a.splits, s_rows, lds);
    if (key < 0) return;
    const int32_t rank = rank_of(a, key), r0 = rb * RB * 16;
    if (r0 >= rank) return;
    const int32_t units = (a.K + kUnit - 1) / kUnit, each = (units + a.splits - 1) / a.splits;
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
        const int32_t k = u * kUnit + 16 * g, n = a.K - k;
#pragma unroll
        for (int q = 0; q < RB; q++) {
            w[q].load_end(ad, min(r0 + 16 * q + c, rank - 1) * a.K + k, a.R * a.K);
            w[q].keep(n);
        }
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int32_t row = s_rows[16 * m + c];
            x[m].load_end(a.x, (row >= 0 ? row : s_rows[0]) * a.xs + k, (a.T - 1) * a.xs + a.K);
            x[m].keep(n);
        }
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
}

// ---- y = add + s B h -----------------------------------------------------------------------------------------------

typedef u32x4 u32x4_any __attribute__((aligned(2)));

__device__ __forceinline__ void store_any(char* p, const uint4& v)
{
    const u32x4 t = {v.x, v.y, v.z, v.w};
    __builtin_nontemporal_store(t, reinterpret_cast<u32x4_any*>(p));
}

// Two 16-byte pieces of each of 16 rows, by lanes c + 16 g: with both pieces of row c in lane c (a of columns before b's), or as memory
// takes them best, eight lanes a line: a of row c % 8 and b of row 8 + c % 8, of the first piece in lanes c < 8, of the second above.
// One goes over into the other by an exchange of lanes c and c +- 8.
__device__ __forceinline__ void swap_halves(uint4& a, uint4& b)
{
    const auto one = [](uint32_t& x, uint32_t& y) {
        const uint32_t t = __builtin_amdgcn_update_dpp(static_cast<int>(y), static_cast<int>(x), 0x128, 0xF, 0x3, false);  // row_ror:8 into c < 8
        x = __builtin_amdgcn_update_dpp(static_cast<int>(x), static_cast<int>(y), 0x128, 0xF, 0xC, false);                 // and into c >= 8
        y = t;
    };
    one(a.x, b.x);
    one(a.y, b.y);
    one(a.z, b.z);
    one(a.w, b.w);
}

// The two bf16 parts of v, rounded: what is left of an infinity is 0.
__device__ __forceinline__ float low_part(float v, float hi) { return fabsf(hi) < INFINITY ? v - hi : 0.0f; }

template <int YT, int WT, int MT> __global__ __launch_bounds__(kThreads) void lora_expand(LoraArgs a)
{
    constexpr int TM = 16 * MT, PW = kParts<WT>;
    constexpr int H = YT == SLHIP_BF16 ? 1 : 2;  // instructions that take h's parts of 16 ranks
    __shared__ int32_t s_rows[TM], lds[kWaves];
    extern __shared__ uint4 s_h[];  // [MT][ranks / 16][H][64]: the second operand of 16 ranks
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), c = lane & 15, g = lane >> 4;
    const int32_t cb = blockIdx.x % a.col_blocks;
    const int32_t key = find_tile<TM>(a, blockIdx.x / a.col_blocks, s_rows, lds);
    if (key == kNoTile || (key < 0 && a.add == a.y)) return;
    const int32_t rank = key < 0 ? 0 : rank_of(a, key), tiles = (rank + 15) / 16;
    const float scale = key < 0 || !a.scale ? 1.0f : a.scale[key];
    const char* const ad = static_cast<const char*>(a.b) + (key < 0 ? 0 : key * a.sb * Vec<WT>::BYTES);
    // 64 columns of a row are kPieces of 16 bytes a lane. Product u has those of 16 columns of which a lane (c, g) gets four in a row,
    // row c's: f32 4 g of the u-th 16, bf16 eight with those of u + 1 (u even), 8 g of the u-th 16.
    constexpr int E = Vec<YT>::N, kPieces = 16 / E;
    const auto column = [&](int32_t n0, int u) {
        return min(n0 + (YT == SLHIP_F32 ? 16 * u + c : 32 * (u >> 1) + 8 * (c >> 2) + 4 * (u & 1) + (c & 3)), a.N - 1);  // behind the last: not stored
    };
    // Where a lane loads and stores (swap_halves): rows c % 8 and 8 + c % 8 of each 16, of pieces 2 p + c / 8.
    const int32_t in = (c >> 3) * 4 * E + g * E;
    const char* from[MT][2];
    char* to[MT][2];
    bool there[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int32_t row = s_rows[16 * m + 8 * h + (c & 7)];
            there[m][h] = row >= 0;
            from[m][h] = static_cast<const char*>(a.add) + ((row >= 0 ? row : s_rows[0]) * a.as + in) * Vec<YT>::BYTES;
            to[m][h] = static_cast<char*>(a.y) + ((row >= 0 ? row : 0) * a.ys + in) * Vec<YT>::BYTES;
        }
    uint4 add[MT][kPieces];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < kPieces; i++) add[m][i] = make_uint4(0, 0, 0, 0);
    Run<WT, 8> w[4];
    uint32_t wp[4];
#pragma unroll
    for (int u = 0; u < 4; u++) wp[u] = static_cast<uint32_t>(column(0, u) * a.R + 8 * (g & 1)) * Vec<WT>::BYTES;
    // whole: 64 columns, whose last 16 ranks end inside the adapter
    const auto is_whole = [&](int32_t n0) { return n0 + 64 + a.spare <= a.N; };
    const auto fetch_w = [&](int32_t n0, int q, bool whole) __attribute__((always_inline)) {
        if (whole) {
            const char* const at = ad + (static_cast<int64_t>(n0) * a.R + 16 * q) * Vec<WT>::BYTES;
#pragma unroll
            for (int u = 0; u < 4; u++) w[u].load(at + wp[u]);
        } else {
#pragma unroll
            for (int u = 0; u < 4; u++) w[u].load_end(ad, column(n0, u) * a.R + 16 * q + 8 * (g & 1), a.N * a.R);
        }
    };
    const auto fetch = [&](int32_t n0) __attribute__((always_inline)) {
        const bool whole = is_whole(n0);
        if (tiles > 0) fetch_w(n0, 0, whole);
        if (!a.add) return;
        if (whole) {
            const int64_t at = static_cast<int64_t>(n0) * Vec<YT>::BYTES;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int i = 0; i < kPieces; i++) {
                    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(from[m][i & 1] + at + (i >> 1) * 128));
                    add[m][i] = make_uint4(v.x, v.y, v.z, v.w);
                }
        } else {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int i = 0; i < kPieces; i++)
                    add[m][i] = load_end<YT>(a.add, (from[m][i & 1] - static_cast<const char*>(a.add)) / Vec<YT>::BYTES + n0 + (i >> 1) * 8 * E, (a.T - 1) * a.as + a.N);
        }
    };
    // thread blocks that run together take neighbouring columns: the same columns of many rows lie in few memory channels
    const int32_t first = (cb * kWaves + wave) * 64, step = a.col_blocks * kWaves * 64;
    if (first < a.N) fetch(first);
    for (int t = tid; t < MT * tiles * 32; t += kThreads) {  // eight ranks of a row
        const int m = t / (tiles * 32), q = t / 32 - m * tiles, l = t & 31;
        const int32_t at = s_rows[16 * m + (l & 15)], r = 16 * q + 8 * (l >> 4);
        float f[8] = {};
        if (at >= 0) {
            const float* h = a.h + static_cast<int64_t>(at) * a.R16 + r;
            const int64_t step = a.T * a.R16;
            for (int s0 = 0; s0 < a.splits; s0 += 8) {
                f32x4 x[8][2];
#pragma unroll
                for (int s = 0; s < 8; s++)
#pragma unroll
                    for (int e = 0; e < 2; e++) x[s][e] = s0 + s < a.splits ? reinterpret_cast<const f32x4*>(h + (s0 + s) * step)[e] : f32x4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < 8; s++)
#pragma unroll
                    for (int e = 0; e < 8; e++) f[e] += x[s][e >> 2][e & 3];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = r + e < rank ? f[e] * scale : 0.0f;
        uint4* to = s_h + ((m * tiles + q) * H) * 64 + l;  // the parts of a row's 16 ranks: lanes l and l + 32
        if constexpr (H == 1) {
            float lo[8];
            to[0] = Vec<SLHIP_BF16>::pack(f);
            Vec<SLHIP_BF16>::unpack(to[0], lo);
#pragma unroll
            for (int e = 0; e < 8; e++) lo[e] = low_part(f[e], lo[e]);
            to[32] = Vec<SLHIP_BF16>::pack(lo);
        } else {
            bf16x8 p[3];
            cut(f, p);
#pragma unroll
            for (int i = 0; i < 3; i++) to[32 * i] = __builtin_bit_cast(uint4, p[i]);
            to[96] = make_uint4(0, 0, 0, 0);
        }
    }
    __syncthreads();
    for (int32_t n0 = first; n0 < a.N; n0 += step) {
        if (n0 > first) fetch(n0);
        const bool whole = is_whole(n0);
        f32x4 acc[MT][4];
        const auto multiply = [&](int q, auto begins) __attribute__((always_inline)) {
            if (16 * q + 16 > rank) {  // ranks behind the last may hold anything
#pragma unroll
                for (int u = 0; u < 4; u++) w[u].keep(rank - 16 * q - 8 * (g & 1));
            }
            bf16x8 pw[4][PW];
#pragma unroll
            for (int u = 0; u < 4; u++) w[u].parts(0, pw[u]);
            if (q + 1 < tiles) fetch_w(n0, q + 1, whole);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int h = H - 1; h >= 0; h--) {
                    const bf16x8 x = __builtin_bit_cast(bf16x8, s_h[((m * tiles + q) * H + h) * 64 + lane]);
#pragma unroll
                    for (int i = PW - 1; i >= 0; i--)
#pragma unroll
                        for (int u = 0; u < 4; u++)
                            acc[m][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pw[u][i], x, begins && h == H - 1 && i == PW - 1 ? f32x4{0, 0, 0, 0} : acc[m][u], 0, 0, 0);
                }
        };
        if (tiles > 0) {
            multiply(0, std::true_type{});
            for (int q = 1; q < tiles; q++) multiply(q, std::false_type{});
        } else {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int u = 0; u < 4; u++) acc[m][u] = f32x4{0, 0, 0, 0};
        }
        const int64_t at = static_cast<int64_t>(n0) * Vec<YT>::BYTES;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int p = 0; p < kPieces; p += 2) {
                uint4 v[2] = {add[m][p], add[m][p + 1]};
                swap_halves(v[0], v[1]);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float f[E];
                    Vec<YT>::unpack(v[i], f);
#pragma unroll
                    for (int e = 0; e < E; e++) f[e] += acc[m][(p + i) * E / 4 + e / 4][e & 3];
                    v[i] = Vec<YT>::pack(f);
                }
                swap_halves(v[0], v[1]);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    char* const place = to[m][i] + at + p * 64;
                    const int32_t n = a.N - (n0 + p * 4 * E + in);
                    if (whole || n >= E) {
                        if (there[m][i]) store_any(place, v[i]);
                    } else if (there[m][i]) {  // the last ones of a row
                        float f[E];
                        Vec<YT>::unpack(v[i], f);
#pragma unroll
                        for (int e = 0; e < E; e++)
                            if (e < n) Vec<YT>::store1(place, e, f[e]);
                    }
                }
            }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------

static int64_t round16(int64_t n) { return (n + 15) & ~int64_t{15}; }

static int64_t work_of(int64_t T, int64_t R)
{
    const int64_t most = T > kSplitRows ? T : kSplitRows;
    return (T * kMostSplits < most ? T * kMostSplits : most) * round16(R) * 4;
}

template <int XT, int WT, int MT> static int shrink(const LoraArgs& a, int64_t blocks, hipStream_t st)
{
    constexpr int few = MT == 1 ? 1 : 2;
    const auto kernel = a.R16 <= 16 ? lora_shrink<XT, WT, few, 1> : a.R16 <= 32 ? lora_shrink<XT, WT, few, 2> : lora_shrink<XT, WT, MT, 4>;
    kernel<<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(a);
    return check_launch("lora_shrink");
}

template <int YT, int WT, int MT> static int expand(const LoraArgs& a, int64_t blocks, hipStream_t st)
{
    const int lds = MT * a.R16 * (YT == SLHIP_BF16 ? 64 : 128);
    if (lds > 60000)
        SLHIP_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&lora_expand<YT, WT, MT>), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    lora_expand<YT, WT, MT><<<static_cast<unsigned>(blocks), kThreads, lds, st>>>(a);
    return check_launch("lora_expand");
}

template <int WT> static int launch(int dtype_x, int dtype_y, LoraArgs& a, hipStream_t st)
{
    const bool few = a.T <= 32 * static_cast<int64_t>(a.B);
    const int first_tile = few ? 16 : a.R16 <= 32 ? 32 : 64, second_tile = few ? 16 : a.R16 <= 32 ? 32 : 64;
    const int64_t first_items = item_count(a.T, a.B, first_tile, 1), items = item_count(a.T, a.B, second_tile, 1);
    a.rank_blocks = a.R16 <= 32 ? 1 : (a.R16 + 63) / 64;
    // ranges of K: enough thread blocks for the machine, of 256 inputs at least
    int64_t splits = (few ? 4096 : 1024) / (first_items * a.rank_blocks), most = a.K / 256;
    if (splits > most) splits = most;
    if (splits > kMostSplits) splits = kMostSplits;
    if (splits > kSplitRows / a.T) splits = kSplitRows / a.T;
    a.splits = splits < 1 ? 1 : static_cast<int32_t>(splits);
    const int64_t cols = (a.N + 64 * kWaves - 1) / (64 * kWaves);
    int64_t steps = few && a.B > 64 ? 1 : (items * cols + 2047) / 2048;
    if (steps > 8) steps = 8;
    a.col_blocks = static_cast<int32_t>((cols + steps - 1) / steps);
    const int64_t first = first_items * a.splits * a.rank_blocks, second = items * a.col_blocks;
    if (first > 0xFFFFFF || second > 0xFFFFFF) return fail(SLHIP_ERR_UNSUPPORTED, "lora: too many rows");
    const bool f32 = dtype_x == SLHIP_F32;
    const int e = few ? f32 ? shrink<SLHIP_F32, WT, 1>(a, first, st) : shrink<SLHIP_BF16, WT, 1>(a, first, st)
                      : f32 ? shrink<SLHIP_F32, WT, 4>(a, first, st) : shrink<SLHIP_BF16, WT, 4>(a, first, st);
    if (e) return e;
    const bool out32 = dtype_y == SLHIP_F32;
    if (second_tile == 16) return out32 ? expand<SLHIP_F32, WT, 1>(a, second, st) : expand<SLHIP_BF16, WT, 1>(a, second, st);
    if (second_tile == 32) return out32 ? expand<SLHIP_F32, WT, 2>(a, second, st) : expand<SLHIP_BF16, WT, 2>(a, second, st);
    return out32 ? expand<SLHIP_F32, WT, 4>(a, second, st) : expand<SLHIP_BF16, WT, 4>(a, second, st);
}

}  // namespace slhip

using namespace slhip;

extern "C" SLHIP_API int64_t slhip_lora_work_bytes(int64_t tokens, int64_t max_rank)
{
    if (tokens < 0 || tokens > 0x7FFFFFFFll - 65536 || max_rank < 1 || max_rank > kMaxRank) {
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
    if (set->adapters > 0x7FFFFFFF || widest > 0x7FFFFFFF || set->K > (1 << 24) || set->N > (1 << 24) || rows->tokens > 0x7FFFFFFFll - 65536)
        return fail(SLHIP_ERR_UNSUPPORTED, "lora: too many adapters, inputs, outputs or rows (a matrix of an adapter has less than 2^31 bytes)");
    if (x_stride < set->K || y_stride < set->N || (add && add_stride < set->N))
        return fail(SLHIP_ERR_INVALID, "lora: a row stride is smaller than the row");
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
    a.spare = static_cast<int32_t>((a.R16 - 1) / a.R);
    a.K = static_cast<int32_t>(set->K);
    a.N = static_cast<int32_t>(set->N);
    a.rank = set->rank;
    a.scale = set->scale;
    a.B = static_cast<int32_t>(rows->requests);
    a.T = rows->tokens;
    a.starts = rows->starts;
    a.adapter = rows->adapter;
    a.h = static_cast<float*>(work);
    int e = error_word(&a.err);
    if (e) return e;
    hipStream_t st = to_stream(stream);
    if (set->dtype == SLHIP_F32) return launch<SLHIP_F32>(dtype_x, dtype_y, a, st);
    if (set->dtype == SLHIP_F16) return launch<SLHIP_F16>(dtype_x, dtype_y, a, st);
    return launch<SLHIP_BF16>(dtype_x, dtype_y, a, st);
}
