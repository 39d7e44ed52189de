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
    int32_t splits, rank_blocks, col_blocks, col_steps;
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

// The rows of tile `item` into s_rows (-1 behind the last), and their adapter; kNoTile where there is none.
template <int TM> __device__ __forceinline__ int32_t find_tile(const LoraArgs& a, int64_t item, int32_t* s_rows, int32_t* lds)
{
    const int lane = threadIdx.x & 63, tid = threadIdx.x;
    if (a.B <= 64) return find_tile_64<TM>(a, item, s_rows);
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

// N neighbours (8 or 16) of which the first n are there; the others are 0.
template <int DT, int N> struct Run {
    static constexpr int kVecs = N * Vec<DT>::BYTES / 16, kPer = Vec<DT>::N;
    uint4 w[kVecs];
    __device__ __forceinline__ void load(const void* p, int64_t at)
    {
        const char* c = static_cast<const char*>(p) + at * Vec<DT>::BYTES;
#pragma unroll
        for (int i = 0; i < kVecs; i++) w[i] = load_any(c + 16 * i);
    }
    __device__ __forceinline__ void load_some(const void* p, int64_t at, int64_t n)
    {
        const char* c = static_cast<const char*>(p) + at * Vec<DT>::BYTES;
#pragma unroll
        for (int i = 0; i < kVecs; i++) {
            w[i] = make_uint4(0, 0, 0, 0);
            if (n >= (i + 1) * kPer) {
                w[i] = load_any(c + 16 * i);
            } else if (n > i * kPer) {
                float f[kPer] = {};
                for (int j = 0; j < kPer; j++)
                    if (i * kPer + j < n) f[j] = Vec<DT>::load1(c, i * kPer + j);
                w[i] = Vec<DT>::pack(f);  // the same bits again
            }
        }
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
    int64_t xp[MT], ap[RB];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int32_t row = s_rows[16 * m + c];
        xp[m] = (row >= 0 ? row : s_rows[0]) * a.xs + 16 * g;
    }
#pragma unroll
    for (int q = 0; q < RB; q++) ap[q] = key * a.sa + static_cast<int64_t>(min(r0 + 16 * q + c, rank - 1)) * a.K + 16 * g;
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
            const int64_t k = static_cast<int64_t>(u + v * kWaves) * kUnit;
#pragma unroll
            for (int q = 0; q < RB; q++)
                if (q == 0 || q < ranks) w[v][q].load(a.a, ap[q] + k);
#pragma unroll
            for (int m = 0; m < MT; m++) x[v][m].load(a.x, xp[m] + k);
        }
#pragma unroll
        for (int v = 0; v < U; v++) multiply(x[v], w[v]);
    }
    for (; u < u1; u += kWaves) {
        Run<XT, 16> x[MT];
        Run<WT, 16> w[RB];
        const int64_t k = static_cast<int64_t>(u) * kUnit, n = a.K - k - 16 * g;
#pragma unroll
        for (int q = 0; q < RB; q++) w[q].load_some(a.a, ap[q] + k, n);
#pragma unroll
        for (int m = 0; m < MT; m++) x[m].load_some(a.x, xp[m] + k, n);
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

// Eight neighbours of a row of add or y, the first n of them.
typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <int DT> struct Eight {
    static constexpr int kVecs = 8 * Vec<DT>::BYTES / 16, kPer = Vec<DT>::N;
    u32x4 w[kVecs];
    __device__ __forceinline__ void load(const void* p, int64_t at)
    {
        const char* c = static_cast<const char*>(p) + at * Vec<DT>::BYTES;
#pragma unroll
        for (int i = 0; i < kVecs; i++) w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(c + 16 * i));
    }
    __device__ __forceinline__ void load_some(const void* p, int64_t at, int32_t n)
    {
        const char* c = static_cast<const char*>(p) + at * Vec<DT>::BYTES;
#pragma unroll
        for (int i = 0; i < kVecs; i++) {
            w[i] = u32x4{0, 0, 0, 0};
            if (n >= 8) {
                w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(c + 16 * i));
            } else if (n > i * kPer) {
                float f[kPer] = {};
                for (int j = 0; j < kPer; j++)
                    if (i * kPer + j < n) f[j] = Vec<DT>::load1(c, i * kPer + j);
                const uint4 v = Vec<DT>::pack(f);  // the same bits again
                w[i] = u32x4{v.x, v.y, v.z, v.w};
            }
        }
    }
    __device__ __forceinline__ void floats(float (&f)[8]) const
    {
#pragma unroll
        for (int i = 0; i < kVecs; i++) Vec<DT>::unpack(make_uint4(w[i].x, w[i].y, w[i].z, w[i].w), &f[i * kPer]);
    }
    __device__ static __forceinline__ void store(void* p, int64_t at, int32_t n, const float (&f)[8])
    {
        char* c = static_cast<char*>(p) + at * Vec<DT>::BYTES;
        if (n >= 8) {
#pragma unroll
            for (int i = 0; i < kVecs; i++) {
                const uint4 w = Vec<DT>::pack(&f[i * kPer]);
                const u32x4 t = {w.x, w.y, w.z, w.w};
                __builtin_nontemporal_store(t, reinterpret_cast<u32x4_any*>(c + 16 * i));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < n) Vec<DT>::store1(c, j, f[j]);
        }
    }
};

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
    int32_t row[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) row[m] = s_rows[16 * m + c];
    const int64_t base = key < 0 ? 0 : key * a.sb;
    // Columns of a product u: a lane gets four in a row, with u + 1 (u even) eight. Those behind the last are others, which are not stored.
    const auto column = [&](int32_t n0, int u) { return min(n0 + 32 * (u >> 1) + 8 * (c >> 2) + 4 * (u & 1) + (c & 3), a.N - 1); };
    Eight<YT> add[MT][2];
    Run<WT, 8> w[4];
    const auto fetch_w = [&](int32_t n0, int q) __attribute__((always_inline)) {
        const int32_t r = 16 * q + 8 * (g & 1);
        if (16 * q + 16 <= rank) {
#pragma unroll
            for (int u = 0; u < 4; u++) w[u].load(a.b, base + static_cast<int64_t>(column(n0, u)) * a.R + r);
        } else {  // ranks behind the last are not read
#pragma unroll
            for (int u = 0; u < 4; u++) w[u].load_some(a.b, base + static_cast<int64_t>(column(n0, u)) * a.R + r, rank - r);
        }
    };
    const auto fetch = [&](int32_t n0) __attribute__((always_inline)) {
        if (tiles > 0) fetch_w(n0, 0);
        if (a.add && n0 + 64 <= a.N) {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int p = 0; p < 2; p++) add[m][p].load(a.add, (row[m] >= 0 ? row[m] : s_rows[0]) * a.as + n0 + 32 * p + 8 * g);
        } else {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const int32_t n = n0 + 32 * p + 8 * g;
                    add[m][p].load_some(a.add, row[m] * a.as + n, a.add && row[m] >= 0 ? a.N - n : 0);
                }
        }
    };
    const int32_t first = (cb * a.col_steps * kWaves + wave) * 64;
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
    for (int j = 0; j < a.col_steps; j++) {
        const int32_t n0 = first + j * kWaves * 64;
        if (n0 >= a.N) break;
        if (j > 0) fetch(n0);
        f32x4 acc[MT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int u = 0; u < 4; u++) acc[m][u] = f32x4{0, 0, 0, 0};
        for (int q = 0; q < tiles; q++) {
            bf16x8 pw[4][PW];
#pragma unroll
            for (int u = 0; u < 4; u++) w[u].parts(0, pw[u]);
            if (q + 1 < tiles) fetch_w(n0, q + 1);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int h = H - 1; h >= 0; h--) {
                    const bf16x8 x = __builtin_bit_cast(bf16x8, s_h[((m * tiles + q) * H + h) * 64 + lane]);
#pragma unroll
                    for (int i = PW - 1; i >= 0; i--)
#pragma unroll
                        for (int u = 0; u < 4; u++) acc[m][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pw[u][i], x, acc[m][u], 0, 0, 0);
                }
        }
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const int32_t n = n0 + 32 * p + 8 * g;
                float f[8];
                add[m][p].floats(f);
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] += acc[m][2 * p + (e >> 2)][e & 3];
                if (row[m] >= 0 && n < a.N) Eight<YT>::store(a.y, row[m] * a.ys + n, a.N - n, f);
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
    const auto kernel = a.R16 <= 16 ? lora_shrink<XT, WT, MT, 1> : a.R16 <= 32 ? lora_shrink<XT, WT, MT, 2> : lora_shrink<XT, WT, MT, 4>;
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

template <int WT, int MT> static int launch(int dtype_x, int dtype_y, LoraArgs& a, hipStream_t st)
{
    const int64_t items = item_count(a.T, a.B, 16 * MT, 1);
    a.rank_blocks = a.R16 <= 32 ? 1 : (a.R16 + 63) / 64;
    // ranges of K: enough thread blocks for the machine, of 512 inputs at least
    int64_t splits = 4096 / (items * a.rank_blocks), most = a.K / 512;
    if (splits > most) splits = most;
    if (splits > kMostSplits) splits = kMostSplits;
    if (splits > kSplitRows / a.T) splits = kSplitRows / a.T;
    a.splits = splits < 1 ? 1 : static_cast<int32_t>(splits);
    const int64_t cols = (a.N + 64 * kWaves - 1) / (64 * kWaves);
    a.col_steps = items * cols > 4096 ? 4 : 1;
    a.col_blocks = static_cast<int32_t>((cols + a.col_steps - 1) / a.col_steps);
    const int64_t first = items * a.splits * a.rank_blocks, second = items * a.col_blocks;
    if (first > 0xFFFFFF || second > 0xFFFFFF) return fail(SLHIP_ERR_UNSUPPORTED, "lora: too many rows");
    const int e = dtype_x == SLHIP_F32 ? shrink<SLHIP_F32, WT, MT>(a, first, st) : shrink<SLHIP_BF16, WT, MT>(a, first, st);
    if (e) return e;
    return dtype_y == SLHIP_F32 ? expand<SLHIP_F32, WT, MT>(a, second, st) : expand<SLHIP_BF16, WT, MT>(a, second, st);
}

template <int WT> static int launch(int dtype_x, int dtype_y, LoraArgs& a, hipStream_t st)
{
    return a.T > 32 * static_cast<int64_t>(a.B) ? launch<WT, 4>(dtype_x, dtype_y, a, st) : launch<WT, 1>(dtype_x, dtype_y, a, st);
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
    if (set->max_rank > kMaxRank) return fail(SLHIP_ERR_UNSUPPORTED, "lora: more than %d ranks", kMaxRank);
    if (rows->requests > kMaxRequests) return fail(SLHIP_ERR_UNSUPPORTED, "lora: more than %d requests", kMaxRequests);
    if (set->adapters > 0x7FFFFFFF || set->K > (1 << 24) || set->N > (1 << 24) || rows->tokens > 0x7FFFFFFFll - 65536)
        return fail(SLHIP_ERR_UNSUPPORTED, "lora: too many adapters, inputs, outputs or rows");
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
