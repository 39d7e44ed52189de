// Causal attention over the 8-bit paged cache (slhip_kv8_attention): the kernels.
//
// Mathematics. For a query row q with position p and keys j <= p (and j > p - window):
//   z_j = scale * ks_b * (q . k_j)  (capped, slopes added), ks_b and vs_b = 2^ev_b the scales of key j's block b,
//   y   = sum_j e^z_j vs_b c_j / sum_j e^z_j,  k_j and c_j the codes.
// With t_j = z_j log2(e) + ev_b and M the running maximum of t_j, w_j = 2^(t_j - M) <= 1 holds the whole weight of code
// c_j, the block's scale included: o = sum_j w_j c_j, l = sum_j w_j 2^-ev_b, y = o / l. So V's codes go to the matrix
// cores as they are, the scale costs nothing (it rides in the addition of the exponent), and what is rounded to f16, w_j,
// is rounded relative to the largest contribution, whatever the scales of the blocks are.
//
// Numbers. int8 and E4M3 codes are exact in f16. A query row is multiplied by the power of two that brings its largest
// value to [2^14, 2^15): bf16 values are then exact in f16 down to 2^-29 of the row's largest (below that they round to
// 2^-40 of it), f32 values are the sum of two f16 parts to 2^-22 (or 2^-40 of the largest). w_j goes to the matrix cores
// scaled by 2^kBias, in f16 (2^-11 of itself, 2^-33 of the largest contribution at least) for bf16 activations, whose
// output is rounded to 2^-8 anyway, and as two f16 parts (2^-22) for f32. Products are exact, sums, maxima and l are f32.
//
// Layout. A tile is 64 keys, four 16-key sub-blocks, and a wave works on NT * 16 query rows of one K/V head: rows are
// (token, query head) pairs, so all query heads of a K/V head share its loads. With mfma 16x16x32 (A[m][8g+j], B[8g+j][n],
// C[4g+r][n] in lane (n or m) + 16 g):
//   S^T = K Q^T: row m of the four 16-key products t = 0..3 is key 4t + m%4 of sub-block m/4, so lane (c, g) ends with
//   t_j of row c for all 16 keys of sub-block g -- one pair of scales, one page, one mask a lane --
//   O^T = V^T P^T: k index 8g + j of step s is key 8s + j of sub-block g, which is what lane (c, g) holds: weights go from
//   the first product to the second without leaving their lane, and V's 16 keys of a dim are one 16-byte load.
// The dims of the first product are taken in the order of the lanes' 16-byte loads (dim 64h + 16g + 8s + j at step h, s).
#pragma once

#include "kv8.hpp"

namespace slhip {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;
constexpr float kBias = 8.0f;  // weights are at most 2^kBias in f16
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNone = -1e30f;  // a maximum of nothing: finite, so that differences with -inf stay numbers

struct Kv8AttnArgs {
    Kv8Dev c;
    const void* q;
    void* y;
    int64_t qt, qh, yt, yh;
    int32_t G;                   // query heads of a K/V head
    float scale, cap;
    int32_t window;              // 0: none
    const float* slopes;
    int32_t min_rows, max_rows;  // the launch takes requests of (min_rows, max_rows] query rows a K/V head
    bool strict;                 // requests above max_rows are an error here (no other launch takes them)
    int32_t units;               // wave tiles: most units a head's requests are cut into, beyond one for each
    int32_t tile_tokens, splits; // block tiles: rows' tokens of a tile, key ranges it is cut into
    float* part;                 // sums of key ranges
};

// ---- codes ----------------------------------------------------------------------------------------------------

// 16 codes as f16: the first 8 and the last 8.
template <int FMT> __device__ __forceinline__ void codes_f16(const uint4& w, f16x8& a, f16x8& b)
{
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
    f16x2 h[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (FMT == SLHIP_KV8_E4M3) {
            h[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d[i], 1.0f, false);
            h[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d[i], 1.0f, true);
        } else {  // bits 0x6400 + u are 1024 + u for u = code + 128
            const uint32_t u = d[i] ^ 0x80808080u;
            const f16x2 k = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
            h[2 * i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - k;
            h[2 * i + 1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - k;
        }
    }
    a = f16x8{h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
    b = f16x8{h[4].x, h[4].y, h[5].x, h[5].y, h[6].x, h[6].y, h[7].x, h[7].y};
}

// Keeps the first n (0..16) of a sub-block's 16 codes; the others become 0.
__device__ __forceinline__ uint4 first_codes(const uint4& w, int n)
{
    const auto m = [n](int j) { const int k = min(max(n - 4 * j, 0), 4); return k == 4 ? 0xFFFFFFFFu : (1u << (8 * k)) - 1; };
    return make_uint4(w.x & m(0), w.y & m(1), w.z & m(2), w.w & m(3));
}

__device__ __forceinline__ f16x2 to_f16x2(float a, float b)
{
    const f32x2_t v = {a, b};
    return __builtin_convertvector(v, f16x2);
}

// ---- lanes ----------------------------------------------------------------------------------------------------

// Over the four lanes of a row (c, c + 16, c + 32, c + 48).
__device__ __forceinline__ float row_max(float v)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float row_sum(float v)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// ---- a lane's key blocks -----------------------------------------------------------------------------------------

// A sub-block of 16 keys from `key`: its block, or block 0 and no keys where there is none to see.
struct SubBlock {
    int64_t at;    // (block * heads + head) of the scales
    int32_t sub;   // which 16 keys of the block
    int32_t keys;  // how many are below `end`
    int32_t bad;   // a block id outside the cache (0 where it is fine: -1 is bad, too)
    int32_t id;
};

// The table entry of the sub-block at `key` (any address in the table where the key is behind `end`).
__device__ __forceinline__ int32_t block_id(const Kv8Dev& c, const int32_t* table, int32_t key, int32_t end)
{
    return table[min(key, end - 1) >> c.shift];
}

__device__ __forceinline__ SubBlock sub_block(const Kv8Dev& c, int32_t id, int32_t head, int32_t key, int32_t end)
{
    SubBlock s;
    const bool here = key < end, fine = id >= 0 && id < c.blocks;
    s.id = id;
    s.bad = here && !fine;
    s.at = static_cast<int64_t>(fine ? id : 0) * c.heads + head;
    s.sub = (key >> 4) & ((1 << (c.shift - 4)) - 1);
    s.keys = here && fine ? min(end - key, 16) : 0;
    return s;
}

// ---- rows -------------------------------------------------------------------------------------------------------

// Query row `row` (token * G + head of the group) of a request, or none.
struct Row {
    int32_t pos;
    float back;   // scale of the scores: scale / the power of two that the row was multiplied by
    float slope;  // slopes[h] * log2(e)
};

// Loads NP f16 parts of the row's lane share: q[p][h][s] holds dims 64h + 16g + 8s + (0..7). Dims past D are 0.
template <int DT, int DP, int NP>
__device__ __forceinline__ Row load_row(const Kv8AttnArgs& a, const Kv8Request& r, int32_t head, int32_t row, bool valid,
                                        f16x8 (&q)[NP][DP / 64][2])
{
    const int g = (threadIdx.x & 63) >> 4;
    const int32_t tok = valid ? row / a.G : 0, qh = head * a.G + (valid ? row % a.G : 0);
    const int64_t base = (static_cast<int64_t>(r.first) + tok) * a.qt + qh * a.qh;
    const bool vec = reinterpret_cast<uintptr_t>(a.q) % (DT == SLHIP_F32 ? 16 : 8) == 0 && (a.qt | a.qh) % 4 == 0;
    float f[DP / 64][16];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < DP / 64; h++) {
        const int d = 64 * h + 16 * g;
        const bool in = valid && d < a.c.D;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            float4 w = make_float4(0, 0, 0, 0);
            if (in) {
                if (vec) {
                    w = load4f<DT>(a.q, base + d + j);
                } else {
                    w = make_float4(Vec<DT>::load1(a.q, base + d + j), Vec<DT>::load1(a.q, base + d + j + 1),
                                    Vec<DT>::load1(a.q, base + d + j + 2), Vec<DT>::load1(a.q, base + d + j + 3));
                }
            }
            f[h][j] = w.x; f[h][j + 1] = w.y; f[h][j + 2] = w.z; f[h][j + 3] = w.w;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) top = max(top, __float_as_uint(f[h][j]) & 0x7FFFFFFFu);
    }
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
    // multiply by 2^(14 - e): biased exponents; rows that are tiny, or not finite, by a power that stays in range
    const int e = static_cast<int>(top >> 23) - 127, up = e > 127 ? 0 : 14 - max(e, -100);
    const float mul = __uint_as_float(static_cast<uint32_t>(127 + min(up, 114)) << 23);
#pragma unroll
    for (int h = 0; h < DP / 64; h++)
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float x0 = f[h][8 * s + j] * mul, x1 = f[h][8 * s + j + 1] * mul;
                const f16x2 hi = to_f16x2(x0, x1);
                q[0][h][s][j] = hi.x;
                q[0][h][s][j + 1] = hi.y;
                if constexpr (NP == 2) {
                    const f16x2 lo = to_f16x2(x0 - static_cast<float>(hi.x), x1 - static_cast<float>(hi.y));
                    q[1][h][s][j] = lo.x;
                    q[1][h][s][j + 1] = lo.y;
                }
            }
    Row o;
    o.pos = r.past + tok;
    o.back = a.scale / mul;
    o.slope = a.slopes ? a.slopes[qh] * kLog2e : 0.0f;
    return o;
}

// tanh to about 2^-23 of itself near 0 and 2^-23 elsewhere: the odd series below 0.15, (1 - e) / (1 + e) with
// e = 2^(-2 |y| log2 e) above it, where the numerator has lost at most three bits.
__device__ __forceinline__ float tanh_f(float y)
{
    const float u = fabsf(y), u2 = u * u;
    const float e = __builtin_amdgcn_exp2f(u * (-2.0f * kLog2e));
    const float big = (1.0f - e) * recip_nr(1.0f + e);
    const float small = u * fmaf(u2, fmaf(u2, fmaf(u2, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    return copysignf(u < 0.15f ? small : big, y);
}

// The softmax of one tile and row: S (codes' products of the lane's 16 keys, key 4t + r at S[t][r]) becomes weights.
// lo <= key < hi of the sub-block are seen. m, l: the row's running maximum, the lane's part of its sum.
struct TileScale {
    float k;         // ks
    float ev, down;  // log2(vs), 1 / vs
};

template <int NP>
__device__ __forceinline__ float tile_softmax(const Kv8AttnArgs& a, f32x4 (&S)[4], const Row& row, const TileScale& sc, int32_t key0,
                                              int lo, int hi, bool masked, float& m, float& l, f16x8 (&p)[NP][2])
{
    const float k2 = row.back * sc.k * kLog2e;
    float mx = -INFINITY;
    if (a.cap > 0.0f) {
        const float in = row.back * sc.k / a.cap, out = a.cap * kLog2e;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) S[t][r] = fmaf(tanh_f(S[t][r] * in), out, sc.ev);
    } else {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) S[t][r] = fmaf(S[t][r], k2, sc.ev);
    }
    if (a.slopes) {
        const float first = static_cast<float>(key0 - row.pos);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) S[t][r] = fmaf(row.slope, first + static_cast<float>(4 * t + r), S[t][r]);
    }
    if (masked) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) S[t][r] = 4 * t + r >= lo && 4 * t + r < hi ? S[t][r] : -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < 4; t++) mx = fmaxf(fmaxf(fmaxf(mx, S[t][0]), fmaxf(S[t][1], S[t][2])), S[t][3]);
    const float was = m;
    m = fmaxf(m, row_max(mx));
    const float shift = m - kBias;
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const int t = 2 * s + (j >> 2), r = j & 3;
            const float w0 = __builtin_amdgcn_exp2f(S[t][r] - shift), w1 = __builtin_amdgcn_exp2f(S[t][r + 1] - shift);
            sum += w0 + w1;
            const f16x2 hi2 = to_f16x2(w0, w1);
            p[0][s][j] = hi2.x;
            p[0][s][j + 1] = hi2.y;
            if constexpr (NP == 2) {
                const f16x2 lo2 = to_f16x2(w0 - static_cast<float>(hi2.x), w1 - static_cast<float>(hi2.y));
                p[1][s][j] = lo2.x;
                p[1][s][j + 1] = lo2.y;
            }
        }
    const float alpha = __builtin_amdgcn_exp2f(was - m);
    l = fmaf(sum, sc.down, l * alpha);
    return alpha;
}

__device__ __forceinline__ TileScale tile_scale(const Kv8Dev& c, const SubBlock& s, float ks, float vs)
{
    // a scale that is NaN makes the weights of the keys that are seen NaN, and must not reach l through those that are not
    const int e = static_cast<int>(__float_as_uint(vs) >> 23 & 0xFF) - 127;
    const bool fine = e <= 126 && e >= -126;
    TileScale o;
    o.k = ks;
    o.ev = fine ? static_cast<float>(e) : vs;
    o.down = fine ? __uint_as_float(static_cast<uint32_t>(127 - e) << 23) : 1.0f;
    return o;
}

// Stores y of a row's lane share: dims 16 dt + 4g + (0..3) of d-tile dt.
template <int DT>
__device__ __forceinline__ void store_dims(const Kv8AttnArgs& a, const Kv8Request& r, int32_t head, int32_t row, int dt, const f32x4& o,
                                           float inv)
{
    const int g = (threadIdx.x & 63) >> 4, d = 16 * dt + 4 * g;
    if (d >= a.c.D) return;
    const int64_t e = (static_cast<int64_t>(r.first) + row / a.G) * a.yt + (head * a.G + row % a.G) * a.yh + d;
    const float f[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    const bool vec = reinterpret_cast<uintptr_t>(a.y) % (DT == SLHIP_F32 ? 16 : 8) == 0 && (a.yt | a.yh) % 4 == 0;
    if (vec) {
        if constexpr (DT == SLHIP_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(a.y) + e) = make_float4(f[0], f[1], f[2], f[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + e) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
    } else {
        for (int j = 0; j < 4; j++) Vec<DT>::store1(a.y, e + j, f[j]);
    }
}

// 1 / l of a row; 0 for a row that saw no key (its o is 0).
__device__ __forceinline__ float row_inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// The keys that some row of the request's rows from token `t0` to `t1` - 1 sees: [first, end), first on a tile's border.
__device__ __forceinline__ void key_range(const Kv8AttnArgs& a, int32_t past, int32_t t0, int32_t t1, int32_t& first, int32_t& end)
{
    end = past + t1;
    first = a.window > 0 ? max(past + t0 - a.window + 1, 0) & ~(kTile - 1) : 0;
}

// ---- few rows: a wave a key tile ---------------------------------------------------------------------------------

// Which requests are cut into which key ranges, from the lengths alone, so that every thread block of a launch finds its
// own without a launch before it: ranges of `chunk` tiles, the smallest multiple of four (a tile for each wave) that makes
// about a.units ranges a head of all requests together, so long requests and short ones give ranges of one size.
struct Unit {
    int32_t request;  // -1: none
    int32_t part;     // which of its ranges
    int32_t parts;    // how many
    int32_t base;     // its first slot among the partial sums (requests of one range have none)
};

__device__ __forceinline__ int32_t request_tiles(const Kv8AttnArgs& a, int32_t i)
{
    const Kv8Request r = kv8_request(a.c, i);
    const int64_t rows = static_cast<int64_t>(r.n) * a.G;
    if (r.n == 0 || rows <= a.min_rows || rows > a.max_rows) return 0;
    int32_t first, end;
    key_range(a, r.past, 0, r.n, first, end);
    return (end - first + kTile - 1) / kTile;
}

__device__ __forceinline__ int32_t ranges_of(int32_t tiles, int32_t chunk) { return (tiles + chunk - 1) / chunk; }

// Finds range `unit` of the launch's requests (FIND_REQUEST: the unit is a request, and all its ranges are asked for).
// All 256 threads of the block call it.
template <bool FIND_REQUEST>
__device__ __forceinline__ Unit find_unit(const Kv8AttnArgs& a, int32_t unit, int32_t& chunk)
{
    __shared__ int64_t s_tiles[4];
    __shared__ int32_t s_ranges[4], s_parts[4];
    __shared__ Unit s_unit;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (a.c.B + 255) / 256, i0 = min(tid * per, a.c.B), i1 = min(i0 + per, a.c.B);
    int64_t tiles = 0;
    int32_t kept = 0;  // of the thread's first request: most batches have one a thread
    for (int i = i0; i < i1; i++) {
        const int32_t n = request_tiles(a, i);
        if (i == i0) kept = n;
        tiles += n;
    }
    int64_t sum = tiles;
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) s_tiles[wave] = sum;
    if (tid == 0) s_unit.request = -1;
    __syncthreads();
    sum = s_tiles[0] + s_tiles[1] + s_tiles[2] + s_tiles[3];
    const int64_t want = (sum + a.units - 1) / a.units;
    chunk = static_cast<int32_t>((want + 3) / 4 * 4);
    if (chunk < 4) chunk = 4;
    int32_t ranges = 0, parts = 0;
    for (int i = i0; i < i1; i++) {
        const int32_t n = ranges_of(i == i0 ? kept : request_tiles(a, i), chunk);
        ranges += n;
        parts += n > 1 ? n : 0;
    }
    int32_t before = ranges, slots = parts;
    for (int o = 1; o < 64; o <<= 1) {
        const int32_t u = __shfl_up(before, o, 64), v = __shfl_up(slots, o, 64);
        if (lane >= o) {
            before += u;
            slots += v;
        }
    }
    if (lane == 63) {
        s_ranges[wave] = before;
        s_parts[wave] = slots;
    }
    __syncthreads();
    before -= ranges;
    slots -= parts;
    for (int w = 0; w < wave; w++) {
        before += s_ranges[w];
        slots += s_parts[w];
    }
    for (int i = i0; i < i1; i++) {
        const int32_t n = ranges_of(i == i0 ? kept : request_tiles(a, i), chunk);
        if (FIND_REQUEST ? i == unit : unit >= before && unit < before + n) s_unit = Unit{i, unit - before, n, slots};
        before += n;
        slots += n > 1 ? n : 0;
    }
    __syncthreads();
    return s_unit;
}

// Sums of a key range, lane by lane as the kernel holds them: [n][dt][lane] of 4 dims, then [n][row] of (m, l).
template <int DP, int NT> struct Partial {
    static constexpr int64_t kDims = static_cast<int64_t>(NT) * (DP / 16) * 64 * 4;
    static constexpr int64_t kFloats = kDims + NT * 16 * 2;
};

template <int FMT, int DP> struct WaveTile {
    uint4 k[4][DP / 64], v[DP / 16];
    float ks, vs;
    SubBlock vb;
};

// Loads a tile's codes and scales for the wave. kid, vid: the table entries of the lane's two sub-blocks.
template <int FMT, int DP>
__device__ __forceinline__ void load_tile(const Kv8AttnArgs& a, int32_t head, int32_t key, int32_t end, int32_t kid, int32_t vid,
                                          WaveTile<FMT, DP>& w)
{
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, D = a.c.D;
    const SubBlock kb = sub_block(a.c, kid, head, key + 16 * (c >> 2), end);
    w.vb = sub_block(a.c, vid, head, key + 16 * g, end);
    const uint8_t* k = a.c.k + ((kb.at << a.c.shift) + kb.sub * 16 + (c & 3)) * D;
#pragma unroll
    for (int h = 0; h < DP / 64; h++) {
        const int d = 64 * h + 16 * g < D ? 64 * h + 16 * g : 0;  // dims past D: any codes, q is 0 there
#pragma unroll
        for (int t = 0; t < 4; t++) w.k[t][h] = load_nt(k + 4 * t * D + d);
    }
    const uint8_t* v = a.c.v + ((w.vb.at << a.c.shift) + w.vb.sub * 16) * D + c * 16;
#pragma unroll
    for (int dt = 0; dt < DP / 16; dt++) w.v[dt] = load_nt(v + (16 * dt < D ? 256 * dt : 0));
    w.ks = a.c.ks[w.vb.at];
    w.vs = a.c.vs[w.vb.at];
}

template <int DT, int FMT, int DP, int NT>
__global__ __launch_bounds__(256) void kv8_attn_waves(Kv8AttnArgs a)
{
    constexpr int NP = DT == SLHIP_F32 ? 2 : 1, ND = DP / 16;
    __shared__ f32x4 s_o[2][NT * ND * 64];
    __shared__ float s_ml[4][NT * 16][2];
    const int lane = threadIdx.x & 63, wave = wave_id(), c = lane & 15, g = lane >> 4;
    const int32_t head = blockIdx.x % a.c.heads;
    int32_t chunk;
    const Unit u = find_unit<false>(a, blockIdx.x / a.c.heads, chunk);
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < a.c.B; i += 256) {
            const Kv8Request r = kv8_request(a.c, i);
            if (r.bad || (a.strict && static_cast<int64_t>(r.n) * a.G > a.max_rows)) raise_request(a.c, i, r);
        }
    }
    if (u.request < 0) return;
    const Kv8Request r = kv8_request(a.c, u.request);
    const int32_t rows = r.n * a.G;
    f16x8 q[NT][NP][DP / 64][2];
    Row row[NT];
    float m[NT], l[NT];
    f32x4 o[NT][ND];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        row[n] = load_row<DT, DP, NP>(a, r, head, 16 * n + c, 16 * n + c < rows, q[n]);
        m[n] = kNone;
        l[n] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < ND; dt++) o[n][dt] = f32x4{0, 0, 0, 0};
    }
    int32_t first, end;
    key_range(a, r.past, 0, r.n, first, end);
    const int32_t k0 = first + (u.part * chunk + wave) * kTile;
    const int32_t stop = min(static_cast<int64_t>(end), first + (static_cast<int64_t>(u.part) + 1) * chunk * kTile);
    if (k0 < stop) {
        WaveTile<FMT, DP> w;
        int32_t kid = block_id(a.c, r.table, k0 + 16 * (c >> 2), end), vid = block_id(a.c, r.table, k0 + 16 * g, end);
        load_tile<FMT, DP>(a, head, k0, end, kid, vid, w);
        kid = block_id(a.c, r.table, k0 + 4 * kTile + 16 * (c >> 2), end);
        vid = block_id(a.c, r.table, k0 + 4 * kTile + 16 * g, end);
        for (int32_t key = k0; key < stop; key += 4 * kTile) {
            WaveTile<FMT, DP> x = w;
            if (key + 4 * kTile < stop) {
                load_tile<FMT, DP>(a, head, key + 4 * kTile, end, kid, vid, w);
                kid = block_id(a.c, r.table, key + 8 * kTile + 16 * (c >> 2), end);
                vid = block_id(a.c, r.table, key + 8 * kTile + 16 * g, end);
            }
            if (x.vb.bad) raise_block(a.c, r.first, r.slot, key + 16 * g, x.vb.id);
            f32x4 S[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int t = 0; t < 4; t++) S[n][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int h = 0; h < DP / 64; h++) {
                    f16x8 k[2];
                    codes_f16<FMT>(x.k[t][h], k[0], k[1]);
#pragma unroll
                    for (int s = 0; s < 2; s++)
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int p = 0; p < NP; p++) S[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[s], q[n][p][h][s], S[n][t], 0, 0, 0);
                }
            const TileScale sc = tile_scale(a.c, x.vb, x.ks, x.vs);
            f16x8 p[NT][NP][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int k0l = key + 16 * g;
                const int hi = min(row[n].pos - k0l + 1, x.vb.keys), lo = a.window > 0 ? row[n].pos - a.window + 1 - k0l : 0;
                const bool masked = __any(hi < 16 || lo > 0);
                const float alpha = tile_softmax<NP>(a, S[n], row[n], sc, k0l, lo, hi, masked, m[n], l[n], p[n]);
                if (__any(alpha != 1.0f)) {
#pragma unroll
                    for (int dt = 0; dt < ND; dt++) o[n][dt] *= alpha;
                }
            }
            // keys that are not there have weight 0, but their codes could be NaN
            if (__any(x.vb.keys < 16)) {
#pragma unroll
                for (int dt = 0; dt < ND; dt++) x.v[dt] = first_codes(x.v[dt], x.vb.keys);
            }
#pragma unroll
            for (int dt = 0; dt < ND; dt++) {
                f16x8 v[2];
                codes_f16<FMT>(x.v[dt], v[0], v[1]);
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < NP; e++) o[n][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[s], p[n][e][s], o[n][dt], 0, 0, 0);
            }
        }
    }
    // the block's four waves: a common maximum, then the sums of waves 2 and 3 into 0 and 1, and 1 into 0
#pragma unroll
    for (int n = 0; n < NT; n++) {
        l[n] = row_sum(l[n]);
        if (g == 0) {
            s_ml[wave][16 * n + c][0] = m[n];
            s_ml[wave][16 * n + c][1] = l[n];
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; n++) {
        float top = m[n];
        for (int w = 0; w < 4; w++) top = fmaxf(top, s_ml[w][16 * n + c][0]);
        float all = 0.0f;
        for (int w = 0; w < 4; w++) all += s_ml[w][16 * n + c][1] * __builtin_amdgcn_exp2f(s_ml[w][16 * n + c][0] - top);
        const float alpha = __builtin_amdgcn_exp2f(m[n] - top);
        m[n] = top;
        l[n] = all;
#pragma unroll
        for (int dt = 0; dt < ND; dt++) o[n][dt] *= alpha;
    }
    for (int step = 2; step > 0; step >>= 1) {
        if (wave >= step && wave < 2 * step) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int dt = 0; dt < ND; dt++) s_o[wave - step][(n * ND + dt) * 64 + lane] = o[n][dt];
        }
        __syncthreads();
        if (wave < step) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int dt = 0; dt < ND; dt++) o[n][dt] += s_o[wave][(n * ND + dt) * 64 + lane];
        }
        __syncthreads();
    }
    if (wave > 0) return;
    float* part = a.part + (static_cast<int64_t>(u.base + u.part) * a.c.heads + head) * Partial<DP, NT>::kFloats;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int32_t at = 16 * n + c;
        if (u.parts == 1) {
            const float inv = row_inverse(l[n]);
            if (at < rows) {
#pragma unroll
                for (int dt = 0; dt < ND; dt++) store_dims<DT>(a, r, head, at, dt, o[n][dt], inv);
            }
        } else {
#pragma unroll
            for (int dt = 0; dt < ND; dt++) reinterpret_cast<f32x4*>(part)[(n * ND + dt) * 64 + lane] = o[n][dt];
            if (g == 0) reinterpret_cast<float2*>(part + Partial<DP, NT>::kDims)[at] = make_float2(m[n], l[n]);
        }
    }
}

// Joins the ranges of a request's head: the common maximum, then the sums relative to it, dims shared out over the waves.
template <int DT, int DP, int NT>
__global__ __launch_bounds__(256) void kv8_attn_join(Kv8AttnArgs a)
{
    constexpr int ND = DP / 16;
    const int lane = threadIdx.x & 63, wave = wave_id(), c = lane & 15;
    const int32_t head = blockIdx.x % a.c.heads;
    int32_t chunk;
    const Unit u = find_unit<true>(a, blockIdx.x / a.c.heads, chunk);
    if (u.parts <= 1) return;
    const Kv8Request r = kv8_request(a.c, u.request);
    const float* part = a.part + (static_cast<int64_t>(u.base) * a.c.heads + head) * Partial<DP, NT>::kFloats;
    const int64_t step = static_cast<int64_t>(a.c.heads) * Partial<DP, NT>::kFloats;
    for (int n = 0; n < NT; n++) {
        if (16 * n >= r.n * a.G) break;
        const float2* ml = reinterpret_cast<const float2*>(part + Partial<DP, NT>::kDims) + 16 * n + c;
        float top = kNone;
        for (int k = 0; k < u.parts; k++) top = fmaxf(top, ml[k * (step / 2)].x);
        for (int dt = wave; dt < ND; dt += 4) {
            f32x4 o = {0, 0, 0, 0};
            float l = 0.0f;
            for (int k = 0; k < u.parts; k++) {
                const float2 v = ml[k * (step / 2)];
                const float by = __builtin_amdgcn_exp2f(v.x - top);
                l = fmaf(v.y, by, l);
                const f32x4 x = reinterpret_cast<const f32x4*>(part + k * step)[(n * ND + dt) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = fmaf(x[j], by, o[j]);
            }
            if (16 * n + c < r.n * a.G) store_dims<DT>(a, r, head, 16 * n + c, dt, o, row_inverse(l));
        }
    }
}

// ---- many rows: a thread block a tile of rows -----------------------------------------------------------------------

// Four waves of NT * 16 rows each share a key tile's codes, converted to f16 once and held in LDS in the order in which
// the matrix instructions take them (a fragment is 64 lanes of 16 bytes: reads and writes without conflicts), two tiles
// deep, the next tile's codes loading meanwhile: one barrier a tile.
template <int DP> struct BlockTile {
    static constexpr int kK = 4 * (DP / 32), kV = (DP / 16) * 2;  // fragments of K: t, h, s; of V: dt, s
};

template <int DT, int FMT, int DP, int NT>
__global__ __launch_bounds__(256) void kv8_attn_blocks(Kv8AttnArgs a)
{
    constexpr int NP = DT == SLHIP_F32 ? 2 : 1, ND = DP / 16, NH = DP / 64;
    constexpr int kK = BlockTile<DP>::kK, kV = BlockTile<DP>::kV;
    extern __shared__ f16x8 s_frag[];  // [2][kK + kV][64]
    const int lane = threadIdx.x & 63, wave = wave_id(), c = lane & 15, g = lane >> 4, D = a.c.D;
    const int32_t head = blockIdx.x % a.c.heads;
    const int64_t rest = blockIdx.x / a.c.heads;
    const int32_t split = static_cast<int32_t>(rest % a.splits);
    // tiles from the last: their key ranges are the longest, and short ones fill the end
    const int64_t item = item_count(a.c.T, a.c.B, a.tile_tokens, 1) - 1 - rest / a.splits;
    const int32_t i = kv8_find(a.c, item, a.tile_tokens, 1);
    const Kv8Request r = kv8_request(a.c, i);
    const int64_t t0 = (item - item_base(a.c.starts[i], i, a.tile_tokens, 1)) * a.tile_tokens;
    if (r.bad && t0 == 0 && head == 0 && split == 0 && threadIdx.x == 0) raise_request(a.c, i, r);
    if (t0 < 0 || t0 >= r.n || static_cast<int64_t>(r.n) * a.G <= a.min_rows) return;
    if (a.strict && static_cast<int64_t>(r.n) * a.G > a.max_rows) {
        if (t0 == 0 && head == 0 && split == 0 && threadIdx.x == 0) raise_request(a.c, i, r);
        return;
    }
    const int32_t t1 = min(static_cast<int64_t>(r.n), t0 + a.tile_tokens);
    const int32_t row0 = static_cast<int32_t>(t0) * a.G, row1 = t1 * a.G;  // rows of the tile
    int32_t first, end;
    key_range(a, r.past, static_cast<int32_t>(t0), t1, first, end);
    {   // this split's part of the range
        const int32_t tiles = (end - first + kTile - 1) / kTile, each = (tiles + a.splits - 1) / a.splits;
        const int64_t from = first + static_cast<int64_t>(split) * each * kTile, to = from + static_cast<int64_t>(each) * kTile;
        first = static_cast<int32_t>(min(from, static_cast<int64_t>(end)));
        end = static_cast<int32_t>(min(to, static_cast<int64_t>(end)));
    }
    f16x8 q[NT][NP][NH][2];
    Row row[NT];
    float m[NT], l[NT];
    f32x4 o[NT][ND];
    int32_t low = 0x7FFFFFFF, high = -1;  // positions of the wave's rows
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int32_t at = row0 + (wave * NT + n) * 16 + c;
        row[n] = load_row<DT, DP, NP>(a, r, head, at, at < row1, q[n]);
        if (at < row1) {
            low = min(low, row[n].pos);
            high = max(high, row[n].pos);
        }
        m[n] = kNone;
        l[n] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < ND; dt++) o[n][dt] = f32x4{0, 0, 0, 0};
    }
    for (int x = 1; x < 16; x <<= 1) {
        low = min(low, __shfl_xor(low, x, 64));
        high = max(high, __shfl_xor(high, x, 64));
    }
    low = __builtin_amdgcn_readfirstlane(low);
    high = __builtin_amdgcn_readfirstlane(high);
    const int32_t all = r.past + r.n;  // keys of the request: codes behind them are not read as keys

    // staging: wave w loads the codes of K's product t = w and of V's dims 16 (w + 4 j)
    constexpr int VJ = ND / 4;
    uint4 ck[NH], cv[VJ];
    float ks = 0, vs = 0;
    SubBlock vb{}, vnext{};
    float ksn = 0, vsn = 0;
    const auto load = [&](int32_t key) {
        const int32_t kid = block_id(a.c, r.table, key + 16 * (c >> 2), all), vid = block_id(a.c, r.table, key + 16 * g, all);
        const SubBlock kb = sub_block(a.c, kid, head, key + 16 * (c >> 2), all);
        vnext = sub_block(a.c, vid, head, key + 16 * g, all);
        const uint8_t* k = a.c.k + ((kb.at << a.c.shift) + kb.sub * 16 + 4 * wave + (c & 3)) * D;
#pragma unroll
        for (int h = 0; h < NH; h++) ck[h] = *reinterpret_cast<const uint4*>(k + (64 * h + 16 * g < D ? 64 * h + 16 * g : 0));
        const uint8_t* v = a.c.v + ((vnext.at << a.c.shift) + vnext.sub * 16) * D + c * 16;
#pragma unroll
        for (int j = 0; j < VJ; j++) {
            const int dt = wave + 4 * j;
            cv[j] = *reinterpret_cast<const uint4*>(v + (16 * dt < D ? 256 * dt : 0));
        }
        ksn = a.c.ks[vnext.at];
        vsn = a.c.vs[vnext.at];
    };
    const auto stage = [&](int buf) {
        f16x8* f = s_frag + buf * (kK + kV) * 64 + lane;
#pragma unroll
        for (int h = 0; h < NH; h++) {
            f16x8 x, z;
            codes_f16<FMT>(ck[h], x, z);
            f[((wave * NH + h) * 2) * 64] = x;
            f[((wave * NH + h) * 2 + 1) * 64] = z;
        }
#pragma unroll
        for (int j = 0; j < VJ; j++) {
            f16x8 x, z;
            codes_f16<FMT>(vnext.keys < 16 ? first_codes(cv[j], vnext.keys) : cv[j], x, z);
            f[(kK + (wave + 4 * j) * 2) * 64] = x;
            f[(kK + (wave + 4 * j) * 2 + 1) * 64] = z;
        }
        vb = vnext;
        ks = ksn;
        vs = vsn;
    };
    int buf = 0;
    if (first < end) {
        load(first);
        stage(0);
    }
    for (int32_t key = first; key < end; key += kTile) {
        const bool more = key + kTile < end;
        const SubBlock b = vb;
        const TileScale sc = tile_scale(a.c, b, ks, vs);
        if (more) load(key + kTile);
        __syncthreads();
        if (b.bad && wave == 0) raise_block(a.c, r.first, r.slot, key + 16 * g, b.id);
        if (key <= high && (a.window <= 0 || key + kTile > low - a.window + 1)) {
            const f16x8* f = s_frag + buf * (kK + kV) * 64 + lane;
            f32x4 S[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int t = 0; t < 4; t++) S[n][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int h = 0; h < NH; h++)
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const f16x8 k = f[((t * NH + h) * 2 + s) * 64];
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int p = 0; p < NP; p++) S[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[n][p][h][s], S[n][t], 0, 0, 0);
                    }
            f16x8 p[NT][NP][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int k0l = key + 16 * g;
                const int hi = min(row[n].pos - k0l + 1, b.keys), lo = a.window > 0 ? row[n].pos - a.window + 1 - k0l : 0;
                const bool masked = __any(hi < 16 || lo > 0);
                const float alpha = tile_softmax<NP>(a, S[n], row[n], sc, k0l, lo, hi, masked, m[n], l[n], p[n]);
                if (__any(alpha != 1.0f)) {
#pragma unroll
                    for (int dt = 0; dt < ND; dt++) o[n][dt] *= alpha;
                }
            }
#pragma unroll
            for (int dt = 0; dt < ND; dt++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const f16x8 v = f[(kK + dt * 2 + s) * 64];
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < NP; e++) o[n][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[n][e][s], o[n][dt], 0, 0, 0);
                }
        }
        buf ^= 1;
        if (more) stage(buf);
    }
    float* part = a.part + blockIdx.x * Partial<DP, 4 * NT>::kFloats;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int32_t at = (wave * NT + n) * 16 + c;
        l[n] = row_sum(l[n]);
        if (a.splits == 1) {
            const float inv = row_inverse(l[n]);
            if (row0 + at < row1) {
#pragma unroll
                for (int dt = 0; dt < ND; dt++) store_dims<DT>(a, r, head, row0 + at, dt, o[n][dt], inv);
            }
        } else {
#pragma unroll
            for (int dt = 0; dt < ND; dt++) reinterpret_cast<f32x4*>(part)[((wave * NT + n) * ND + dt) * 64 + lane] = o[n][dt];
            if (g == 0) reinterpret_cast<float2*>(part + Partial<DP, 4 * NT>::kDims)[at] = make_float2(m[n], l[n]);
        }
    }
}

// Joins the splits of a row tile; a thread block joins 16 rows, dims shared out over its waves.
template <int DT, int DP, int NT>
__global__ __launch_bounds__(256) void kv8_attn_blocks_join(Kv8AttnArgs a)
{
    constexpr int ND = DP / 16;
    const int lane = threadIdx.x & 63, wave = wave_id(), c = lane & 15;
    const int32_t head = blockIdx.x % a.c.heads, n = blockIdx.y;
    const int64_t back = blockIdx.x / a.c.heads, item = item_count(a.c.T, a.c.B, a.tile_tokens, 1) - 1 - back;
    const int32_t i = kv8_find(a.c, item, a.tile_tokens, 1);
    const Kv8Request r = kv8_request(a.c, i);
    const int64_t t0 = (item - item_base(a.c.starts[i], i, a.tile_tokens, 1)) * a.tile_tokens;
    if (t0 < 0 || t0 >= r.n || static_cast<int64_t>(r.n) * a.G <= a.min_rows) return;
    if (a.strict && static_cast<int64_t>(r.n) * a.G > a.max_rows) return;
    const int32_t t1 = min(static_cast<int64_t>(r.n), t0 + a.tile_tokens);
    const int32_t row0 = static_cast<int32_t>(t0) * a.G, row1 = t1 * a.G;
    const float* part = a.part + (back * a.splits * a.c.heads + head) * Partial<DP, 4 * NT>::kFloats;
    const int64_t step = static_cast<int64_t>(a.c.heads) * Partial<DP, 4 * NT>::kFloats;
    const float2* ml = reinterpret_cast<const float2*>(part + Partial<DP, 4 * NT>::kDims) + 16 * n + c;
    if (row0 + 16 * n >= row1) return;
    float top = kNone;
    for (int k = 0; k < a.splits; k++) top = fmaxf(top, ml[k * (step / 2)].x);
    for (int dt = wave; dt < ND; dt += 4) {
        f32x4 o = {0, 0, 0, 0};
        float l = 0.0f;
        for (int k = 0; k < a.splits; k++) {
            const float2 v = ml[k * (step / 2)];
            const float by = __builtin_amdgcn_exp2f(v.x - top);
            l = fmaf(v.y, by, l);
            const f32x4 x = reinterpret_cast<const f32x4*>(part + k * step)[(n * ND + dt) * 64 + lane];
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = fmaf(x[j], by, o[j]);
        }
        if (row0 + 16 * n + c < row1) store_dims<DT>(a, r, head, row0 + 16 * n + c, dt, o, row_inverse(l));
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------

// What a call launches, from what the host knows.
struct Kv8AttnPlan {
    int32_t wave_rows;    // 0: no few-row launch, else 16 or 32
    bool blocks;          // the many-row launch
    int32_t block_rows;   // its rows a tile
    int64_t wave_grid, block_items, work_bytes;
    int32_t units, splits, tile_tokens;
};

template <int DT, int FMT> int kv8_attn_launch(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st);

template <int DT, int FMT, int DP> static int kv8_attn_run(const Kv8AttnArgs& args, const Kv8AttnPlan& p, hipStream_t st)
{
    Kv8AttnArgs a = args;
    if (p.wave_rows) {
        a.min_rows = 0;
        a.max_rows = p.blocks ? p.wave_rows : args.max_rows;
        a.strict = !p.blocks;
        a.units = p.units;
        const unsigned grid = static_cast<unsigned>(p.wave_grid), joins = static_cast<unsigned>(a.c.B) * a.c.heads;
        constexpr int NT2 = DP <= 128 ? 2 : 1;  // 32 rows (make_plan asks for them up to 128 dims)
        if (p.wave_rows == 16) kv8_attn_waves<DT, FMT, DP, 1><<<grid, 256, 0, st>>>(a);
        else kv8_attn_waves<DT, FMT, DP, NT2><<<grid, 256, 0, st>>>(a);
        const int e = check_launch("kv8_attn_waves");
        if (e) return e;
        if (p.wave_rows == 16) kv8_attn_join<DT, DP, 1><<<joins, 256, 0, st>>>(a);
        else kv8_attn_join<DT, DP, NT2><<<joins, 256, 0, st>>>(a);
        const int s = check_launch("kv8_attn_join");
        if (s) return s;
    }
    if (!p.blocks) return SLHIP_OK;
    constexpr int NT = DT == SLHIP_F32 || DP == 256 ? 1 : 2;
    a.min_rows = p.wave_rows;
    a.max_rows = args.max_rows;
    a.strict = args.strict;
    a.tile_tokens = p.tile_tokens;
    a.splits = p.splits;
    const unsigned lds = 2 * (BlockTile<DP>::kK + BlockTile<DP>::kV) * 64 * sizeof(f16x8);
    const auto kernel = kv8_attn_blocks<DT, FMT, DP, NT>;
    if (lds > 65536) SLHIP_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    kernel<<<static_cast<unsigned>(p.block_items * p.splits * a.c.heads), 256, lds, st>>>(a);
    const int s = check_launch("kv8_attn_blocks");
    if (s || p.splits == 1) return s;
    kv8_attn_blocks_join<DT, DP, NT><<<dim3(static_cast<unsigned>(p.block_items * a.c.heads), 4 * NT), 256, 0, st>>>(a);
    return check_launch("kv8_attn_blocks_join");
}

template <int DT, int FMT> int kv8_attn_by_dim(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st)
{
    if (a.c.D <= 64) return kv8_attn_run<DT, FMT, 64>(a, p, st);
    if (a.c.D <= 128) return kv8_attn_run<DT, FMT, 128>(a, p, st);
    return kv8_attn_run<DT, FMT, 256>(a, p, st);
}

}  // namespace slhip
