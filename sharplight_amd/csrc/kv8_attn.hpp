// Causal attention over the 8-bit paged cache (slhip_kv8_attention): the kernels.
//
// Mathematics. For a query row q with position p and keys j <= p (and j > p - window):
//   z_j = scale * ks_b * (q . k_j)  (capped, slopes added), ks_b and vs_b = 2^ev_b the scales of key j's block b,
//   y   = sum_j e^z_j vs_b c_j / sum_j e^z_j,  k_j and c_j the codes.
// With t_j = z_j log2(e) + ev_b and M the running maximum of t_j (or a little less: tile_max), w_j = 2^(t_j - M) holds the
// whole weight of code c_j, the block's scale included: o = sum_j w_j c_j, l = sum_j w_j 2^-ev_b, y = o / l. So V's codes go
// to the matrix cores as they are, the scale costs nothing (it rides in the addition of the exponent), and what is rounded
// to f16, w_j, is rounded relative to the largest one, whatever the scales of the blocks are (and whatever the codes: beside a key
// of zeros that has all but 2^-33 of the weight, the others' values are lost).
//
// Numbers. int8 and E4M3 codes are exact in f16. A query row is multiplied by the power of two that brings its largest
// value to [2^14, 2^15): bf16 values are then exact in f16 down to 2^-29 of the row's largest (below that they round to
// 2^-40 of it), f32 values are the sum of two f16 parts to 2^-22 (or 2^-40 of the largest). w_j goes to the matrix cores
// scaled by 2^kBias, in f16 (2^-11 of itself, or 2^-33 of the largest) for bf16 activations, whose
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

#include <type_traits>

#include "kv8.hpp"

namespace slhip {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;
constexpr float kBias = 8.0f;   // weights are 2^kBias in f16 for t_j = M
constexpr float kSlack = 7.0f;  // and at most 2^(kBias + kSlack), below f16's largest
constexpr float kExact = 0x1p20f;
constexpr int kLeastCut = 4;  // key tiles of a many-row tile that are worth a thread block of their own
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kStart = 2;

// What becomes of a score before its exponential: nothing but the scale; a cap, slopes or a scale that is not positive; or a cap
// above kFastCap, for bf16 activations in kernels of their own (f32 ones cap all scores alike).
// Up to kFastCap the scores of bf16 activations are capped by tanh y = 1 - 2 / (1 + e^(2 y)), off by up to 2^-22 whatever y is: a
// score by 2^-22 of the cap, its weight by 2^-14 of itself at most (2^-16 with a cap of 50), whose f16 part is off by 2^-11.
// It takes half of tanh_f's instructions: a prompt of 4096, 32 query heads of 64 on 8, int8 codes, 163 us, with tanh_f 249. (As a branch
// in one kernel tanh_f costs smaller caps two registers more, and with them a third wave a SIMD: 176 us.)
constexpr int kPlain = 0, kReshaped = 1, kFarCap = 2;
constexpr float kFastCap = 256.0f;

constexpr float kNone = -3.40282347e38f;  // a maximum of nothing: the least number, so that differences with -inf stay numbers

struct Kv8AttnArgs {
    Kv8Dev c;
    const void* q;
    void* y;
    int64_t qt, qh, yt, yh;
    int32_t G;                   // query heads of a K/V head
    float cap;
    float factor, most;          // of what the cap takes (scale / cap), or of the scores; its largest size in a row
    float lost;                  // what a row that is not finite is multiplied by
    int32_t window;              // 0: none
    const float* slopes;
    int32_t max_rows;              // few-row work: requests of up to so many query rows a K/V head
    bool strict;                   // requests above max_rows are an error (nothing else takes them)
    int32_t block_min, block_max;  // many-row tiles: requests of (block_min, block_max] rows; above is an error
    int32_t workers;             // few-row thread blocks
    bool direct;                 // one for each request's head, which share nothing
    int32_t tile_tokens;         // many-row tiles: tokens of a tile
    int64_t items;               // of a head
    int32_t splits, share;       // key ranges that each is cut into; or (share > 0) how many more than tiles a head has of them
    float *part, *part2;         // sums of key ranges: of workers, of tiles
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

// A sub-block of 16 keys: where its codes are in the cache, or block 0's and no keys where there is none to see.
struct SubBlock {
    uint32_t id;   // the block
    int32_t sub;   // which 16 keys of it
    int32_t keys;  // how many are below `end`
    int32_t bad;   // the table's entry is no block of the cache (it is in `entry`)
    int32_t entry;
};

// The table entry of the sub-block at `key` (another of the request's where the key is behind `end`).
__device__ __forceinline__ int32_t block_id(const Kv8Dev& c, const int32_t* table, int32_t key, int32_t end)
{
    return table[static_cast<uint32_t>(min(key, end - 1)) >> c.shift];
}

__device__ __forceinline__ SubBlock sub_block(const Kv8Dev& c, int32_t entry, int32_t key, int32_t end)
{
    SubBlock s;
    const bool here = key < end, fine = static_cast<uint32_t>(entry) < static_cast<uint32_t>(c.blocks);
    s.entry = entry;
    s.bad = here && !fine;
    s.id = here && fine ? entry : 0;
    s.sub = (key >> 4) & ((1 << (c.shift - 4)) - 1);
    s.keys = here && fine ? min(end - key, 16) : 0;
    return s;
}

// A K/V head's codes and scales of block 0, and the bytes from a block to the next.
struct HeadBase {
    const uint8_t *k, *v, *ks, *vs;
    uint32_t codes, scales;
    uint32_t slab;  // bytes of 16 keys
};

__device__ __forceinline__ HeadBase head_base(const Kv8Dev& c, int32_t head)
{
    HeadBase h;
    h.slab = 16 * c.D;
    const uint32_t codes = h.slab << (c.shift - 4);  // of a block's head: at most 2^16
    h.k = c.k + static_cast<int64_t>(head) * codes;
    h.v = c.v + static_cast<int64_t>(head) * codes;
    h.ks = reinterpret_cast<const uint8_t*>(c.ks + head);
    h.vs = reinterpret_cast<const uint8_t*>(c.vs + head);
    h.codes = c.heads * codes;
    h.scales = c.heads * 4;
    return h;
}

// Byte offset of a sub-block's codes from HeadBase::k or ::v.
__device__ __forceinline__ uint64_t codes_at(const HeadBase& h, const SubBlock& s)
{
    return static_cast<uint64_t>(s.id) * h.codes + __umul24(s.sub, h.slab);
}

// ---- rows -------------------------------------------------------------------------------------------------------

// Query row `row` (token * G + head of the group) of a request, or none.
struct Row {
    int32_t pos;
    float back;   // factor / the power of two that the row was multiplied by
    float slope;  // slopes[h] * log2(e)
};

// The lane's share of a row as it lies in memory: dims 64h + 16g + (0..15) of step h.
template <int DT, int DP> struct RawRow {
    static constexpr int kVecs = DT == SLHIP_F32 ? 4 : 2;
    uint4 w[DP / 64][kVecs];
};

template <int DT, int DP>
__device__ __forceinline__ void fetch_row(const Kv8AttnArgs& a, const Kv8Request& r, int32_t head, int32_t row, bool valid, RawRow<DT, DP>& raw)
{
    constexpr int kVecs = RawRow<DT, DP>::kVecs, per = Vec<DT>::N;
    const int g = (threadIdx.x & 63) >> 4;
    const int64_t base = (static_cast<int64_t>(r.first) + row / a.G) * a.qt + (head * a.G + row % a.G) * a.qh;
    const bool vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.qt | a.qh) % per == 0;
#pragma unroll
    for (int h = 0; h < DP / 64; h++) {
        const int d = 64 * h + 16 * g;
        const bool in = valid && d < a.c.D;
#pragma unroll
        for (int i = 0; i < kVecs; i++) {
            raw.w[h][i] = make_uint4(0, 0, 0, 0);
            const int64_t at = base + d + i * per;
            if (in && vec) {
                raw.w[h][i] = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.q) + at * Vec<DT>::BYTES);
            } else if (in) {
                float f[per];
                for (int j = 0; j < per; j++) f[j] = Vec<DT>::load1(a.q, at + j);
                raw.w[h][i] = Vec<DT>::pack(f);  // the same bits again
            }
        }
    }
}

// NP f16 parts of the row's lane share: q[p][h][s] holds dims 64h + 16g + 8s + (0..7). Dims past D are 0.
template <int DT, int DP, int NP, int SCORES>
__device__ __forceinline__ Row make_row(const Kv8AttnArgs& a, const Kv8Request& r, int32_t head, int32_t row, bool valid,
                                        const RawRow<DT, DP>& raw, f16x8 (&q)[NP][DP / 64][2])
{
    constexpr int kVecs = RawRow<DT, DP>::kVecs, per = Vec<DT>::N;
    const int32_t tok = valid ? row / a.G : 0, qh = head * a.G + (valid ? row % a.G : 0);
    float f[DP / 64][16];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < DP / 64; h++) {
#pragma unroll
        for (int i = 0; i < kVecs; i++) Vec<DT>::unpack(raw.w[h][i], &f[h][i * per]);
#pragma unroll
        for (int j = 0; j < 16; j++) top = max(top, __float_as_uint(f[h][j]) & 0x7FFFFFFFu);
    }
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
    // multiply by 2^(14 - e): biased exponents; rows that are tiny by a power that stays in range. A row that is not finite is NaN;
    // under a cap an infinity is more than the largest number (and has one f16 part).
    const bool finite = top < 0x7F800000u;
    const int e = static_cast<int>(top >> 23) - 127;
    const float power = __uint_as_float(static_cast<uint32_t>(127 + 14 - max(e, -100)) << 23);
    const float mul = finite ? power : SCORES == kPlain ? __uint_as_float(0x7FC00000u) : a.lost;
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
                    const bool two = SCORES == kPlain || finite;
                    const f16x2 lo = to_f16x2(two ? x0 - static_cast<float>(hi.x) : 0.0f, two ? x1 - static_cast<float>(hi.y) : 0.0f);
                    q[1][h][s][j] = lo.x;
                    q[1][h][s][j + 1] = lo.y;
                }
            }
    Row o;
    o.pos = r.past + tok;
    o.back = a.factor / mul;
    // Finite after a block's scale too, or a product of 0 would be no number under a cap. (Products are multiples of 2^-33, scales
    // at least 2^-40: what is not 0 is past the cap with 2^86 already.)
    if (SCORES != kPlain) o.back = __builtin_amdgcn_fmed3f(o.back, -a.most, a.most);
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

struct TileScale {
    float k;         // ks
    float ev, down;  // log2(vs), 1 / vs
};

// The softmax of one tile and row, in two steps. A lane has the row's products with its sub-block's 16 keys.
struct TileRow {
    float S[16];       // scores: weight j is 2^(S[j] * mul + shift)
    float mul, shift;
    float sum;         // of the weights so far
};

// Scores, and the row's M (m, in TileRow's terms). M need not be the maximum: it moves up to it only where the maximum is above
// it by more than kSlack, so that the sums so far are seldom multiplied (rescale; a row's maximum moves in every second tile
// of the first 64, and 32 or 64 products a tile are as many as its exponentials). lo <= j < hi are the keys that are seen.
template <int DT, int SCORES, class Rescale>
__device__ __forceinline__ void tile_max(const Kv8AttnArgs& a, const f32x4 (&products)[4], const Row& row, const TileScale& sc, int32_t key0,
                                         int lo, int hi, bool masked, float& m, TileRow& t, const Rescale& rescale)
{
    // t = fma(S, mul, add) with mul > 0, so the largest S is the largest t. Capped or sloped scores, and those of a scale that
    // is not positive, are turned into t themselves.
    float (&S)[16] = t.S;
    float mul = fmaxf(row.back * sc.k * kLog2e, 1.17549435e-38f), add = sc.ev;  // (a masked S is -inf: not times 0)
#pragma unroll
    for (int j = 0; j < 16; j++) S[j] = products[j >> 2][j & 3];
    if constexpr (SCORES != kPlain) {
        if (a.cap > 0.0f) {
            const float in = row.back * sc.k, out = a.cap * kLog2e;
            if constexpr (DT == SLHIP_F32 || SCORES == kFarCap) {
#pragma unroll
                for (int j = 0; j < 16; j++) S[j] = fmaf(tanh_f(S[j] * in), out, add);
            } else {
                const float twice = in * (2.0f * kLog2e), both = out + add;
#pragma unroll
                for (int j = 0; j < 16; j++)
                    S[j] = fmaf(__builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(S[j] * twice)), -2.0f * out, both);
            }
        } else {
            mul = row.back * sc.k * kLog2e;
#pragma unroll
            for (int j = 0; j < 16; j++) S[j] = fmaf(S[j], mul, add);
        }
        if (a.slopes) {
            const float far = row.slope * static_cast<float>(key0 - row.pos);
#pragma unroll
            for (int j = 0; j < 16; j++) S[j] += fmaf(row.slope, static_cast<float>(j), far);
        }
        mul = 1.0f;
        add = 0.0f;
    }
    if (masked) {
#pragma unroll
        for (int j = 0; j < 16; j++) S[j] = j < hi ? S[j] : -INFINITY;
        if (__any(lo > 0)) {  // at a window's border only
#pragma unroll
            for (int j = 0; j < 16; j++) S[j] = j >= lo ? S[j] : -INFINITY;
        }
        if (hi <= max(lo, 0)) {  // none is seen: the block's scales, which may be no numbers, do not count
            mul = 1.0f;
            add = 0.0f;
        }
    }
    float mx = S[0];
#pragma unroll
    for (int j = 1; j < 15; j += 2) mx = fmaxf(fmaxf(mx, S[j]), S[j + 1]);
    mx = fmaxf(mx, S[15]);
    const float top = row_max(fmaf(mx, mul, add));
    const bool up = top - m > kSlack;
    if (__any(up)) {
        const float to = up ? top : m;
        rescale(__builtin_amdgcn_exp2f(m - to));
        m = to;
    }
    t.mul = mul;
    t.shift = add - (m - kBias);
    t.sum = 0.0f;
    if (__any(fabsf(m) > kExact)) {  // the roundings of S * mul + shift could add up to a weight past f16: t first, then t - M
#pragma unroll
        for (int j = 0; j < 16; j++) S[j] = fmaf(S[j], mul, add) - m;
        t.mul = 1.0f;
        t.shift = kBias;
    }
}

// Weights 8 s + j and 8 s + j + 1 (j even), into P's parts.
template <int NP> __device__ __forceinline__ void tile_weights(TileRow& t, int s, int j, f16x8 (&p)[NP][2])
{
    const float w0 = __builtin_amdgcn_exp2f(fmaf(t.S[8 * s + j], t.mul, t.shift));
    const float w1 = __builtin_amdgcn_exp2f(fmaf(t.S[8 * s + j + 1], t.mul, t.shift));
    t.sum += w0 + w1;  // not of the f16 parts: l weighs them by 1 / vs, and a block of tiny values has no f16 weights left
    const f16x2 hi = to_f16x2(w0, w1);
    p[0][s][j] = hi.x;
    p[0][s][j + 1] = hi.y;
    if constexpr (NP == 2) {  // (as fused multiply-adds, which take the f16 part as it is)
        const f16x2 lo = to_f16x2(fmaf(-static_cast<float>(hi.x), 1.0f, w0), fmaf(-static_cast<float>(hi.y), 1.0f, w1));
        p[1][s][j] = lo.x;
        p[1][s][j + 1] = lo.y;
    }
}

__device__ __forceinline__ TileScale tile_scale(float ks, float vs)
{
    // a scale that is NaN makes the weights of the keys that are seen NaN, and must not reach l through those that are not
    const int e = static_cast<int>(__float_as_uint(vs) >> 23 & 0xFF) - 127;
    const bool fine = e <= 126;
    TileScale o;
    o.k = ks;
    o.ev = fine && ks == ks ? static_cast<float>(e) : __uint_as_float(0x7FC00000u);
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

// How heads come to thread blocks: kShared, by the line below (or directly, where the launch holds many-row tiles too); kDirect,
// a thread block a head, with nothing carried from one to the next, which takes 60 registers less; kLean, that with K's and V's
// codes in the same registers one after the other, for three waves a SIMD (two of 256 dims or 32 rows): many short contexts are all
// latency, of which the waves hide each other's. (Of f32 and 256 dims, or 32 rows of 128 with reshaped scores, 4 to 20 registers
// go to scratch for that.) Times by kShared, kDirect and kLean, 8 K/V heads of 128, a row each: one
// request of 501 tokens 9.4, 7.7 and 8.5 us; 256 of up to 251 33, 28 and 24 us; 400 of up to 701 81, 74 and 67 us. 100 of up to
// 401, 4 heads of 256: 30 us shared, 17 lean.
constexpr int kShared = 0, kDirect = 1, kLean = 2;

// Every wave takes key tiles of its own, with all of a K/V head's rows: codes go from memory into registers and from there to
// the matrix cores, nothing through LDS, and no wave waits for another before a head's end. HBM bounds it, and the latency
// of a head's beginning (lengths, table, codes) and end (the four waves' join). Measured, 8 K/V heads of 128: 64 sequences of
// 1 to 4095 tokens, bf16 and E4M3, 61 us with the join (264 MB, 4.3 TB/s); 2 of up to 131000, f32 and int8, 66 us (337 MB,
// 5.1 TB/s). Of 4 heads of 256, whose codes leave registers for one wave a SIMD: 16 windows of 4096 tokens 31 us (2.9 TB/s).

// The work of all requests of a launch, in rounds of four key tiles (one for each wave of a thread block), is one line --
// request by request, head by head -- that `workers` thread blocks share out in equal pieces, whatever the lengths are. A
// piece that begins or ends inside a head's keys leaves partial sums, of which a worker has two at most: of the head that it
// goes on with in slot 2 w, of one that it begins in slot 2 w + 1. Where a piece lies follows from the lengths alone, so every
// worker finds its own without a launch before it, and the join finds the workers of a head by a division.
// Beginning a head costs as much as kStart rounds (query and table loads, the join of the four waves), which stand on the
// line before its rounds: without them the workers of short requests end last (64 sequences of 1 to 4095 tokens: 78
// us, with them 68).
struct Line {
    int64_t each;     // steps of a worker
    int64_t total;    // steps of all
    int64_t before;   // steps of a head of the requests before `request`
    int32_t request;  // the request looked for
    int32_t steps;    // its steps a head: kStart and its rounds (0: it is not the launch's)
    Kv8Request r;
};

// Quotients of numbers that fit 32 bits in all but the longest batches.
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d)
{
    if (((n | d) >> 32) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
    return n / d;
}

__device__ __forceinline__ int32_t request_steps(const Kv8AttnArgs& a, const Kv8Request& r)
{
    const int64_t rows = static_cast<int64_t>(r.n) * a.G;
    if (r.n == 0 || rows > a.max_rows) return 0;
    int32_t first, end;
    key_range(a, r.past, 0, r.n, first, end);
    return (end - first + 4 * kTile - 1) / (4 * kTile) + kStart;
}

constexpr int kMaxGroups = 65536 / 64;  // of 64 requests

// The line, and on it the request of worker `at` (of request `at` itself if BY_REQUEST). The requests are taken in groups of
// 64, a lane each; the waves of the thread block share out the groups' sums, and each then looks again at the one group that
// holds the request. Wave-uniform; all 256 threads call it.
template <bool BY_REQUEST> __device__ __forceinline__ Line find_line(const Kv8AttnArgs& a, int32_t at)
{
    __shared__ int32_t s_group[kMaxGroups];
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int32_t groups = (a.c.B + 63) / 64;
    Line f{0, 0, 0, -1, 0, {}};
    Kv8Request mine{};         // the lane's request in the group looked at
    int32_t kept = 0, up = 0;  // its steps, and their inclusive sum
    const auto look = [&](int32_t group) {
        const int32_t i = group * 64 + lane;
        mine = kv8_request(a.c, i < a.c.B ? i : 0);
        kept = i < a.c.B ? request_steps(a, mine) : 0;
        up = wave_scan(kept);
    };
    int32_t group = 0;
    int64_t sum = 0, before = 0;  // steps of all requests, of those before the group
    if (groups == 1) {
        look(0);
        sum = __builtin_amdgcn_readlane(up, 63);
    } else {
        for (int32_t j = wave; j < groups; j += 4) {
            look(j);
            if (lane == 63) s_group[j] = up;
        }
        __syncthreads();
        for (int32_t j = 0; j < groups; j += 64) sum += __builtin_amdgcn_readlane(wave_scan(j + lane < groups ? s_group[j + lane] : 0), 63);
    }
    f.total = sum * a.c.heads;
    f.each = quotient(f.total + a.workers - 1, a.workers);
    if (f.each < 1) f.each = 1;
    if (!BY_REQUEST && at * f.each >= f.total) return f;
    // requests that end before the piece begins, in whole groups and then in the group
    const auto under = [&](int64_t end) { return end * a.c.heads <= at * f.each; };
    if (groups > 1) {
        for (int32_t j = 0; j < groups; j += 64) {
            const int32_t g = wave_scan(j + lane < groups ? s_group[j + lane] : 0);
            const int32_t k = BY_REQUEST ? at / 64 - j : __popcll(__ballot(j + lane < groups && under(before + g)));
            if (k < 64) {
                group = j + k;
                if (k > 0) before += __builtin_amdgcn_readlane(g, k - 1);
                break;
            }
            before += __builtin_amdgcn_readlane(g, 63);
        }
        look(group);
    }
    const int k = BY_REQUEST ? at & 63 : __popcll(__ballot(under(before + up)));  // below 64: the piece begins in the group
    f.request = group * 64 + k;
    f.steps = __builtin_amdgcn_readlane(kept, k);
    f.before = before + __builtin_amdgcn_readlane(up, k) - f.steps;
    f.r.first = __builtin_amdgcn_readlane(mine.first, k);
    f.r.n = __builtin_amdgcn_readlane(mine.n, k);
    f.r.past = __builtin_amdgcn_readlane(mine.past, k);
    f.r.slot = __builtin_amdgcn_readlane(mine.slot, k);
    f.r.bad = f.r.n == 0;
    f.r.table = a.c.pages + (f.r.bad ? 0 : f.r.slot * a.c.bps);
    return f;
}

// Sums of a key range, lane by lane as the kernels hold them: [n][dt][lane] of 4 dims, then [n][row] of (m, l).
template <int DP, int NT> struct Partial {
    static constexpr int64_t kDims = static_cast<int64_t>(NT) * (DP / 16) * 64 * 4;
    static constexpr int64_t kFloats = kDims + NT * 16 * 2;
};

template <int DP, int NT> constexpr int waves_lds() { return (2 * NT * (DP / 16) * 64 * 4 + 4 * NT * 16 * 2) * 4; }

template <int DT, int FMT, int DP, int NT, int DIRECT, int SCORES>
__device__ __forceinline__ void attn_waves(const Kv8AttnArgs& a, const int32_t worker, char* lds)
{
    constexpr int NP = DT == SLHIP_F32 ? 2 : 1, ND = DP / 16, NH = DP / 64;
    f32x4* s_o = reinterpret_cast<f32x4*>(lds);                                       // [2][NT * ND * 64]
    float2* s_ml = reinterpret_cast<float2*>(lds + 2 * NT * ND * 64 * sizeof(f32x4));  // [4][NT * 16]
    const int lane = threadIdx.x & 63, wave = wave_id(), c = lane & 15, g = lane >> 4, D = a.c.D;
    if (worker == a.workers - 1) {  // (of a shared line, the one with the least to do)
        for (int i = threadIdx.x; i < a.c.B; i += 256) {
            const Kv8Request r = kv8_request(a.c, i);
            if (r.bad || (a.strict && static_cast<int64_t>(r.n) * a.G > a.max_rows)) raise_request(a.c, i, r);
        }
    }

    // A head's share of the piece, and what its loads go by.
    struct Segment {
        const int32_t* table;
        int32_t row0, n, past, slot;  // of the request
        int32_t i, steps, head;
        int32_t end, k0, last;  // the request's keys; the wave's first tile; where its tiles end
        int32_t whole, goes_on;
        __device__ __forceinline__ void take(const Kv8Request& r) { table = r.table; row0 = r.first; n = r.n; past = r.past; slot = r.slot; }
        __device__ __forceinline__ Kv8Request request() const { return {row0, n, past, slot, false, table}; }
    } cur, next;
    int64_t pos = 0, stop;  // on the line
    int32_t step = 0;
    if (DIRECT != kShared || a.direct) {
        cur.i = worker / a.c.heads;
        cur.head = worker - cur.i * a.c.heads;
        const Kv8Request r = kv8_request(a.c, cur.i);
        cur.take(r);
        cur.steps = request_steps(a, r);
        stop = cur.steps;
    } else {
        const Line line = find_line<false>(a, worker);
        if (line.request < 0) return;
        pos = worker * line.each;
        stop = min(pos + line.each, line.total);
        cur.i = line.request;
        cur.take(line.r);
        cur.steps = line.steps;
        const int64_t in = pos - line.before * a.c.heads;
        cur.head = static_cast<int32_t>(quotient(in, cur.steps));
        step = static_cast<int32_t>(in - static_cast<int64_t>(cur.head) * cur.steps);
    }
    if (cur.steps == 0) return;
    const int64_t begin = pos;
    // The share of the head that cur points at from `step` on; false if the piece ends before its rounds.
    const auto share = [&](Segment& s) __attribute__((always_inline)) {
        const int32_t until = static_cast<int32_t>(min(static_cast<int64_t>(s.steps), step + (stop - pos)));
        s.goes_on = pos == begin && step >= kStart;
        pos += until - step;
        const int32_t from = max(step - kStart, 0), count = until - kStart - from;
        if (count <= 0) return false;
        int32_t first;
        key_range(a, s.past, 0, s.n, first, s.end);
        s.k0 = first + (from * 4 + wave) * kTile;
        s.last = static_cast<int32_t>(min(static_cast<int64_t>(s.end), first + (static_cast<int64_t>(from) + count) * 4 * kTile));
        s.whole = count == s.steps - kStart;
        return true;
    };
    const auto advance = [&](Segment& s) __attribute__((always_inline)) {  // to the next head on the line, while the piece lasts
        step = 0;
        for (;;) {
            if (pos >= stop) return false;
            if (++s.head == a.c.heads) {
                s.head = 0;
                do {
                    const Kv8Request r = kv8_request(a.c, ++s.i);  // there is one: steps are left on the line
                    s.take(r);
                    s.steps = request_steps(a, r);
                } while (s.steps == 0);
            }
            if (share(s)) return true;
        }
    };
    if (!share(cur) && !advance(cur)) return;

    constexpr bool LEAN = DIRECT == kLean;
    constexpr bool kEarly = DT != SLHIP_F32 && DP <= 128;  // (f32 queries and 256 dims leave no registers for that)
    // K's codes are loaded again as soon as the first product has used them, V's after the second: each then has the other
    // product and the softmax to arrive in, and the codes need registers once. The next head's first tile and queries are on
    // their way while the four waves join this one's sums.
    RawRow<DT, DP> raw[NT];
    uint4 k[4][NH], v[ND];
    float ks, vs;
    const uint8_t* vp;
    SubBlock vb;
    int32_t kid, vid;
    const auto look = [&](const Segment& s, int32_t key) __attribute__((always_inline)) {
        kid = block_id(a.c, s.table, key + 16 * (c >> 2), s.end);
        vid = block_id(a.c, s.table, key + 16 * g, s.end);
    };
    const auto aim = [&](const Segment& s, int32_t key) __attribute__((always_inline)) {  // K's codes and the scales of the tile at `key`; where V's codes are
        const HeadBase base = head_base(a.c, s.head);
        const SubBlock kb = sub_block(a.c, kid, key + 16 * (c >> 2), s.end);
        vb = sub_block(a.c, vid, key + 16 * g, s.end);
        const uint8_t* kp = base.k + codes_at(base, kb) + (c & 3) * D;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int h = 0; h < NH; h++)  // dims past D: any codes, q is 0 there
                k[t][h] = *reinterpret_cast<const uint4*>(kp + 4 * t * D + (64 * h + 16 * g < D ? 64 * h + 16 * g : 0));
        const uint64_t at = static_cast<uint64_t>(vb.id) * base.scales;
        ks = *reinterpret_cast<const float*>(base.ks + at);
        vs = *reinterpret_cast<const float*>(base.vs + at);
        vp = base.v + codes_at(base, vb) + c * 16;
        look(s, key + 4 * kTile);
    };
    const auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int dt = 0; dt < ND; dt++) v[dt] = load_nt(vp + (16 * dt < D ? 256 * dt : 0));
    };
    // Queries first (they are used first), then the first tile, if the wave has one.
    const auto open = [&](const Segment& s) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NT; n++) fetch_row<DT, DP>(a, s.request(), s.head, 16 * n + c, 16 * n + c < s.n * a.G, raw[n]);
        if (s.k0 < s.last) {
            aim(s, s.k0);
            if (!LEAN) load_v();
        }
    };
    look(cur, min(cur.k0, cur.end - 1));
    open(cur);
    for (;;) {
        const Kv8Request r = cur.request();
        const int32_t rows = r.n * a.G, head = cur.head;
        next = cur;
        const bool another = DIRECT == kShared && advance(next);
        f16x8 q[NT][NP][NH][2];
        Row row[NT];
        float m[NT], l[NT];
        f32x4 o[NT][ND];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            row[n] = make_row<DT, DP, NP, SCORES>(a, r, head, 16 * n + c, 16 * n + c < rows, raw[n], q[n]);
            m[n] = kNone;
            l[n] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < ND; dt++) o[n][dt] = f32x4{0, 0, 0, 0};
        }
        // One tile; `more`: the next one is loaded meanwhile. (Without a branch: where the paths of one meet, the compiler would
        // wait for what was loaded on either.)
        const auto tile = [&](int32_t key, auto more) __attribute__((always_inline)) {
            f32x4 S[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int t = 0; t < 4; t++) S[n][t] = f32x4{0, 0, 0, 0};
            // two 16-key products (and two dim tiles below) take turns, so that none waits for its own last product
#pragma unroll
            for (int t = 0; t < 4; t += 2)
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    f16x8 x[2][2];
                    codes_f16<FMT>(k[t][h], x[0][0], x[0][1]);
                    codes_f16<FMT>(k[t + 1][h], x[1][0], x[1][1]);
#pragma unroll
                    for (int s = 0; s < 2; s++)
#pragma unroll
                        for (int e = 0; e < NP; e++)
#pragma unroll
                            for (int u = 0; u < 2; u++)
#pragma unroll
                                for (int n = 0; n < NT; n++) S[n][t + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[u][s], q[n][e][h][s], S[n][t + u], 0, 0, 0);
                }
            TileScale sc = tile_scale(ks, vs);
            const int32_t keys = vb.keys;
            if (vb.bad) raise_block(a.c, r.first, r.slot, key + 16 * g, vb.entry);
            if constexpr (LEAN) {
                __builtin_amdgcn_sched_barrier(0);
                load_v();
                __builtin_amdgcn_sched_barrier(0);
            } else if constexpr (more) {
                // scales in registers of their own, or the next ones' arrival is waited for to move them
                asm volatile("" : "+v"(sc.k), "+v"(sc.ev), "+v"(sc.down));
                __builtin_amdgcn_sched_barrier(0);
                aim(cur, key + 4 * kTile);
                __builtin_amdgcn_sched_barrier(0);
            }
            f16x8 p[NT][NP][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int k0l = key + 16 * g;
                const int hi = min(row[n].pos - k0l + 1, keys), lo = a.window > 0 ? row[n].pos - a.window + 1 - k0l : 0;
                const bool masked = __any(hi < 16 || lo > 0);
                TileRow t;
                tile_max<DT, SCORES>(a, S[n], row[n], sc, k0l, lo, hi, masked, m[n], t, [&](float alpha) __attribute__((always_inline)) {
                    l[n] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < ND; dt++) o[n][dt] *= alpha;
                });
#pragma unroll
                for (int j = 0; j < 16; j += 2) tile_weights<NP>(t, j >> 3, j & 7, p[n]);
                l[n] = fmaf(t.sum, sc.down, l[n]);
            }
            // keys that are not there have weight 0, but their codes could be NaN
            if (__any(keys < 16)) {
#pragma unroll
                for (int dt = 0; dt < ND; dt++) v[dt] = first_codes(v[dt], keys);
            }
#pragma unroll
            for (int dt = 0; dt < ND; dt += 2) {
                f16x8 x[2][2];
                codes_f16<FMT>(v[dt], x[0][0], x[0][1]);
                codes_f16<FMT>(v[dt + 1], x[1][0], x[1][1]);
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int e = 0; e < NP; e++)
#pragma unroll
                        for (int u = 0; u < 2; u++)
#pragma unroll
                            for (int n = 0; n < NT; n++) o[n][dt + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[u][s], p[n][e][s], o[n][dt + u], 0, 0, 0);
            }
            if constexpr (more) {
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (LEAN) aim(cur, key + 4 * kTile);
                else load_v();
            }
        };
        if (cur.k0 < cur.last) {
            int32_t key = cur.k0;
            for (; key + 4 * kTile < cur.last; key += 4 * kTile) tile(key, std::true_type{});
            tile(key, std::false_type{});
        }
        if (another) {
            look(next, min(next.k0, next.end - 1));
            if (kEarly) open(next);
        }
        __builtin_amdgcn_sched_barrier(0);
        // the four waves: a common maximum, then the sums of waves 2 and 3 into 0 and 1, and 1 into 0
#pragma unroll
        for (int n = 0; n < NT; n++) {
            l[n] = row_sum(l[n]);
            if (g == 0) s_ml[wave * NT * 16 + 16 * n + c] = make_float2(m[n], l[n]);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float top = m[n];
            for (int w = 0; w < 4; w++) top = fmaxf(top, s_ml[w * NT * 16 + 16 * n + c].x);
            float all = 0.0f;
            for (int w = 0; w < 4; w++) {
                const float2 x = s_ml[w * NT * 16 + 16 * n + c];
                all += x.y * __builtin_amdgcn_exp2f(x.x - top);
            }
            const float alpha = __builtin_amdgcn_exp2f(m[n] - top);
            m[n] = top;
            l[n] = all;
#pragma unroll
            for (int dt = 0; dt < ND; dt++) o[n][dt] *= alpha;
        }
        for (int half = 2; half > 0; half >>= 1) {
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int dt = 0; dt < ND; dt++) s_o[((wave - half) * NT * ND + n * ND + dt) * 64 + lane] = o[n][dt];
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int dt = 0; dt < ND; dt++) o[n][dt] += s_o[(wave * NT * ND + n * ND + dt) * 64 + lane];
            }
            __syncthreads();
        }
        if (wave == 0) {
            float* part = a.part + (2 * static_cast<int64_t>(worker) + (cur.goes_on ? 0 : 1)) * Partial<DP, NT>::kFloats;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int32_t at = 16 * n + c;
                if (cur.whole) {
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
        if (!another) return;
        if (!kEarly) open(next);
        cur = next;
    }
}

// ---- joins ----------------------------------------------------------------------------------------------------------

// Joins `count` partial sums of 16 rows, the k-th at at(k): four at a time, relative to the largest maximum so far. The
// thread block's waves share out the dims, or (BY_PART) the sums of d-tile dt0, which they then join through LDS.
// put(dt, o, l) gets what the wave has of d-tile dt.
template <int DP, int NT, bool BY_PART, class At, class Put>
__device__ __forceinline__ void join_rows(const At& at, int32_t count, int n, int dt0, const Put& put)
{
    constexpr int ND = DP / 16;
    const int lane = threadIdx.x & 63, wave = wave_id(), c = lane & 15;
    for (int dt = BY_PART ? dt0 : wave; dt < (BY_PART ? dt0 + 1 : ND); dt += 4) {
        f32x4 o = {0, 0, 0, 0};
        float l = 0.0f, top = kNone;
        for (int32_t k = BY_PART ? wave : 0; k < count; k += BY_PART ? 16 : 4) {
            float2 ml[4];
            f32x4 x[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int32_t j = k + u * (BY_PART ? 4 : 1);
                const float* p = at(min(j, count - 1));
                ml[u] = reinterpret_cast<const float2*>(p + Partial<DP, NT>::kDims)[16 * n + c];
                x[u] = reinterpret_cast<const f32x4*>(p)[(n * ND + dt) * 64 + lane];
                if (j >= count) ml[u].x = -INFINITY;  // the last one again, with no weight
            }
            const float was = top;
#pragma unroll
            for (int u = 0; u < 4; u++) top = fmaxf(top, ml[u].x);
            const float alpha = __builtin_amdgcn_exp2f(was - top);
            l *= alpha;
            o *= alpha;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float by = __builtin_amdgcn_exp2f(ml[u].x - top);
                l = fmaf(ml[u].y, by, l);
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = fmaf(x[u][j], by, o[j]);
            }
        }
        if constexpr (BY_PART) {
            __shared__ f32x4 s_o[4][64];
            __shared__ float2 s_ml[4][64];
            s_o[wave][lane] = o;
            s_ml[wave][lane] = make_float2(top, l);
            __syncthreads();
            if (wave > 0) return;
            for (int w = 1; w < 4; w++) top = fmaxf(top, s_ml[w][lane].x);
            o = f32x4{0, 0, 0, 0};
            l = 0.0f;
            for (int w = 0; w < 4; w++) {
                const float by = __builtin_amdgcn_exp2f(s_ml[w][lane].x - top);
                l = fmaf(s_ml[w][lane].y, by, l);
                o += s_o[w][lane] * by;
            }
        }
        put(dt, o, l);
    }
}

// The sums of a request's head over the workers that share it. index: (request, head, n[, dt]).
template <int DT, int DP, int NT, bool BY_PART>
__device__ __forceinline__ void join_waves(const Kv8AttnArgs& a, int64_t index)
{
    constexpr int ND = DP / 16;
    const int dt0 = BY_PART ? static_cast<int>(index % ND) : 0;
    if (BY_PART) index /= ND;
    const int n = static_cast<int>(index % NT);
    index /= NT;
    const int32_t head = static_cast<int32_t>(index % a.c.heads);
    const Line f = find_line<true>(a, static_cast<int32_t>(index / a.c.heads));
    if (f.steps == 0) return;
    const int64_t from = f.before * a.c.heads + static_cast<int64_t>(head) * f.steps + kStart;  // its first round
    const int64_t w0 = quotient(from, f.each), w1 = quotient(from + f.steps - kStart - 1, f.each);
    const Kv8Request& r = f.r;
    const int32_t row = 16 * n + (threadIdx.x & 15);
    if (w0 == w1 || 16 * n >= r.n * a.G) return;
    const int64_t slot0 = 2 * w0 + (w0 * f.each < from ? 1 : 0);
    const auto at = [&](int32_t k) { return a.part + (k == 0 ? slot0 : 2 * (w0 + k)) * Partial<DP, NT>::kFloats; };
    join_rows<DP, NT, BY_PART>(at, static_cast<int32_t>(w1 - w0 + 1), n, dt0, [&](int dt, const f32x4& o, float l) {
        if (row < r.n * a.G) store_dims<DT>(a, r, head, row, dt, o, row_inverse(l));
    });
}

// A key range of a row tile: number `split` of the `cuts` that the tile is cut into; their sums are parts first + 0 .. of the
// head. cuts = 0: there is none.
struct Cut {
    Kv8Request r;
    int32_t tile, split, cuts;
    int64_t first;
};

// The row tiles of a request that is of the many-row work.
__device__ __forceinline__ int32_t request_tiles(const Kv8AttnArgs& a, const Kv8Request& r)
{
    const int64_t rows = static_cast<int64_t>(r.n) * a.G;
    return rows <= a.block_min || rows > a.block_max ? 0 : (r.n + a.tile_tokens - 1) / a.tile_tokens;
}

// Range `index` of a head, or the first one of row tile `index` (BY_TILE). Tiles that fill the machine are not cut; of up to 64
// requests, whose lengths a wave has at once, those with longer contexts are cut into more ranges (all tiles of a request into
// as many as its last), so that `share` ranges besides the tiles are about as long as each other; of more requests all
// tiles are cut alike. Whole row tiles come from the last: their key ranges are the longest, and short ones fill the end.
// Wave-uniform.
template <bool BY_TILE> __device__ __forceinline__ Cut find_cut(const Kv8AttnArgs& a, int64_t index, bool raise)
{
    Cut f{};
    if (a.share == 0) {
        const int64_t back = BY_TILE ? index : index / a.splits;
        const Kv8Item it = kv8_find(a.c, a.items - 1 - back, a.tile_tokens, 1);
        if (raise && (threadIdx.x & 63) == 0 && it.piece == 0 && (it.r.bad || static_cast<int64_t>(it.r.n) * a.G > a.block_max)) raise_request(a.c, it.i, it.r);
        if (it.piece < 0 || it.piece >= request_tiles(a, it.r)) return f;
        f.r = it.r;
        f.tile = static_cast<int32_t>(it.piece);
        f.first = back * a.splits;
        f.split = BY_TILE ? 0 : static_cast<int32_t>(index - f.first);
        f.cuts = a.splits;
        return f;
    }
    const int lane = threadIdx.x & 63, i = min(lane, a.c.B - 1);
    const Kv8Request mine = kv8_request(a.c, i);
    const int32_t tiles = lane < a.c.B ? request_tiles(a, mine) : 0;
    if (raise && index == 0 && lane < a.c.B && (mine.bad || static_cast<int64_t>(mine.n) * a.G > a.block_max)) raise_request(a.c, i, mine);
    int32_t first, end;
    key_range(a, mine.past, (tiles - 1) * a.tile_tokens, mine.n, first, end);
    const int32_t length = (end - first + kTile - 1) / kTile;
    const int32_t all = __builtin_amdgcn_readlane(wave_scan(tiles * length), 63), each = max((all + a.share - 1) / a.share, kLeastCut);
    const int32_t cuts = (length + each - 1) / each, up = wave_scan(tiles * cuts);
    const int k = BY_TILE ? max(__popcll(__ballot(lane < a.c.B && item_base(a.c.starts[i], i, a.tile_tokens, 1) <= index)) - 1, 0)
                          : __popcll(__ballot(up <= index));
    if (k >= a.c.B) return f;
    const int32_t t = __builtin_amdgcn_readlane(tiles, k), cut = __builtin_amdgcn_readlane(cuts, k);
    const int64_t from = __builtin_amdgcn_readlane(up, k) - static_cast<int64_t>(t) * cut;
    const int64_t piece = BY_TILE ? index - item_base(__builtin_amdgcn_readlane(mine.first, k), k, a.tile_tokens, 1) : quotient(index - from, max(cut, 1));
    if (piece < 0 || piece >= t || from < 0 || from + static_cast<int64_t>(t) * cut > a.items + a.share) return f;
    f.r.first = __builtin_amdgcn_readlane(mine.first, k);
    f.r.n = __builtin_amdgcn_readlane(mine.n, k);
    f.r.past = __builtin_amdgcn_readlane(mine.past, k);
    f.r.slot = __builtin_amdgcn_readlane(mine.slot, k);
    f.r.bad = false;
    f.r.table = a.c.pages + f.r.slot * a.c.bps;
    f.tile = static_cast<int32_t>(piece);
    f.first = from + piece * cut;
    f.split = BY_TILE ? 0 : static_cast<int32_t>(index - f.first);
    f.cuts = cut;
    return f;
}

// The sums of a row tile over its key ranges. index: (tile, head, n).
template <int DT, int DP, int NT> __device__ __forceinline__ void join_blocks(const Kv8AttnArgs& a, int64_t index)
{
    const int n = static_cast<int>(index % NT);
    index /= NT;
    const int32_t head = static_cast<int32_t>(index % a.c.heads);
    const Cut f = find_cut<true>(a, index / a.c.heads, false);
    if (f.cuts < 2) return;
    const Kv8Request& r = f.r;
    const int32_t row0 = f.tile * a.tile_tokens * a.G, row1 = min(r.n, (f.tile + 1) * a.tile_tokens) * a.G;
    if (row0 + 16 * n >= row1) return;
    const int32_t row = row0 + 16 * n + (threadIdx.x & 15);
    const auto at = [&](int32_t k) { return a.part2 + ((f.first + k) * a.c.heads + head) * Partial<DP, NT>::kFloats; };
    join_rows<DP, NT, false>(at, f.cuts, n, 0, [&](int dt, const f32x4& o, float l) {
        if (row < row1) store_dims<DT>(a, r, head, row, dt, o, row_inverse(l));
    });
}

// ---- many rows: a thread block a tile of rows -----------------------------------------------------------------------

// Four waves of NT * 16 rows each share a key tile's codes, converted to f16 once and held in LDS in the order in which
// the matrix instructions take them (a fragment is 64 lanes of 16 bytes: reads and writes without conflicts), two tiles
// deep, the next tile's codes loading meanwhile: one barrier a tile. The vector unit (exponentials, f16 conversions) bounds
// it next to the matrix cores. Measured: a prompt of 8192, 32 query heads of 128 on 8, bf16 and E4M3, 557 us (990 TFLOP/s of
// the 1310 that a large bf16 product reaches) at 2.25 GHz, 612 us at the 2.05 that the clock falls to under a long load;
// vector unit 66% and matrix cores 42% of the cycles.
// Of 256 dims the tiles take most of a CU's LDS; there one thread block has eight waves, for two on each SIMD. (A prompt of
// 4096, 16 query heads of 256 on 4, bf16: 276 us with four waves, 170 with eight; 150 of 30 to 574, 16 on 8, f32: 1048 and 757.)
constexpr int block_waves(int dp) { return dp == 256 ? 8 : 4; }

template <int DP> struct BlockTile {
    static constexpr int kK = 4 * (DP / 32), kV = (DP / 16) * 2;  // fragments of K: t, h, s; of V: dt, s
};

template <int DP> constexpr int blocks_lds() { return 2 * (BlockTile<DP>::kK + BlockTile<DP>::kV) * 64 * static_cast<int>(sizeof(f16x8)); }

template <int DT, int FMT, int DP, int NT, int SCORES>
__device__ __forceinline__ void attn_blocks(const Kv8AttnArgs& a, const int64_t index, char* lds)
{
    constexpr int NP = DT == SLHIP_F32 ? 2 : 1, ND = DP / 16, NH = DP / 64;
    constexpr int kK = BlockTile<DP>::kK, kV = BlockTile<DP>::kV, W = block_waves(DP);
    f16x8* s_frag = reinterpret_cast<f16x8*>(lds);  // [2][kK + kV][64]
    const int lane = threadIdx.x & 63, wave = wave_id(), c = lane & 15, g = lane >> 4, D = a.c.D;
    const int32_t head = static_cast<int32_t>(index % a.c.heads);
    const Cut cut = find_cut<false>(a, index / a.c.heads, head == 0 && wave == 0);
    if (cut.cuts == 0) return;
    const Kv8Request& r = cut.r;
    const int32_t t0 = cut.tile * a.tile_tokens, t1 = min(r.n, t0 + a.tile_tokens);
    const int32_t row0 = t0 * a.G, row1 = t1 * a.G;  // rows of the tile
    int32_t first, end;
    key_range(a, r.past, t0, t1, first, end);
    {   // this part of the range
        const int32_t tiles = (end - first + kTile - 1) / kTile, each = (tiles + cut.cuts - 1) / cut.cuts;
        const int64_t from = first + static_cast<int64_t>(cut.split) * each * kTile, to = from + static_cast<int64_t>(each) * kTile;
        first = static_cast<int32_t>(min(from, static_cast<int64_t>(end)));
        end = static_cast<int32_t>(min(to, static_cast<int64_t>(end)));
    }
    RawRow<DT, DP> raw[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int32_t at = row0 + (wave * NT + n) * 16 + c;
        fetch_row<DT, DP>(a, r, head, at, at < row1, raw[n]);
    }
    const int32_t all = r.past + r.n;  // keys of the request: codes behind them are not read as keys

    // Staging: wave w takes codes of K's product t = w % 4 (of eight waves, half its dims) and of V's dims 16 (w + W j). Table entries are a tile ahead of
    // the codes that they lead to, codes are loaded two tiles ahead of the products that take them and converted one tile
    // ahead. Past the range's last tile that one is loaded again.
    constexpr int KJ = 4 * NH / W, VJ = ND / W;
    const int h0 = (wave >> 2) * KJ;
    uint4 ck[KJ], cv[VJ];
    SubBlock next;
    float ksn, vsn;
    int32_t kid, vid;
    const HeadBase base = head_base(a.c, head);
    // the lane's first codes in a sub-block (dims past D: any codes, q is 0 there and the sums are not stored)
    const uint8_t* const kbase = base.k + (4 * (wave & 3) + (c & 3)) * D + (16 * g < D ? 16 * g : 0);
    const uint8_t* const vbase = base.v + (16 * wave < D ? 256 * wave : 0) + c * 16;
    const int32_t border = max(first + ((end - first - 1) & ~(kTile - 1)), 0);  // the last tile
    const auto look = [&](int32_t key) __attribute__((always_inline)) {
        key = min(key, border);
        kid = block_id(a.c, r.table, key + 16 * (c >> 2), all);
        vid = block_id(a.c, r.table, key + 16 * g, all);
    };
    const auto load = [&](int32_t key) __attribute__((always_inline)) {
        const int32_t at = min(key, border);
        const SubBlock kb = sub_block(a.c, kid, at + 16 * (c >> 2), all);
        next = sub_block(a.c, vid, at + 16 * g, all);
        const uint8_t* k = kbase + codes_at(base, kb);
#pragma unroll
        for (int h = 0; h < KJ; h++) ck[h] = *reinterpret_cast<const uint4*>(k + (64 * (h0 + h) + 16 * g < D ? 64 * (h0 + h) : 0));
        const uint8_t* v = vbase + codes_at(base, next);
#pragma unroll
        for (int j = 0; j < VJ; j++) cv[j] = *reinterpret_cast<const uint4*>(v + (16 * (wave + W * j) < D ? 256 * W * j : 0));
        const uint64_t scales = static_cast<uint64_t>(next.id) * base.scales;
        ksn = *reinterpret_cast<const float*>(base.ks + scales);
        vsn = *reinterpret_cast<const float*>(base.vs + scales);
        look(key + kTile);
    };
    const auto clip = [&]() __attribute__((always_inline)) {  // V's codes of keys that are not there
        if (__any(next.keys < 16)) {
#pragma unroll
            for (int j = 0; j < VJ; j++) cv[j] = first_codes(cv[j], next.keys);
        }
    };
    const auto stage = [&](f16x8* f, int i) __attribute__((always_inline)) {  // load i of the KJ + VJ
        f16x8 x, z;
        const int at = i < KJ ? ((wave & 3) * NH + h0 + i) * 2 : kK + (wave + W * (i - KJ)) * 2;
        codes_f16<FMT>(i < KJ ? ck[i < KJ ? i : 0] : cv[i < KJ ? 0 : i - KJ], x, z);
        f[at * 64] = x;
        f[(at + 1) * 64] = z;
    };
    // The first codes are on their way while the queries become f16 parts. (A range of no tiles loads others of the request.)
    look(first);
    load(first);
    __builtin_amdgcn_sched_barrier(0);
    f16x8 q[NT][NP][NH][2];
    Row row[NT];
    float m[NT], l[NT];
    f32x4 o[NT][ND];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int32_t at = row0 + (wave * NT + n) * 16 + c;
        row[n] = make_row<DT, DP, NP, SCORES>(a, r, head, at, at < row1, raw[n], q[n]);
        m[n] = kNone;
        l[n] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < ND; dt++) o[n][dt] = f32x4{0, 0, 0, 0};
    }
    if (first < end) {
        const auto scales = [&](int32_t key) __attribute__((always_inline)) {
            TileScale sc = tile_scale(ksn, vsn);
            // in registers of their own, or the next scales' arrival is waited for to move them
            asm volatile("" : "+v"(sc.k), "+v"(sc.ev), "+v"(sc.down));
            if (next.bad && wave == 0) raise_block(a.c, r.first, r.slot, min(key, border) + 16 * g, next.entry);
            return sc;
        };
        clip();
#pragma unroll
        for (int i = 0; i < KJ + VJ; i++) stage(s_frag + lane, i);
        TileScale sc = scales(first);
        int32_t keys = next.keys;
        load(first + kTile);
        int buf = 0;
        for (int32_t key = first; key < end; key += kTile, buf ^= 1) {
            const f16x8* f = s_frag + buf * (kK + kV) * 64 + lane;
            f16x8* g2 = s_frag + (buf ^ 1) * (kK + kV) * 64 + lane;
            clip();
            __syncthreads();
            // Matrix and vector instructions are put in turns by hand: a wave issues in order, and while one product runs,
            // a few conversions (of the next tile) or exponentials (of the second half of the keys) fit in its shadow.
            // Fragments are read four ahead of their products, of two 16-key products (of all dim tiles) in turns, so that no
            // sum waits for its own last product.
            f32x4 S[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int t = 0; t < 4; t++) S[n][t] = f32x4{0, 0, 0, 0};
            constexpr int R = 5;  // fragments held: the one in use and four on their way
            f16x8 ring[R];
            const auto fetch = [&](int i) __attribute__((always_inline)) {  // K's [t pair][h][s][t], then V's [s][dt]
                const int j = i / 4, v = i - kK;
                const int at = i < kK ? ((2 * (j / NH) + (i & 1)) * NH + j % NH) * 2 + ((i >> 1) & 1) : kK + v % ND * 2 + v / ND;
                ring[i % R] = f[at * 64];
            };
#pragma unroll
            for (int i = 0; i < R - 1; i++) fetch(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kK; i++) {
                const int j = i / 4, t = 2 * (j / NH) + (i & 1), s = (i >> 1) & 1;
                if (i + R - 1 < kK) fetch(i + R - 1);
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int n = 0; n < NT; n++) S[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[i % R], q[n][p][j % NH][s], S[n][t], 0, 0, 0);
                if (i % (kK / (KJ + VJ)) == 0 && i / (kK / (KJ + VJ)) < KJ + VJ) stage(g2, i / (kK / (KJ + VJ)));
                __builtin_amdgcn_sched_barrier(0);
            }
            const TileScale sn = scales(key + kTile);
            const int32_t keys_next = next.keys;
            __builtin_amdgcn_sched_barrier(0);
            load(key + 2 * kTile);
            __builtin_amdgcn_sched_barrier(0);
            TileRow t[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int k0l = key + 16 * g;
                const int hi = min(row[n].pos - k0l + 1, keys), lo = a.window > 0 ? row[n].pos - a.window + 1 - k0l : 0;
                const bool masked = __any(hi < 16 || lo > 0);
                tile_max<DT, SCORES>(a, S[n], row[n], sc, k0l, lo, hi, masked, m[n], t[n], [&](float alpha) __attribute__((always_inline)) {
                    l[n] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < ND; dt++) o[n][dt] *= alpha;
                });
            }
            f16x8 p[NT][NP][2];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < R - 1; i++) fetch(kK + i);
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 8; j += 2) tile_weights<NP>(t[n], 0, j, p[n]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kV; i++) {
                const int s = i / ND, dt = i % ND;
                if (i + R - 1 < kV) fetch(kK + i + R - 1);
#pragma unroll
                for (int e = 0; e < NP; e++)
#pragma unroll
                    for (int n = 0; n < NT; n++) o[n][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[(kK + i) % R], p[n][e][s], o[n][dt], 0, 0, 0);
                // the other half's weights, 4 NT pairs over the turns of the first half
#pragma unroll
                for (int w = 0; w < 4 * NT; w++)
                    if (s == 0 && w * ND / (4 * NT) == dt) tile_weights<NP>(t[w % NT], 1, 2 * (w / NT), p[w % NT]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int n = 0; n < NT; n++) l[n] = fmaf(t[n].sum, sc.down, l[n]);
            sc = sn;
            keys = keys_next;
        }
    }
    float* part = a.part2 + ((cut.first + cut.split) * a.c.heads + head) * Partial<DP, W * NT>::kFloats;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int32_t at = (wave * NT + n) * 16 + c;
        l[n] = row_sum(l[n]);
        if (cut.cuts == 1) {
            const float inv = row_inverse(l[n]);
            if (row0 + at < row1) {
#pragma unroll
                for (int dt = 0; dt < ND; dt++) store_dims<DT>(a, r, head, row0 + at, dt, o[n][dt], inv);
            }
        } else {
#pragma unroll
            for (int dt = 0; dt < ND; dt++) reinterpret_cast<f32x4*>(part)[((wave * NT + n) * ND + dt) * 64 + lane] = o[n][dt];
            if (g == 0) reinterpret_cast<float2*>(part + Partial<DP, W * NT>::kDims)[at] = make_float2(m[n], l[n]);
        }
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------

// Matrix tiles of 16 rows that a wave of a many-row tile works on: two where two waves a SIMD find registers for them.
constexpr int block_tiles(bool f32, int dp) { return dp == 256 || (f32 && dp == 128) ? 1 : 2; }

// What a call launches, from what the host knows.
struct Kv8AttnPlan {
    int32_t wave_tiles;  // few-row launch: 0 none, else matrix tiles of 16 rows (1, 2)
    bool blocks;         // many-row tiles
    bool by_part;        // the few-row join shares out the sums of a head, not its dims
    bool few_heads;      // of direct work: all have a place at once
};

constexpr int block_threads(int dp, int nb) { return nb > 0 ? 64 * block_waves(dp) : 256; }

// Thread blocks of the many-row tiles, then of the few-row work: one launch, so that neither waits for the other's end.
template <int DT, int FMT, int DP, int NT, int NB, int DIRECT, int SCORES>
__global__ __launch_bounds__(block_threads(DP, NB), DIRECT == kShared && (NB == 0 && DP == 256 || NT == 2) ? 1 : 2) void kv8_attn(Kv8AttnArgs a)
{
    extern __shared__ __align__(16) char lds[];
    if constexpr (NT > 0 && NB > 0) {
        const unsigned blocks = gridDim.x - a.workers;
        if (blockIdx.x < blocks) attn_blocks<DT, FMT, DP, NB, SCORES>(a, blockIdx.x, lds);
        else attn_waves<DT, FMT, DP, NT, kShared, SCORES>(a, blockIdx.x - blocks, lds);
    } else if constexpr (NT > 0) {
        attn_waves<DT, FMT, DP, NT, DIRECT, SCORES>(a, blockIdx.x, lds);
    } else {
        attn_blocks<DT, FMT, DP, NB, SCORES>(a, blockIdx.x, lds);
    }
}

template <int DT, int DP, int NT, int NB, bool BY_PART>
__global__ __launch_bounds__(256) void kv8_attn_join(Kv8AttnArgs a, int64_t wave_joins)
{
    if (blockIdx.x < wave_joins) join_waves<DT, DP, NT, BY_PART>(a, blockIdx.x);
    else join_blocks<DT, DP, block_waves(DP) * NB>(a, blockIdx.x - wave_joins);
}

template <int DT, int FMT, int SCORES> int kv8_attn_launch(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st);

template <int DT, int FMT, int DP, int NT, int NB, int SCORES, int DIRECT = kShared>
static int kv8_attn_start(const Kv8AttnArgs& a, hipStream_t st)
{
    constexpr int waves = NT > 0 ? waves_lds<DP, NT ? NT : 1>() : 0, blocks = NB > 0 ? blocks_lds<DP>() : 0, lds = waves > blocks ? waves : blocks;
    const auto kernel = kv8_attn<DT, FMT, DP, NT, NB, DIRECT, SCORES>;
    if (lds > 65536) SLHIP_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    const int64_t grid = (NT > 0 ? a.workers : 0) + (NB > 0 ? (a.share ? a.items + a.share : a.items * a.splits) * a.c.heads : 0);
    kernel<<<static_cast<unsigned>(grid), block_threads(DP, NB), lds, st>>>(a);
    return check_launch("kv8_attn");
}

template <int DT, int FMT, int DP, int SCORES> static int kv8_attn_run(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st)
{
    constexpr int NB = block_tiles(DT == SLHIP_F32, DP), NT2 = DP <= 128 ? 2 : 1;  // make_plan asks for two up to 128 dims
    constexpr int kOne = DP <= 128 ? kDirect : kLean;
    int e = SLHIP_OK;
    if constexpr (DP <= 128) {
        if (p.blocks && p.wave_tiles) e = kv8_attn_start<DT, FMT, DP, 1, NB, SCORES>(a, st);
    }
    const bool both = DP <= 128 && p.blocks && p.wave_tiles;  // (of 256 dims the two want different thread blocks: two launches)
    if (p.blocks && !both) e = kv8_attn_start<DT, FMT, DP, 0, NB, SCORES>(a, st);
    if (e) return e;
    if (p.wave_tiles && !both) {
        if (p.wave_tiles == 2) e = a.direct ? kv8_attn_start<DT, FMT, DP, NT2, 0, SCORES, kLean>(a, st) : kv8_attn_start<DT, FMT, DP, NT2, 0, SCORES>(a, st);
        else if (!a.direct) e = kv8_attn_start<DT, FMT, DP, 1, 0, SCORES>(a, st);
        else e = p.few_heads ? kv8_attn_start<DT, FMT, DP, 1, 0, SCORES, kOne>(a, st) : kv8_attn_start<DT, FMT, DP, 1, 0, SCORES, kLean>(a, st);
    }
    if (e) return e;
    const int64_t waves = p.wave_tiles && !a.direct ? static_cast<int64_t>(a.c.B) * a.c.heads * p.wave_tiles * (p.by_part ? DP / 16 : 1) : 0;
    const int64_t blocks = p.blocks && (a.share || a.splits > 1) ? a.items * a.c.heads * block_waves(DP) * NB : 0;
    if (waves + blocks == 0) return SLHIP_OK;
    const unsigned grid = static_cast<unsigned>(waves + blocks);
    if (p.wave_tiles == 2) {
        if (p.by_part) kv8_attn_join<DT, DP, NT2, NB, true><<<grid, 256, 0, st>>>(a, waves);
        else kv8_attn_join<DT, DP, NT2, NB, false><<<grid, 256, 0, st>>>(a, waves);
    } else {
        if (p.by_part) kv8_attn_join<DT, DP, 1, NB, true><<<grid, 256, 0, st>>>(a, waves);
        else kv8_attn_join<DT, DP, 1, NB, false><<<grid, 256, 0, st>>>(a, waves);
    }
    return check_launch("kv8_attn_join");
}

template <int DT, int FMT, int SCORES> int kv8_attn_by_dim(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st)
{
    if (a.c.D <= 64) return kv8_attn_run<DT, FMT, 64, SCORES>(a, p, st);
    if (a.c.D <= 128) return kv8_attn_run<DT, FMT, 128, SCORES>(a, p, st);
    return kv8_attn_run<DT, FMT, 256, SCORES>(a, p, st);
}

}  // namespace slhip
