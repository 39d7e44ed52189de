// Verification of drafted tokens, and the draw of the next one (slhip_draft_verify).
//
// Mathematics. Row t of the target's logits z: p(v) = e^((z_v - M) / tau) / S, S = sum_v e^((z_v - M) / tau), M = max z; q the same
// of the draft's logits. Draft x is accepted while u q(x) < p(x). What is drawn behind the accepted ones has the weights
// max(p - q, 0) of the refused draft's row, or p of the last row: the first v whose inclusive sum is above w times the sum of all.
//
// Every row's S is needed for its p(x), so the rows are read once for their sums (HBM bounds it), in chunks that lie in
// registers: a wave's maximum first, then one exponential a logit, no running rescale. Which row is drawn from follows from all
// of a request's sums. The sums of p's chunks are there already; those of max(p - q, 0) take that one row of both a second time. The
// place in a chunk takes it once more.
//
// Numbers. A choice changes where a sum passes a random number. An acceptance has one such border, p(x): f32 exponentials (of arguments with one rounding:
// log2(e) / tau in two parts, or all terms of a sum would be off the same way), 16 of them added in f32 and the rest in f64, move it by some 2^-24, and are what rows
// that are compared with draft logits have. A draw has as many borders as there are tokens, so that one of them lies within 2^-26 of the random number in one
// draw of some thousands (sums of f32 exponentials gave another token than f64's in 2e-4 to 3e-4 of the draws from 50257 to 151936 tokens): all that is drawn by is of f64
// exponentials to 2^-39. Those are the sums of the rows that may be drawn from as they are (a request's last one, and all without draft logits), and what is made of
// the one row behind a refused draft.
//
// Measured: the sums of 257 rows of 151936 f32 logits and of 193 draft rows (273 MB) 47.0 us, 5.8 TB/s (with f32 exponentials alone 45.6), in bf16 (137 MB) 34.2, of
// which the vector unit works 91%; of 256 rows of 50257 bf16 logits (25.7 MB) 15.7 us (f32 11.4; without any 9.8: the loads, all on their way at once, do not hide the
// exponentials, and two chunks a thread block, the second one loaded behind the first, take 17.4), of 64 rows 7.0. What follows is a latency: 256 draws 7.7 us in one
// launch (choose), 64 7.2, 16 requests' looked-up drafts 7.1; 64 requests with draft logits 5.6 (decide), 13.7 (2432 chunks of p and q, 78 MB out of the last-level
// cache; bf16 13.0) and 6.8 (pick; bf16 7.9); one request with drafts 6.6 (38 chunks that decide for themselves) and 5.4.
#include <math.h>

#include "step.hpp"

namespace slhip {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kDrawThreads = 1024, kDrawWaves = 16;  // of what follows the rows' sums: few thread blocks, so a latency
constexpr int kChunkVecs = 1024;                     // 16-byte vectors of a chunk: 16 KB
constexpr int kTerms = 16;                           // powers that are added in f32
constexpr int64_t kMaxVocab = 1 << 24;
template <int DT> constexpr int kChunk = kChunkVecs * Vec<DT>::N;  // logits of a chunk

struct ChunkStat {
    float m;      // the largest logit; NaN where the chunk holds a NaN or an infinity above
    int32_t arg;  // its first place (rows of greedy requests)
    double s;     // sum of e^((z - m) / tau), without the row's draft where that was chosen
};

// What is drawn for a request, and from what.
enum : int32_t { kDone = 0, kFromTarget = 1, kFromRest = 2, kFromOthers = 3 };  // nothing; p; max(p - q, 0); p without the draft
struct Pick {
    int32_t kind, row, place, token;  // the row, its place in the request, its draft
    double mp, cp, sum, mq, cq, ratio;  // maxima, log2(e) / tau, the sum of p's powers, that sum / q's
    double own;                       // the draft's power of p
    int32_t held;                     // where its chunks' shares are held in LDS (-1: nowhere)
    int32_t exact;                    // its sums of all rows are the ones to draw by
};

// A chunk of the drawn row, where drafts were drawn: sums of its powers of p and of q, of p - ratio q where that is above 0, and of q there.
struct ChunkSums {
    double p, q, rest, above;
};

struct DraftArgs {
    const void *target, *draft;
    int64_t zs, qs;  // row strides
    int64_t T;
    int32_t B, V, chunks;
    const int32_t *starts, *ids;
    const float *tau, *tau_q, *accept, *sample;
    int32_t *out, *n_out;
    int64_t out_stride;
    const int32_t* past;
    int32_t *kept, *dropped;
    float* logp;
    ChunkStat* stats;  // [T][2][chunks]
    Pick* picks;       // [B]
    ChunkSums* sums;   // [B][chunks]
    uint32_t* err;
};

struct Heat {
    float tau;     // 1 for greedy requests
    bool greedy, bad;
};

__device__ __forceinline__ Heat heat_of(const float* tau, int32_t i)
{
    const float t = tau ? tau[i] : 1.0f;
    Heat h;
    h.greedy = t <= 0.0f;
    h.bad = t != t;
    h.tau = h.greedy || h.bad ? 1.0f : fminf(fmaxf(t, 0x1p-40f), 0x1p40f);
    return h;
}

// A thread's logits of a chunk: vectors of 16 bytes, a block's TH threads side by side, in the order of the vocabulary from one step
// to the next. Places past the vocabulary are -inf.
template <int DT, int TH> struct Logits {
    static constexpr int N = Vec<DT>::N, kVecs = kChunkVecs / TH, kEach = kVecs * N;
    uint4 w[kVecs];
    __device__ static __forceinline__ int32_t place(int32_t chunk, int j) { return chunk * kChunk<DT> + (j * TH + static_cast<int>(threadIdx.x)) * N; }
    __device__ __forceinline__ void load(const void* rows, int64_t row, int64_t stride, int32_t V, int32_t chunk)
    {
        const char* p = static_cast<const char*>(rows) + row * stride * Vec<DT>::BYTES;
        if ((chunk + 1) * kChunk<DT> <= V) {  // whole: no branch between the loads
#pragma unroll
            for (int j = 0; j < kVecs; j++) w[j] = load_any(p + static_cast<int64_t>(place(chunk, j)) * Vec<DT>::BYTES);
            return;
        }
#pragma unroll
        for (int j = 0; j < kVecs; j++) {
            const int32_t v = place(chunk, j);
            if (v + N <= V) {
                w[j] = load_any(p + static_cast<int64_t>(v) * Vec<DT>::BYTES);
            } else {
                float z[N];
                for (int k = 0; k < N; k++) z[k] = v + k < V ? Vec<DT>::load1(p, v + k) : -INFINITY;
                w[j] = Vec<DT>::pack(z);  // the same bits again
            }
        }
    }
};

// v of another lane by a DPP move, 0 where there is none.
template <int CTRL, int ROWS = 0xF> __device__ __forceinline__ double dpp64(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ __forceinline__ double lane64(double v, int lane)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Over 16 lanes, in every lane (swaps in quads, then mirrors: group_sum).
__device__ __forceinline__ double row_sum64(double v)
{
    v += dpp64<0xB1>(v);
    v += dpp64<0x4E>(v);
    v += dpp64<0x141>(v);
    return v + dpp64<0x140>(v);
}

// Over the wave, wave-uniform.
__device__ __forceinline__ double wave_sum64(double v)
{
    v = row_sum64(v);
    return (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
}

// Inclusive sums over the wave (wave_scan's steps).
__device__ __forceinline__ double wave_scan64(double v)
{
    v += dpp64<0x111>(v);
    v += dpp64<0x112>(v);
    v += dpp64<0x114>(v);
    v += dpp64<0x118>(v);
    v += dpp64<0x142, 0xA>(v);
    return v + dpp64<0x143, 0xC>(v);
}

// Of lanes that are alike in l & 3, in every one of them.
__device__ __forceinline__ double sum_by_four(double v)
{
    v += dpp64<0x124>(v);  // a row's quads: it turned by 4 and by 8
    v += dpp64<0x128>(v);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// Four sums over the wave together, number l & 3 in lane l: each step over lanes also halves what a lane holds.
__device__ __forceinline__ double wave_sums64(const double (&s)[4])
{
    const int lane = threadIdx.x & 63;
    const bool odd = lane & 1, high = lane & 2;
    const double a = (odd ? s[1] : s[0]) + dpp64<0xB1>(odd ? s[0] : s[1]), b = (odd ? s[3] : s[2]) + dpp64<0xB1>(odd ? s[2] : s[3]);
    return sum_by_four((high ? b : a) + dpp64<0x4E>(high ? a : b));
}

constexpr double kLog2e64 = 1.44269504088896340736;

// e^((z - m) / tau) = 2^((z - m) c) of z <= m, to 2^-39 of itself, and not below 2^-1000. 2^f, |f| <= 1/2, is the polynomial of degree 8 that is 1 at 0 and whose
// largest relative error is least (2^-39.7; found by exchange of that error's extrema).
constexpr int kTogether = 4;
constexpr double kNone = 0x1p-999;  // 2^-1000, of a rounded factor
struct Power {
    double m, c, least;
    __device__ __forceinline__ Power(double m_, double c_) : m(m_), c(c_), least(-1000.0f * __builtin_amdgcn_rcpf(static_cast<float>(c_))) {}
    // Of K logits step by step together (a step waits for the one before), as 2^f and the power of two that it is to be multiplied with.
    template <int K> __device__ __forceinline__ void parts(const float* z, double (&w)[K], double (&scale)[K]) const
    {
        // what is added to it is rounded to a whole number, in the lower bits: here with an exponent's bias
        constexpr double kWhole = 0x1.8p52 + 1023;
        constexpr double kTerm[] = {0x1.66348837ae4fdp-20, 0x1.00ee071f2a659p-16, 0x1.4306c115fa167p-13, 0x1.5d872975bfeabp-10, 0x1.3b2ab7f3b35e4p-7,
                                    0x1.c6b08defc2653p-5, 0x1.ebfbdff7c5a77p-3, 0x1.62e42fef7a78bp-1, 1.0};
        double d[K];
#pragma unroll
        for (int e = 0; e < K; e++) d[e] = fmax(z[e] - m, least);
#pragma unroll
        for (int e = 0; e < K; e++) {
            const double n = fma(d[e], c, kWhole);
            d[e] = fma(d[e], c, kWhole - n);
            scale[e] = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, n) << 52);
            w[e] = kTerm[0];
        }
#pragma unroll
        for (int t = 1; t < 9; t++)
#pragma unroll
            for (int e = 0; e < K; e++) w[e] = fma(w[e], d[e], kTerm[t]);
    }
    template <int K> __device__ __forceinline__ void of(const float* z, double (&w)[K]) const
    {
        double scale[K];
        parts(z, w, scale);
#pragma unroll
        for (int e = 0; e < K; e++) w[e] *= scale[e];
    }
    __device__ __forceinline__ double at(float z) const
    {
        double w[1];
        of(&z, w);
        return w[0];
    }
    // `to` and the power.
    __device__ __forceinline__ double add(float z, double to) const
    {
        double w[1], scale[1];
        parts(&z, w, scale);
        return fma(w[0], scale[0], to);
    }
    // 0 for all that is as small, -inf among it.
    __device__ __forceinline__ double or_none(float z) const
    {
        const double v = at(z);
        return v > kNone ? v : 0.0;
    }
};

// The same in f32: to (2 + |log2 e|) 2^-23 of itself, 0 below 2^-126. log2(e) / tau is taken as two parts, the second one positive: -inf times it is -inf. (An element
// takes 8 issue slots so, in f64 18.)
struct PowerF32 {
    float m, hi, lo;
    __device__ __forceinline__ PowerF32(float m_, double c) : m(m_)
    {
        const float near = static_cast<float>(c);
        hi = near > c ? __uint_as_float(__float_as_uint(near) - 1) : near;
        lo = fmaxf(static_cast<float>(c - hi), 0x1p-100f);  // (c is above 2^-40)
    }
    __device__ __forceinline__ float at(float z) const { return __builtin_amdgcn_exp2f(fmaf(z - m, hi, (z - m) * lo)); }
};

// ---- the sums of all rows ------------------------------------------------------------------------------------------

template <int DT, bool DRAFT> __global__ __launch_bounds__(kThreads) void draft_stats(DraftArgs a)
{
    __shared__ float s_m[kWaves];
    __shared__ double s_s[kWaves];
    __shared__ int32_t s_arg[kWaves];
    typedef Logits<DT, kThreads> Mine;
    constexpr int N = Mine::N, kVecs = Mine::kVecs, kMats = DRAFT ? 2 : 1;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int64_t item = blockIdx.x, t = item / (a.chunks * kMats);
    const int32_t rest = static_cast<int32_t>(item - t * (a.chunks * kMats)), mat = rest / a.chunks, chunk = rest - mat * a.chunks;
    Mine x;
    if (mat == 0) x.load(a.target, t, a.zs, a.V, chunk);
    if (t >= a.starts[a.B]) return;
    const int32_t i = row_request(a.starts, a.B, t);
    const Heat target = heat_of(a.tau, i), h = mat == 0 || !a.tau_q ? target : heat_of(a.tau_q, i);
    if (mat == 1) {  // not of greedy requests, nor of the row that has no draft
        if (target.greedy || h.greedy || t + 1 >= a.starts[i + 1]) return;
        x.load(a.draft, t, a.qs, a.V, chunk);
    }
    // Where drafts are chosen, the chunk that holds the row's is summed without it. Those rows and requests' last ones may be drawn from by these sums.
    const bool last = t + 1 >= a.starts[i + 1], chosen = !DRAFT || (a.tau_q && a.tau_q[i] <= 0.0f);
    const int32_t drafted = mat == 0 && !target.greedy && !last && chosen && t + 1 < a.T ? a.ids[t + 1] : -1;
    const bool holds = drafted >= 0 && drafted < a.V && drafted / kChunk<DT> == chunk, exact = mat == 0 && !target.greedy && (last || chosen);
    float z[Mine::kEach];
#pragma unroll
    for (int j = 0; j < kVecs; j++) Vec<DT>::unpack(x.w[j], &z[j * N]);
    float m = z[0];
#pragma unroll
    for (int j = 1; j < kVecs * N; j++) m = __builtin_elementwise_maximum(m, z[j]);  // a NaN stays
    const bool bad = !(m < INFINITY);
    m = group_max<64>(m);
    if (__any(bad)) m = INFINITY;
    if (holds) {
#pragma unroll
        for (int j = 0; j < kVecs * N; j++) z[j] = Mine::place(chunk, j / N) + j % N == drafted ? -INFINITY : z[j];
    }
    const double c = kLog2e64 / h.tau;
    double sum = 0.0;
    if (!exact) {
        const PowerF32 power(m, c);
        float s[kVecs * N / kTerms] = {};
#pragma unroll
        for (int j = 0; j < kVecs * N; j++) s[j / kTerms] += power.at(z[j]);
#pragma unroll
        for (int j = 0; j < kVecs * N / kTerms; j++) sum += s[j];
    } else {
        const Power power(m, c);
#pragma unroll
        for (int j = 0; j < kVecs * N; j++) sum = power.add(z[j], sum);
    }
    sum = wave_sum64(sum);
    int32_t arg = 0x7FFFFFFF;
    if (target.greedy) {
#pragma unroll
        for (int j = kVecs * N - 1; j >= 0; j--)
            if (z[j] == m) arg = Mine::place(chunk, j / N) + j % N;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) arg = min(arg, __shfl_xor(arg, o, 64));
    }
    if (lane == 0) {
        s_m[wave] = m;
        s_s[wave] = sum;
        s_arg[wave] = arg;
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // each wave's sum is of its own maximum; a lane each
        const float mine = lane < kWaves ? s_m[lane] : -INFINITY;
        m = group_max_dpp<16>(mine);
        double v = mine > -INFINITY ? s_s[lane & (kWaves - 1)] * Power(m, c).at(mine) : 0.0;
        v += dpp64<0xB1>(v);
        v += dpp64<0x4E>(v);
        arg = 0x7FFFFFFF;
        for (int w = 0; w < kWaves; w++)
            if (s_m[w] == m) arg = min(arg, s_arg[w]);
        if (lane == 0) a.stats[(t * 2 + mat) * a.chunks + chunk] = ChunkStat{m == INFINITY ? NAN : m, arg, v};
    }
}

// ---- what is accepted ----------------------------------------------------------------------------------------------

// A row of a matrix: its maximum, its sum and 1 / sum, the lowest place of the maximum, whether it can be used; and its draft's logit and share.
struct RowStat {
    double m, s, inv, share;  // (share: of its draft)
    int32_t arg;
    bool fine;
    float z;
};

constexpr int kHeld = 4;  // chunks of a lane that it looks at once: a vocabulary of 262144

// The chunks of a row together, by 16 lanes. arg: its first place is wanted; shares: of the first 64 chunks, in units of the row's sum before its division.
__device__ __forceinline__ RowStat row_stat(const ChunkStat* st, int32_t chunks, double c, bool arg, double* shares)
{
    const int lane = threadIdx.x & 15;
    ChunkStat x[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; j++) {
        x[j] = st[min(lane + 16 * j, chunks - 1)];
        if (lane + 16 * j >= chunks) x[j].m = -INFINITY;
    }
    float m = -INFINITY;
    bool bad = false;
    const auto look = [&](float v) {
        bad |= v != v;
        m = fmaxf(m, v);
    };
#pragma unroll
    for (int j = 0; j < kHeld; j++) look(x[j].m);
    for (int32_t k = lane + 16 * kHeld; k < chunks; k += 16) look(st[k].m);
    m = group_max_dpp<16>(bad ? INFINITY : m);
    RowStat r;
    r.fine = m < INFINITY && m > -INFINITY;
    r.m = m;
    double s = 0.0;
    int32_t first = 0x7FFFFFFF;
    const Power power(r.m, c);
    const auto take = [&](const ChunkStat& v) {
        const double part = v.m > -INFINITY ? v.s * power.at(v.m) : 0.0;
        s += part;
        if (v.m == m) first = min(first, v.arg);
        return part;
    };
#pragma unroll
    for (int j = 0; j < kHeld; j++) {
        const double part = take(x[j]);
        if (shares) shares[lane + 16 * j] = part;
    }
    for (int32_t k = lane + 16 * kHeld; k < chunks; k += 16) take(st[k]);
    r.s = row_sum64(s);
    if (arg) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) first = min(first, __shfl_xor(first, o, 64));
    }
    r.arg = first;
    return r;
}

struct DecideLds {
    RowStat row[16];        // of a pass: target's rows, or target's and draft's in turns
    double shares[16][64];  // of their first chunks, target's rows where no drafts were drawn
};

// What request i's accepted drafts are, and what is drawn behind them, by the whole block. `write`: into the outputs too.
template <int DT, bool SHARES> __device__ __forceinline__ Pick decide(const DraftArgs& a, int32_t i, bool write, DecideLds& lds)
{
    const int tid = threadIdx.x, lane = tid & 63, group = tid >> 4;
    const int64_t s0 = a.starts[i], s1 = a.starts[i + 1];
    const bool inside = s0 >= 0 && s1 >= s0 && s1 <= a.T, fits = inside && s1 - s0 <= a.out_stride;
    const int32_t n = fits ? static_cast<int32_t>(s1 - s0) : 0;
    const Heat hp = heat_of(a.tau, i), hq = a.tau_q ? heat_of(a.tau_q, i) : hp;
    const double cp = kLog2e64 / hp.tau, cq = kLog2e64 / hq.tau;
    const bool drawn = a.draft && !hp.greedy && !hq.greedy;  // else the drafts were chosen: q is 1 there
    const int mats = drawn ? 2 : 1, rows = 16 / mats;
    int32_t* out = a.out + i * a.out_stride;
    float* logp = a.logp ? a.logp + i * a.out_stride : nullptr;
    int32_t stop = n, first = 0, draft = -1;  // the place of the token behind the accepted drafts; the pass's first row; the refused draft
    for (; first < n; first += rows) {
        const int32_t count = min(n - first, rows), place = first + group / mats, mat = group & (mats - 1);
        const int32_t mine = first + lane;
        const bool row = lane < count && mine < n - 1;  // the lane's row has a draft
        const int32_t x = row ? a.ids[s0 + mine + 1] : 0;
        const double u = row ? a.accept[s0 + mine] : 0.0;
        if (group < 16 && place < n && (mat == 0 || place < n - 1)) {
            const int64_t t = s0 + place;
            const int32_t v = place < n - 1 ? a.ids[t + 1] : 0;
            float z = -INFINITY;
            if (v >= 0 && v < a.V) z = Vec<DT>::load1(mat ? a.draft : a.target, t * (mat ? a.qs : a.zs) + v);
            const double c = mat ? cq : cp;
            RowStat r = row_stat(a.stats + (t * 2 + mat) * a.chunks, a.chunks, c, hp.greedy, SHARES ? lds.shares[group] : nullptr);
            r.fine &= !(mat ? hq.bad : hp.bad);
            r.z = z;
            const Power power(r.m, c);
            const double own = power.or_none(z);
            if (!drawn && !hp.greedy && place < n - 1) r.s += own;  // (its chunk's sum is without it)
            r.inv = 1.0 / r.s;
            r.share = own * r.inv;
            if ((tid & 15) == 0) lds.row[group] = r;
        }
        __syncthreads();
        // each wave looks at all rows of the pass, a lane each
        const RowStat &p = lds.row[(lane & (rows - 1)) * mats], &q = lds.row[(lane & (rows - 1)) * mats + mats - 1];
        const bool known = x >= 0 && x < a.V;
        bool good = false;
        if (row && p.fine && known) {
            if (hp.greedy) good = x == p.arg;
            else if (!drawn || q.fine) good = u * (drawn ? q.share : 1.0) < p.share;
        }
        const uint64_t refused = ~__ballot(good) & ((uint64_t{1} << count) - 1);
        if (refused) stop = first + __ffsll(static_cast<long long>(refused)) - 1;
        if (stop < n) draft = __builtin_amdgcn_readlane(x, stop - first);
        if (write && tid < 64) {
            if (good && mine < stop) {
                out[mine] = x;
                if (logp) logp[mine] = static_cast<float>((static_cast<double>(p.z) - p.m) * (cp / kLog2e64) - log(p.s));
            }
            if (row && !known && mine == stop)
                raise_error(a.err, kErrDraftToken, static_cast<uint32_t>(i), static_cast<uint32_t>(mine), static_cast<uint32_t>(x), static_cast<uint32_t>(a.V), 0, 0);
        }
        if (stop < n) break;
        __syncthreads();  // the next pass writes the rows
    }
    Pick k{};
    k.kind = kDone;
    k.held = -1;
    int32_t token = -1;
    float lp = NAN;
    if (n > 0) {
        const RowStat &p = lds.row[(stop - first) * mats], &q = lds.row[(stop - first) * mats + mats - 1];
        const bool last = stop == n - 1;
        k.row = static_cast<int32_t>(s0) + stop;
        k.place = stop;
        if (p.fine && hp.greedy) {
            token = p.arg;
            lp = static_cast<float>(-log(p.s));
        } else if (p.fine) {
            k.token = last ? -1 : draft;
            k.kind = last ? kFromTarget : !drawn ? kFromOthers : q.fine ? kFromRest : kFromTarget;
            k.mp = p.m;
            k.cp = cp;
            k.sum = p.s;
            if (k.kind == kFromRest) {
                k.mq = q.m;
                k.cq = cq;
                k.ratio = p.s * q.inv;
            }
            k.exact = last || !drawn;
            k.own = p.share * p.s;
            k.held = SHARES ? (stop - first) * mats : -1;
        }
    }
    if (!write) return k;
    if (tid == 0) {
        if (n > 0 && k.kind == kDone) {
            out[stop] = token;
            if (logp) logp[stop] = lp;
        }
        a.n_out[i] = n > 0 ? stop + 1 : 0;
        if (a.kept) a.kept[i] = (a.past ? a.past[i] : 0) + (n > 0 ? stop + 1 : 0);
        if (a.dropped) a.dropped[i] = n > 0 ? n - stop - 1 : inside ? static_cast<int32_t>(s1 - s0) : 0;  // (too many rows: all of them)
        if (!fits)
            raise_error(a.err, kErrKvRequest, static_cast<uint32_t>(i), static_cast<uint32_t>(i), a.past ? static_cast<uint32_t>(a.past[i]) : 0,
                        static_cast<uint32_t>(s1 - s0), static_cast<uint32_t>(static_cast<uint64_t>(s1 - s0) >> 32), 0);
    }
    for (int64_t j = (n > 0 ? stop + 1 : 0) + tid; j < a.out_stride; j += kDrawThreads) {
        out[j] = -1;
        if (logp) logp[j] = 0.0f;
    }
    return k;
}

// ---- the draw ------------------------------------------------------------------------------------------------------

// A thread's 16 bytes of a chunk, and their weights as the kind says: of max(p - q, 0) or of p, in units of p's powers.
template <int DT> struct Draws {
    static constexpr int N = Vec<DT>::N;
    typedef Logits<DT, kDrawThreads> Mine;
    static_assert(Mine::kVecs == 1);
    Mine x, y;
    __device__ __forceinline__ void load(const DraftArgs& a, const Pick& k, int32_t kind, int32_t chunk)
    {
        x.load(a.target, k.row, a.zs, a.V, chunk);
        if (kind == kFromRest) y.load(a.draft, k.row, a.qs, a.V, chunk);
    }
    __device__ __forceinline__ void logits(float (&z)[N]) const { Vec<DT>::unpack(x.w[0], z); }
    __device__ static __forceinline__ void powers(const uint4& w, double m, double c, double (&p)[N])
    {
        float z[N];
        Vec<DT>::unpack(w, z);
        Power(m, c).of(z, p);
#pragma unroll
        for (int e = 0; e < N; e++) p[e] = p[e] > kNone ? p[e] : 0.0;
    }
    __device__ __forceinline__ double rest(const Pick& k, double (&w)[N]) const
    {
#pragma clang fp contract(off)  // p - q of equal numbers is 0, not the rounding of a product
        double q[N], s = 0.0;
        powers(x.w[0], k.mp, k.cp, w);
        powers(y.w[0], k.mq, k.cq, q);
#pragma unroll
        for (int e = 0; e < N; e++) {
            w[e] = fmax(w[e] - q[e] * k.ratio, 0.0);
            s += w[e];
        }
        return s;
    }
    __device__ __forceinline__ double own(const Pick& k, int32_t kind, int32_t at, double (&w)[N]) const
    {
        double s = 0.0;
        powers(x.w[0], k.mp, k.cp, w);
        if (kind == kFromOthers && k.token >= at && k.token < at + N) {
#pragma unroll
            for (int e = 0; e < N; e++) w[e] = at + e == k.token ? 0.0 : w[e];
        }
#pragma unroll
        for (int e = 0; e < N; e++) s += w[e];
        return s;
    }
};

// A chunk's sums, by the whole block, number j in thread j. ratio is of the rows' f32 sums: where that puts a place on the wrong side of 0, p - ratio q is
// 2^-20 of p or less, and `rest` is corrected by the ratio's error times `above`.
template <int DT> __device__ __forceinline__ double chunk_sums(const DraftArgs& a, const Pick& k, int32_t chunk, double (&lds)[kDrawWaves][4])
{
    constexpr int N = Vec<DT>::N;
    const bool both = k.kind == kFromRest;
    double s[4] = {};
    float z[N], v[N];
    Draws<DT> mine;
    mine.load(a, k, k.kind, chunk);
    Vec<DT>::unpack(mine.x.w[0], z);
    if (both) Vec<DT>::unpack(mine.y.w[0], v);
    const Power of_p(k.mp, k.cp), of_q(k.mq, k.cq);
#pragma unroll
    for (int e = 0; e < N; e += kTogether) {
        double p[kTogether], q[kTogether];
        of_p.of(&z[e], p);
#pragma unroll
        for (int i = 0; i < kTogether; i++) s[0] += p[i];
        if (both) {
            of_q.of(&v[e], q);
#pragma unroll
            for (int i = 0; i < kTogether; i++) {
                const double rest = fma(-k.ratio, q[i], p[i]);
                s[1] += q[i];
                s[2] += fmax(rest, 0.0);
                s[3] += rest > 0.0 ? q[i] : 0.0;
            }
        }
    }
    const int lane = threadIdx.x & 63;
    const double sum = wave_sums64(s);
    if (lane < 4) lds[wave_id()][lane] = sum;
    __syncthreads();
    return sum_by_four(lds[lane >> 2][lane & 3]);
}

// What is below it counts as 0: a chunk that is above has a place that is above 2^-1000 (a random number of 0 is above no other's sum).
constexpr double kLeastShare = 0x1p-900;

// The draw itself, by the whole block, in units of p's powers. Where the draft was drawn and refused, chunk c's weight is of its sums[c]; else of the target's chunk
// sums, which leave a chosen draft out (a difference would leave nothing beside a draft of nearly all).
// Every wave finds the chunk for itself, a lane for one or more neighbours, and all of them the place in it, 16 bytes a thread.
template <int DT, bool DRAWN> __device__ __forceinline__ void pick(const DraftArgs& a, int32_t i, Pick k, float u, const double* shares)
{
    constexpr int N = Vec<DT>::N;
    __shared__ double s_part[kDrawWaves], s_log;
    __shared__ int32_t s_flags[kDrawWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int32_t each = (a.chunks + 63) / 64, c0 = min(lane * each, a.chunks), c1 = min(c0 + each, a.chunks);
    const ChunkStat* st = a.stats + static_cast<int64_t>(k.row) * 2 * a.chunks;
    const ChunkSums* sums = a.sums + static_cast<int64_t>(i) * a.chunks;
    int32_t kind = k.kind;
    const int32_t other = kind == kFromOthers && k.token >= 0 && k.token < a.V ? k.token / kChunk<DT> : -1;
    const bool summed = DRAWN && !k.exact;
    double correct = 0.0;  // of the ratio
    ChunkSums near{};      // of the lane's first chunk
    if (summed) {
        if (c0 < c1) near = sums[c0];
        double p = near.p, q = near.q;
        for (int32_t c = c0 + 1; c < c1; c++) {
            p += sums[c].p;
            q += sums[c].q;
        }
        k.sum = wave_sum64(p);
        if (kind == kFromRest) {
            const double exact = k.sum / wave_sum64(q);
            correct = exact - k.ratio;
            k.ratio = exact;
        }
    }
    const auto weight = [&](int32_t c) {
        double v, least = kLeastShare;
        if (summed) {
            const ChunkSums x = c == c0 ? near : sums[c];
            v = x.p;
            if (kind == kFromRest) {
                v = x.rest - correct * x.above;
                least = fmax(least, 0x1p-36 * (v + k.ratio * x.above));  // (below it are roundings: there may be no place that has a weight)
            }
        } else if (!DRAWN && c < 16 * kHeld) {
            v = shares[c];
        } else {
            const ChunkStat x = st[c];
            v = x.m > -INFINITY ? x.s * Power(k.mp, k.cp).at(x.m) : 0.0;
        }
        return (v > least ? v : 0.0) + (kind == kFromTarget && c == other ? k.own : 0.0);
    };
    const auto sum_of = [&]() {
        double s = 0.0;
        for (int32_t c = c0; c < c1; c++) s += weight(c);
        return s;
    };
    double mine = sum_of(), up = wave_scan64(mine);
    if (!(lane64(up, 63) > 0.0)) {  // p and q are equal, or the draft has all of p: p
        kind = kFromTarget;
        mine = sum_of();
        up = wave_scan64(mine);
    }
    const double r = lane64(up, 63) * (u > 0.0f ? u : 0.0f);
    // the chunk: the first whose inclusive sum is above r, or the last one with a weight
    const uint64_t some = __ballot(mine > 0.0), above = __ballot(mine > 0.0 && up > r);
    const bool end = !above;  // rounding: the last weight of all
    const int from = above ? __ffsll(static_cast<long long>(above)) - 1 : some ? 63 - __clzll(static_cast<long long>(some)) : 0;
    double base = lane64(up - mine, from);
    int32_t chunk = min(from * each, a.chunks - 1);
    if (each > 1) {
        double sum = base;
        for (int32_t c = chunk, last = min(chunk + each, a.chunks); c < last; c++) {
            const double v = weight(c);
            if (v > 0.0) {
                base = sum;
                chunk = c;
            }
            sum += v;
            if (!end && v > 0.0 && sum > r) break;
        }
    }
    Draws<DT> of;
    of.load(a, k, kind, chunk);
    if (a.logp && wave == 0) s_log = log(k.sum);  // while the loads are on their way
    const int32_t at = Logits<DT, kDrawThreads>::place(chunk, 0);
    double w[N];
    const double s = kind == kFromRest ? of.rest(k, w) : of.own(k, kind, at, w);
    double c = wave_scan64(s);
    if (lane == 63) s_part[wave] = c;
    c -= s;
    __syncthreads();
    {  // the waves before
        const double v = s_part[lane & (kDrawWaves - 1)];
        c += base + row_sum64((lane & (kDrawWaves - 1)) < wave ? v : 0.0);
    }
    // the first thread whose inclusive sum is above r, or the last one with a weight, and the place among its own
    const uint64_t found = __ballot(s > 0.0 && c + s > r), held = __ballot(s > 0.0);
    if (lane == 0) s_flags[wave] = (found && !end ? 1 : 0) + (held ? 2 : 0);
    __syncthreads();
    const int32_t flags = s_flags[lane & (kDrawWaves - 1)];
    const uint64_t waves = (uint64_t{1} << kDrawWaves) - 1, finds = __ballot(flags & 1) & waves, holds = __ballot(flags & 2) & waves;
    const auto highest = [](uint64_t lanes) { return lanes ? 63 - __clzll(static_cast<long long>(lanes)) : 0; };
    if (wave != (finds ? __ffsll(static_cast<long long>(finds)) - 1 : highest(holds))) return;
    if (lane != (finds ? __ffsll(static_cast<long long>(found)) - 1 : highest(held))) return;
    float z[N];
    of.logits(z);
    int32_t token = at;
    float logit = z[0];
    bool there = false;
#pragma unroll
    for (int n = 0; n < N; n++) {
        const double v = w[n];
        c += v;
        if (v > 0.0 && !there) {
            token = at + n;
            logit = z[n];
            there = finds && c > r;
        }
    }
    a.out[i * a.out_stride + k.place] = token;
    if (a.logp) a.logp[i * a.out_stride + k.place] = static_cast<float>((logit - k.mp) * (k.cp / kLog2e64) - s_log);
}

// Drafts that were chosen, or none: the sums of p are there, a thread block a request does the rest.
template <int DT> __global__ __launch_bounds__(kDrawThreads) void draft_choose(DraftArgs a)
{
    __shared__ DecideLds lds;
    const float u = a.T > 0 ? a.sample[blockIdx.x] : 0.0f;
    const Pick k = decide<DT, true>(a, blockIdx.x, true, lds);
    if (k.kind != kDone) pick<DT, false>(a, blockIdx.x, k, u, lds.shares[k.held]);
}

// Drafts that were drawn: what is accepted, then a thread block for each chunk of the row that is drawn from. Few chunks in all (kDecides) are
// a latency: each then decides for itself, in one launch.
template <int DT> __global__ __launch_bounds__(kDrawThreads) void draft_decide(DraftArgs a)
{
    __shared__ DecideLds lds;
    const Pick k = decide<DT, false>(a, blockIdx.x, true, lds);
    if (threadIdx.x == 0) a.picks[blockIdx.x] = k;
}

constexpr int64_t kDecides = 512;
constexpr unsigned kRequestsY = 32768;  // of a launch's second dimension

template <int DT, bool DECIDES> __global__ __launch_bounds__(kDrawThreads) void draft_sums(DraftArgs a)
{
    __shared__ double s_sum[kDrawWaves][4];
    const int32_t i = blockIdx.z * kRequestsY + blockIdx.y, chunk = blockIdx.x;
    if (i >= a.B) return;
    Pick k;
    if constexpr (DECIDES) {
        __shared__ DecideLds lds;
        k = decide<DT, false>(a, i, chunk == 0, lds);
        if (chunk == 0 && threadIdx.x == 0) a.picks[i] = k;
    } else {
        k = a.picks[i];
    }
    if (k.kind == kDone || k.exact) return;
    const double s = chunk_sums<DT>(a, k, chunk, s_sum);
    if (threadIdx.x < 4) reinterpret_cast<double*>(a.sums + static_cast<int64_t>(i) * a.chunks + chunk)[threadIdx.x] = s;
}

template <int DT> __global__ __launch_bounds__(kDrawThreads) void draft_pick(DraftArgs a)
{
    const float u = a.T > 0 ? a.sample[blockIdx.x] : 0.0f;
    const Pick k = a.picks[blockIdx.x];
    if (k.kind != kDone) pick<DT, true>(a, blockIdx.x, k, u, nullptr);
}

// ---- host ----------------------------------------------------------------------------------------------------------

static int64_t round16(int64_t n) { return (n + 15) & ~int64_t{15}; }

// The workspace: chunk sums of all rows, the picks, their chunks' sums.
static int64_t work_of(int64_t B, int64_t T, int64_t chunks)
{
    return T * 2 * chunks * static_cast<int64_t>(sizeof(ChunkStat)) + round16(B * static_cast<int64_t>(sizeof(Pick))) + B * chunks * static_cast<int64_t>(sizeof(ChunkSums));
}

// chunks: of the smaller kind, f32's.
static int check_sizes(int64_t B, int64_t T, int64_t V, int64_t* chunks)
{
    if (B < 0 || T < 0 || V < 1) return fail(SLHIP_ERR_INVALID, "draft_verify: bad size");
    *chunks = V > kMaxVocab ? 0 : (V + kChunk<SLHIP_F32> - 1) / kChunk<SLHIP_F32>;
    // (products of what is below 2^24 only: any numbers may come)
    if (B > 65536 || V > kMaxVocab || T > 0xFFFFFF || T * *chunks * 2 > 0xFFFFFF || B * *chunks > 0xFFFFFF)
        return fail(SLHIP_ERR_UNSUPPORTED, "draft_verify: too many requests, rows or tokens of the vocabulary");
    return SLHIP_OK;
}

template <int DT> static int launch(DraftArgs& a, hipStream_t st)
{
    a.chunks = (a.V + kChunk<DT> - 1) / kChunk<DT>;
    const unsigned rows = static_cast<unsigned>(a.T * a.chunks), B = static_cast<unsigned>(a.B);
    // a request's chunks after one another (with the requests first, 2432 chunks take 18.6 us instead of 12.9); in one dimension they could have 2^32 threads
    const dim3 chunks(static_cast<unsigned>(a.chunks), B < kRequestsY ? B : kRequestsY, (B + kRequestsY - 1) / kRequestsY);
    if (rows > 0) {
        if (a.draft)
            draft_stats<DT, true><<<rows * 2, kThreads, 0, st>>>(a);
        else
            draft_stats<DT, false><<<rows, kThreads, 0, st>>>(a);
        const int e = check_launch("draft_stats");
        if (e) return e;
    }
    if (!a.draft) {
        draft_choose<DT><<<B, kDrawThreads, 0, st>>>(a);
        return check_launch("draft_choose");
    }
    if (static_cast<int64_t>(B) * a.chunks <= kDecides) {
        draft_sums<DT, true><<<chunks, kDrawThreads, 0, st>>>(a);
    } else {
        draft_decide<DT><<<B, kDrawThreads, 0, st>>>(a);
        const int e = check_launch("draft_decide");
        if (e) return e;
        draft_sums<DT, false><<<chunks, kDrawThreads, 0, st>>>(a);
    }
    const int e = check_launch("draft_sums");
    if (e) return e;
    draft_pick<DT><<<B, kDrawThreads, 0, st>>>(a);
    return check_launch("draft_pick");
}

}  // namespace slhip

using namespace slhip;

extern "C" SLHIP_API int64_t slhip_draft_verify_work_bytes(int64_t requests, int64_t tokens, int64_t vocab)
{
    int64_t chunks;
    if (check_sizes(requests, tokens, vocab, &chunks)) return -1;
    return work_of(requests, tokens, chunks);
}

extern "C" SLHIP_API int slhip_draft_verify(int dtype, const void* target, int64_t target_stride, const void* draft, int64_t draft_stride,
                                            const slhip_drafts* d, void* work, int64_t work_bytes, slhip_stream stream)
{
    if (!d) return fail(SLHIP_ERR_INVALID, "draft_verify: arguments are null");
    if (dtype != SLHIP_F32 && dtype != SLHIP_BF16) return fail(SLHIP_ERR_UNSUPPORTED, "draft_verify: dtype %d not supported", dtype);
    int64_t chunks;
    int e = check_sizes(d->requests, d->tokens, d->vocab, &chunks);
    if (e) return e;
    if (d->out_stride < 0 || d->out_stride > 0x7FFFFFFF) return fail(SLHIP_ERR_INVALID, "draft_verify: bad stride of the tokens");
    if (target_stride < d->vocab || (draft && draft_stride < d->vocab))
        return fail(SLHIP_ERR_INVALID, "draft_verify: a row stride is smaller than the vocabulary");
    if (d->requests == 0) return SLHIP_OK;
    if (!d->starts || !d->n_out || (d->out_stride > 0 && !d->out)) return fail(SLHIP_ERR_INVALID, "draft_verify: starts, out and n_out are required");
    if (d->tokens > 0 && (!target || !d->ids || !d->accept || !d->sample))
        return fail(SLHIP_ERR_INVALID, "draft_verify: target, ids, accept and sample are required");
    const int64_t need = work_of(d->requests, d->tokens, chunks);
    if (!work || !aligned16(work) || work_bytes < need)
        return fail(SLHIP_ERR_INVALID, "draft_verify: the workspace has %lld bytes, %lld are needed (16-byte aligned)",
                    static_cast<long long>(work ? work_bytes : 0), static_cast<long long>(need));
    DraftArgs a{};
    a.target = target;
    a.draft = draft;
    a.zs = target_stride;
    a.qs = draft_stride;
    a.T = d->tokens;
    a.B = static_cast<int32_t>(d->requests);
    a.V = static_cast<int32_t>(d->vocab);
    a.starts = d->starts;
    a.ids = d->ids;
    a.tau = d->temperature;
    a.tau_q = d->draft_temperature;
    a.accept = d->accept;
    a.sample = d->sample;
    a.out = d->out;
    a.n_out = d->n_out;
    a.out_stride = d->out_stride;
    a.past = d->past;
    a.kept = d->kept;
    a.dropped = d->dropped;
    a.logp = d->logp;
    a.stats = static_cast<ChunkStat*>(work);
    a.picks = reinterpret_cast<Pick*>(a.stats + a.T * 2 * chunks);
    a.sums = reinterpret_cast<ChunkSums*>(reinterpret_cast<char*>(a.picks) + round16(a.B * static_cast<int64_t>(sizeof(Pick))));
    e = error_word(&a.err);
    if (e) return e;
    return dtype == SLHIP_F32 ? launch<SLHIP_F32>(a, to_stream(stream)) : launch<SLHIP_BF16>(a, to_stream(stream));
}
