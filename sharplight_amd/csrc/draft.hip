// Verification of drafted tokens, and the draw of the next one (slhip_draft_verify).
//
// Mathematics. Row t of the target's logits z: p(v) = e^((z_v - M) / tau) / S, S = sum_v e^((z_v - M) / tau), M = max z; q the same
// of the draft's logits. Draft x is accepted while u q(x) < p(x). What is drawn behind the accepted ones has the weights
// max(p - q, 0) of the refused draft's row, or p of the last row: the first v whose inclusive sum is above w times the sum of all.
//
// Every row's S is needed for its p(x), so the rows are read once for their sums (HBM bounds it), in chunks that lie in
// registers: a chunk's maximum first, then one exponential a logit, no running rescale. Which row is drawn from follows from all
// of a request's sums; that row alone is read again, for sums of weights chunk by chunk, and one chunk a third time, for the
// place in it.
//
// Numbers. A choice changes where a sum passes a random number, so what two implementations may differ in is kept small: chunk
// sums are f32 exponentials of arguments with one rounding (log2(e) / tau in two parts, or all terms of a sum would be off the same
// way), everything behind them f64: the rows' sums, p(x), q(x), and the drawn row's weights, whose differences p - q cancel.
#include <float.h>
#include <math.h>

#include "step.hpp"

namespace slhip {

constexpr int kChunk = 4096;       // logits of a chunk
constexpr int kThreads = 256;
constexpr int kEach = kChunk / kThreads;
constexpr int kDecide = 1024;      // threads of draft_decide
constexpr int64_t kMaxVocab = 1 << 24;

struct ChunkStat {
    float m;      // the largest logit; NaN where the chunk holds a NaN or an infinity above
    int32_t arg;  // its first place (rows of greedy requests)
    double s;     // sum of e^((z - m) / tau)
};

// What is drawn for a request, and from what.
enum : int32_t { kDone = 0, kFromTarget = 1, kFromRest = 2, kFromOthers = 3 };  // nothing; p; max(p - q, 0); p without the draft
struct Pick {
    int32_t kind, row, place, token;  // the row, its place in the request, its draft
    double mp, cp, ip, mq, cq, iq;    // maxima, log2(e) / tau, 1 / sums
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
    double* sums;      // [B][chunks]
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

// A thread's logits of a chunk: vectors of 16 bytes, a block's threads side by side, in the order of the vocabulary from one step
// to the next. Places past the vocabulary are -inf.
template <int DT> struct Logits {
    static constexpr int N = Vec<DT>::N, kVecs = kEach / N;
    float z[kEach];
    __device__ static __forceinline__ int32_t place(int32_t chunk, int j) { return chunk * kChunk + (j * kThreads + static_cast<int>(threadIdx.x)) * N; }
    __device__ __forceinline__ void load(const void* rows, int64_t row, int64_t stride, int32_t V, int32_t chunk)
    {
        const char* p = static_cast<const char*>(rows) + row * stride * Vec<DT>::BYTES;
        uint4 w[kVecs];
#pragma unroll
        for (int j = 0; j < kVecs; j++) {
            const int32_t v = place(chunk, j);
            w[j] = make_uint4(0, 0, 0, 0);
            if (v + N <= V) w[j] = load_any(p + static_cast<int64_t>(v) * Vec<DT>::BYTES);
        }
#pragma unroll
        for (int j = 0; j < kVecs; j++) {
            const int32_t v = place(chunk, j);
            Vec<DT>::unpack(w[j], &z[j * N]);
            if (v + N > V) {
                for (int k = 0; k < N; k++) z[j * N + k] = v + k < V ? Vec<DT>::load1(p, v + k) : -INFINITY;
            }
        }
    }
};

__device__ __forceinline__ double wave_sum64(double v)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// 2^y to 2^-40 of itself for y <= 0 (0 below -1000): the series of 2^f, |f| <= 1/2.
__device__ __forceinline__ double exp2_64(double y)
{
    const double n = rint(y), f = (y - n) * 0.693147180559945309417;
    double r = 1.0 / 39916800.0;
    r = fma(r, f, 1.0 / 3628800.0);
    r = fma(r, f, 1.0 / 362880.0);
    r = fma(r, f, 1.0 / 40320.0);
    r = fma(r, f, 1.0 / 5040.0);
    r = fma(r, f, 1.0 / 720.0);
    r = fma(r, f, 1.0 / 120.0);
    r = fma(r, f, 1.0 / 24.0);
    r = fma(r, f, 1.0 / 6.0);
    r = fma(r, f, 0.5);
    r = fma(r, f, 1.0);
    r = fma(r, f, 1.0);
    return y < -1000.0 ? 0.0 : ldexp(r, static_cast<int>(n));
}

constexpr double kLog2e64 = 1.44269504088896340736;

__device__ __forceinline__ double share_of(float z, double m, double c) { return z == -INFINITY ? 0.0 : exp2_64((static_cast<double>(z) - m) * c); }

// ---- the sums of all rows ------------------------------------------------------------------------------------------

template <int DT, bool DRAFT> __global__ __launch_bounds__(kThreads) void draft_stats(DraftArgs a)
{
    __shared__ float s_m[kThreads / 64];
    __shared__ double s_s[kThreads / 64];
    __shared__ int32_t s_arg[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = wave_id();
    constexpr int kMats = DRAFT ? 2 : 1;
    const int64_t item = blockIdx.x, t = item / (a.chunks * kMats);
    const int32_t rest = static_cast<int32_t>(item - t * (a.chunks * kMats)), mat = rest / a.chunks, chunk = rest - mat * a.chunks;
    Logits<DT> x;
    if (mat == 0) x.load(a.target, t, a.zs, a.V, chunk);
    if (t >= a.starts[a.B]) return;
    const int32_t i = row_request(a.starts, a.B, t);
    const Heat target = heat_of(a.tau, i), h = mat == 0 || !a.tau_q ? target : heat_of(a.tau_q, i);
    if (mat == 1) {  // not of greedy requests, nor of the row that has no draft
        if (target.greedy || h.greedy || t == a.starts[i + 1] - 1) return;
        x.load(a.draft, t, a.qs, a.V, chunk);
    }
    float m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < kEach; j++) {
        m = fmaxf(m, x.z[j]);
        bad |= !(x.z[j] < INFINITY);
    }
    m = group_max<64>(m);
    if (__any(bad)) m = INFINITY;
    if (lane == 0) s_m[wave] = m;
    __syncthreads();
    m = s_m[0];
    for (int w = 1; w < kThreads / 64; w++) m = fmaxf(m, s_m[w]);
    const double c = kLog2e64 / h.tau;
    const float hi = static_cast<float>(c), lo = static_cast<float>(c - hi);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < kEach; j++) {
        const float d = fmaxf(x.z[j] - m, -0x1p60f);
        s += __builtin_amdgcn_exp2f(fmaf(d, hi, d * lo));
    }
    const double sum = wave_sum64(s);
    int32_t arg = 0x7FFFFFFF;
    if (target.greedy) {
#pragma unroll
        for (int j = kEach - 1; j >= 0; j--)
            if (x.z[j] == m) arg = Logits<DT>::place(chunk, j / Logits<DT>::N) + j % Logits<DT>::N;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) arg = min(arg, __shfl_xor(arg, o, 64));
    }
    if (lane == 0) {
        s_s[wave] = sum;
        s_arg[wave] = arg;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        ChunkStat o{m == INFINITY ? NAN : m, s_arg[0], s_s[0]};
        for (int w = 1; w < kThreads / 64; w++) {
            o.s += s_s[w];
            o.arg = min(o.arg, s_arg[w]);
        }
        if (m == -INFINITY) o.s = 0.0;
        a.stats[(t * 2 + mat) * a.chunks + chunk] = o;
    }
}

// ---- what is accepted ----------------------------------------------------------------------------------------------

struct RowStat {
    double m, s;
    int32_t arg;
    bool fine;
};

// The chunks of a row together, by a whole wave.
__device__ __forceinline__ RowStat row_stat(const DraftArgs& a, int64_t t, int mat, double c)
{
    const ChunkStat* st = a.stats + (t * 2 + mat) * a.chunks;
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    bool bad = false;
    for (int32_t k = lane; k < a.chunks; k += 64) {
        const float x = st[k].m;
        bad |= x != x;
        m = fmaxf(m, x);
    }
    m = group_max<64>(m);
    RowStat r;
    r.fine = !__any(bad) && m > -INFINITY;
    r.m = m;
    double s = 0.0;
    int32_t arg = 0x7FFFFFFF;
    for (int32_t k = lane; k < a.chunks; k += 64) {
        const ChunkStat x = st[k];
        if (x.m > -INFINITY) s += x.s * exp2_64((static_cast<double>(x.m) - r.m) * c);
        if (x.m == m) arg = min(arg, x.arg);
    }
    r.s = wave_sum64(s);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) arg = min(arg, __shfl_xor(arg, o, 64));
    r.arg = arg;
    return r;
}

template <int DT> __global__ __launch_bounds__(kDecide) void draft_decide(DraftArgs a)
{
    constexpr int kWaves = kDecide / 64, kRows = kWaves / 2;  // rows of a pass: a wave for the target's sums, one for the draft's
    __shared__ RowStat s_row[kRows][2];
    __shared__ int32_t s_stop;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int32_t i = blockIdx.x;
    const int64_t s0 = a.starts[i], s1 = a.starts[i + 1];
    const bool fits = s0 >= 0 && s1 >= s0 && s1 <= a.T && s1 - s0 <= a.out_stride;
    const int32_t n = fits ? static_cast<int32_t>(s1 - s0) : 0;
    const Heat hp = heat_of(a.tau, i), hq = a.tau_q ? heat_of(a.tau_q, i) : hp;
    const double cp = kLog2e64 / hp.tau, cq = kLog2e64 / hq.tau;
    const bool drawn = a.draft && !hp.greedy && !hq.greedy;  // else the drafts were chosen: q is 1 there
    int32_t* out = a.out + i * a.out_stride;
    float* logp = a.logp ? a.logp + i * a.out_stride : nullptr;
    int32_t stop = n;  // the place of the token behind the accepted drafts
    for (int32_t first = 0; first < n && stop == n; first += kRows) {
        const int32_t count = min(n - first, kRows), j = wave >> 1;
        if (j < count && ((wave & 1) == 0 || (drawn && first + j < n - 1))) {
            const RowStat r = row_stat(a, s0 + first + j, wave & 1, wave & 1 ? cq : cp);
            if (lane == 0) s_row[j][wave & 1] = r;
        }
        __syncthreads();
        if (wave == 0) {
            const int32_t place = first + lane;
            const int64_t t = s0 + place;
            const bool row = lane < count && place < n - 1;  // it has a draft
            const RowStat &p = s_row[lane & (kRows - 1)][0], &q = s_row[lane & (kRows - 1)][1];
            const int32_t x = row ? a.ids[t + 1] : 0;
            const bool fine = row && p.fine && !hp.bad, known = x >= 0 && x < a.V;
            bool good = false;
            float z = 0.0f;
            if (fine && known) {
                z = Vec<DT>::load1(a.target, t * a.zs + x);
                if (hp.greedy) {
                    good = x == p.arg;
                } else if (!drawn || (q.fine && !hq.bad)) {
                    const double qx = drawn ? share_of(Vec<DT>::load1(a.draft, t * a.qs + x), q.m, cq) / q.s : 1.0;
                    good = static_cast<double>(a.accept[t]) * qx < share_of(z, p.m, cp) / p.s;
                }
            }
            const uint64_t refused = ~__ballot(good) & ((uint64_t{1} << count) - 1);
            const int32_t to = refused ? first + __ffsll(static_cast<long long>(refused)) - 1 : n;
            if (good && place < to) {
                out[place] = x;
                if (logp) logp[place] = static_cast<float>((static_cast<double>(z) - p.m) * (cp / kLog2e64) - log(p.s));
            }
            if (fine && !known && place == to)
                raise_error(a.err, kErrDraftToken, static_cast<uint32_t>(i), static_cast<uint32_t>(place), static_cast<uint32_t>(x), static_cast<uint32_t>(a.V), 0, 0);
            if (lane == 0) s_stop = to;
        }
        __syncthreads();
        stop = s_stop;
        if (stop == n) __syncthreads();  // the next pass writes s_row
    }
    if (wave != 0) return;
    if (lane == 0) {
        Pick k{};
        k.kind = kDone;
        if (n > 0) {
            const int32_t j = stop % kRows;
            const RowStat &p = s_row[j][0], &q = s_row[j][1];
            const int64_t t = s0 + stop;
            const bool last = stop == n - 1;
            k.row = static_cast<int32_t>(t);
            k.place = stop;
            if (!p.fine || hp.bad) {
                out[stop] = -1;
                if (logp) logp[stop] = NAN;
            } else if (hp.greedy) {
                out[stop] = p.arg;
                if (logp) logp[stop] = static_cast<float>(-log(p.s));
            } else {
                k.token = last ? -1 : a.ids[t + 1];
                k.kind = last ? kFromTarget : !drawn ? kFromOthers : q.fine && !hq.bad ? kFromRest : kFromTarget;
                k.mp = p.m;
                k.cp = cp;
                k.ip = 1.0 / p.s;
                k.mq = q.m;
                k.cq = cq;
                k.iq = 1.0 / q.s;
            }
            a.n_out[i] = stop + 1;
        } else {
            a.n_out[i] = 0;
            if (!fits)
                raise_error(a.err, kErrKvRequest, static_cast<uint32_t>(i), static_cast<uint32_t>(i), a.past ? static_cast<uint32_t>(a.past[i]) : 0,
                            static_cast<uint32_t>(s1 - s0), static_cast<uint32_t>(static_cast<uint64_t>(s1 - s0) >> 32), 0);
        }
        a.picks[i] = k;
        if (a.kept) a.kept[i] = (a.past ? a.past[i] : 0) + (n > 0 ? stop + 1 : 0);
        if (a.dropped) a.dropped[i] = n > 0 ? n - stop - 1 : 0;
    }
    for (int64_t j = (n > 0 ? stop + 1 : 0) + lane; j < a.out_stride; j += 64) {
        out[j] = -1;
        if (logp) logp[j] = 0.0f;
    }
}

// ---- the draw ------------------------------------------------------------------------------------------------------

// The weights of a thread's logits of a chunk. `all`: p, whatever the pick's kind is.
template <int DT> __device__ __forceinline__ void weights(const DraftArgs& a, const Pick& k, int32_t chunk, bool all, double (&w)[kEach])
{
#pragma clang fp contract(off)  // p - q of equal numbers is 0, not the rounding of a product
    Logits<DT> x;
    x.load(a.target, k.row, a.zs, a.V, chunk);
#pragma unroll
    for (int j = 0; j < kEach; j++) w[j] = share_of(x.z[j], k.mp, k.cp) * k.ip;
    if (all || k.kind == kFromTarget) return;
    if (k.kind == kFromOthers) {
#pragma unroll
        for (int j = 0; j < kEach; j++)
            if (Logits<DT>::place(chunk, j / Logits<DT>::N) + j % Logits<DT>::N == k.token) w[j] = 0.0;
        return;
    }
    x.load(a.draft, k.row, a.qs, a.V, chunk);
#pragma unroll
    for (int j = 0; j < kEach; j++) w[j] = fmax(w[j] - share_of(x.z[j], k.mq, k.cq) * k.iq, 0.0);
}

// The sum over the thread block, in every thread.
__device__ __forceinline__ double block_sum(double v, double* lds)
{
    v = wave_sum64(v);
    if ((threadIdx.x & 63) == 0) lds[wave_id()] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < kThreads / 64; w++) s += lds[w];
    __syncthreads();
    return s;
}

template <int DT> __device__ __forceinline__ double chunk_sum(const DraftArgs& a, const Pick& k, int32_t chunk, bool all, double* lds)
{
    double w[kEach], s = 0.0;
    weights<DT>(a, k, chunk, all, w);
#pragma unroll
    for (int j = 0; j < kEach; j++) s += w[j];
    return block_sum(s, lds);
}

template <int DT> __global__ __launch_bounds__(kThreads) void draft_sums(DraftArgs a)
{
    __shared__ double lds[kThreads / 64];
    const int32_t i = blockIdx.x / a.chunks, chunk = blockIdx.x - i * a.chunks;
    const Pick k = a.picks[i];
    if (k.kind == kDone) return;
    const double s = chunk_sum<DT>(a, k, chunk, false, lds);
    if (threadIdx.x == 0) a.sums[static_cast<int64_t>(i) * a.chunks + chunk] = s;
}

// Inclusive sums over the thread block.
__device__ __forceinline__ double block_scan(double v, double* lds)
{
    const int lane = threadIdx.x & 63, wave = wave_id();
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; w++) v += lds[w];
    __syncthreads();
    return v;
}

template <int DT> __global__ __launch_bounds__(kThreads) void draft_pick(DraftArgs a)
{
    __shared__ double lds[kThreads / 64];
    __shared__ int32_t s_place, s_last;
    __shared__ double s_before;
    constexpr int N = Logits<DT>::N;
    const int32_t i = blockIdx.x, tid = threadIdx.x;
    const Pick k = a.picks[i];
    if (k.kind == kDone) return;
    double* sums = a.sums + static_cast<int64_t>(i) * a.chunks;
    double mine = 0.0;
    for (int32_t c = tid; c < a.chunks; c += kThreads) mine += sums[c];
    double total = block_sum(mine, lds);
    const bool all = !(total > 0.0);  // p and q are equal: p
    if (all) {
        for (int32_t c = 0; c < a.chunks; c++) {
            const double s = chunk_sum<DT>(a, k, c, true, lds);
            if (tid == 0) sums[c] = s;
        }
        __syncthreads();
        mine = 0.0;
        for (int32_t c = tid; c < a.chunks; c += kThreads) mine += sums[c];
        total = block_sum(mine, lds);
    }
    const float u = a.sample[i];
    const double r = total * (u > 0.0f ? u : 0.0f);
    // the chunk: the first whose inclusive sum is above r, or the last one with a weight
    if (tid == 0) {
        s_place = 0x7FFFFFFF;
        s_last = 0;
    }
    double before = 0.0;
    int32_t chunk = -1;
    __syncthreads();
    for (int32_t c0 = 0; c0 < a.chunks && chunk < 0; c0 += kThreads) {
        const int32_t c = c0 + tid;
        const double v = c < a.chunks ? sums[c] : 0.0, up = before + block_scan(v, lds);
        if (v > 0.0) {
            atomicMax(&s_last, c);
            if (up > r) atomicMin(&s_place, c);
        }
        __syncthreads();
        if (s_place != 0x7FFFFFFF) chunk = s_place;
        if (c == chunk) s_before = up - v;
        if (tid == kThreads - 1) lds[0] = up;
        __syncthreads();
        before = chunk < 0 ? lds[0] : s_before;
        __syncthreads();
    }
    const bool end = chunk < 0;  // rounding: the last weight of all
    if (end) chunk = s_last;
    if (tid == 0) {
        s_place = 0x7FFFFFFF;
        s_last = 0;
    }
    __syncthreads();
    double w[kEach];
    weights<DT>(a, k, chunk, all, w);
#pragma unroll
    for (int j = 0; j < kEach; j += N) {
        double s = 0.0;
        for (int e = 0; e < N; e++) s += w[j + e];
        const double up = before + block_scan(s, lds);
        double c = up - s;
        const int32_t at = Logits<DT>::place(chunk, j / N);
        int32_t last = -1, place = -1;
        for (int e = 0; e < N; e++) {
            c += w[j + e];
            if (w[j + e] > 0.0) {
                last = at + e;
                if (place < 0 && c > r) place = at + e;
            }
        }
        if (last >= 0) atomicMax(&s_last, last);
        if (place >= 0 && !end) atomicMin(&s_place, place);
        if (tid == kThreads - 1) lds[0] = up;
        __syncthreads();
        before = lds[0];
        __syncthreads();
    }
    if (tid == 0) {
        const int32_t token = s_place != 0x7FFFFFFF ? s_place : s_last;
        a.out[i * a.out_stride + k.place] = token;
        if (a.logp)
            a.logp[i * a.out_stride + k.place] =
                static_cast<float>((static_cast<double>(Vec<DT>::load1(a.target, k.row * a.zs + token)) - k.mp) * (k.cp / kLog2e64) + log(k.ip));
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------

static int64_t round16(int64_t n) { return (n + 15) & ~int64_t{15}; }

// The workspace: chunk sums of all rows, the picks, their chunks' sums.
static int64_t work_of(int64_t B, int64_t T, int64_t chunks)
{
    return T * 2 * chunks * static_cast<int64_t>(sizeof(ChunkStat)) + round16(B * static_cast<int64_t>(sizeof(Pick))) + round16(B * chunks * 8);
}

static int check_sizes(int64_t B, int64_t T, int64_t V)
{
    if (B < 0 || T < 0 || V < 1) return fail(SLHIP_ERR_INVALID, "draft_verify: bad size");
    const int64_t chunks = (V + kChunk - 1) / kChunk;
    if (B > 65536 || V > kMaxVocab || T * chunks * 2 > 0xFFFFFF || B * chunks > 0xFFFFFF)
        return fail(SLHIP_ERR_UNSUPPORTED, "draft_verify: too many requests, rows or tokens of the vocabulary");
    return SLHIP_OK;
}

template <int DT> static int launch(const DraftArgs& a, hipStream_t st)
{
    const int64_t rows = a.T * a.chunks;
    if (rows > 0) {
        if (a.draft)
            draft_stats<DT, true><<<static_cast<unsigned>(rows * 2), kThreads, 0, st>>>(a);
        else
            draft_stats<DT, false><<<static_cast<unsigned>(rows), kThreads, 0, st>>>(a);
        const int e = check_launch("draft_stats");
        if (e) return e;
    }
    draft_decide<DT><<<static_cast<unsigned>(a.B), kDecide, 0, st>>>(a);
    int e = check_launch("draft_decide");
    if (e) return e;
    draft_sums<DT><<<static_cast<unsigned>(a.B * a.chunks), kThreads, 0, st>>>(a);
    e = check_launch("draft_sums");
    if (e) return e;
    draft_pick<DT><<<static_cast<unsigned>(a.B), kThreads, 0, st>>>(a);
    return check_launch("draft_pick");
}

}  // namespace slhip

using namespace slhip;

extern "C" SLHIP_API int64_t slhip_draft_verify_work_bytes(int64_t requests, int64_t tokens, int64_t vocab)
{
    if (check_sizes(requests, tokens, vocab)) return -1;
    return work_of(requests, tokens, (vocab + kChunk - 1) / kChunk);
}

extern "C" SLHIP_API int slhip_draft_verify(int dtype, const void* target, int64_t target_stride, const void* draft, int64_t draft_stride,
                                            const slhip_drafts* d, void* work, int64_t work_bytes, slhip_stream stream)
{
    if (!d) return fail(SLHIP_ERR_INVALID, "draft_verify: arguments are null");
    if (dtype != SLHIP_F32 && dtype != SLHIP_BF16) return fail(SLHIP_ERR_UNSUPPORTED, "draft_verify: dtype %d not supported", dtype);
    int e = check_sizes(d->requests, d->tokens, d->vocab);
    if (e) return e;
    if (d->out_stride < 0 || d->out_stride > 0x7FFFFFFF) return fail(SLHIP_ERR_INVALID, "draft_verify: bad stride of the tokens");
    if (target_stride < d->vocab || (draft && draft_stride < d->vocab))
        return fail(SLHIP_ERR_INVALID, "draft_verify: a row stride is smaller than the vocabulary");
    if (d->requests == 0) return SLHIP_OK;
    if (!d->starts || !d->n_out || (d->out_stride > 0 && !d->out)) return fail(SLHIP_ERR_INVALID, "draft_verify: starts, out and n_out are required");
    if (d->tokens > 0 && (!target || !d->ids || !d->accept || !d->sample))
        return fail(SLHIP_ERR_INVALID, "draft_verify: target, ids, accept and sample are required");
    const int64_t chunks = (d->vocab + kChunk - 1) / kChunk, need = work_of(d->requests, d->tokens, chunks);
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
    a.chunks = static_cast<int32_t>(chunks);
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
    a.sums = reinterpret_cast<double*>(reinterpret_cast<char*>(a.picks) + round16(a.B * static_cast<int64_t>(sizeof(Pick))));
    e = error_word(&a.err);
    if (e) return e;
    return dtype == SLHIP_F32 ? launch<SLHIP_F32>(a, to_stream(stream)) : launch<SLHIP_BF16>(a, to_stream(stream));
}
