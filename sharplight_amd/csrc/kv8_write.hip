// Write of a step's K and V into the 8-bit paged cache (slhip_kv8_write).
//
// Mathematics: a block and head's scale is a power of two 2^e (e >= -40), the smallest that holds the largest value:
// amax <= Q 2^e with Q = 127 (int8) or 448 (E4M3). x / 2^e is then exact and a code is one rounding (to nearest even) of
// it, so every implementation gets the same bits; a scale that grows does so by 2^d, d >= 1, and the codes that are there
// already are rounded by that factor. The exponent comes from the bits of amax: amax = 1.f * 2^x is at most Q 2^e for
// e = x - 8 (E4M3, Q = 1.75 * 2^8) or x - 6 (int8, Q = 1.984375 * 2^6), plus one where 1.f is above that leading part.
//
// Layout: one work item is (request, block, head, K or V), 16 tokens of it a wave: block_size / 16 waves share an item's
// largest value through LDS (none for blocks of 16). A wave holds its 16 tokens in registers between the maximum and the
// codes, so every value is read once. K goes [token][D]: a lane takes 8 values of a token (one 16-byte load of bf16) and
// stores 8 codes. V goes [D][16 tokens]: a lane takes a pair of dims of all 16 tokens (4-byte loads that cover a token's
// row between them) and stores 16 + 16 bytes, so neither needs a transpose. What bounds it: HBM for a prompt, launch and
// the chain starts -> table -> scale for a decode step.
// Measured, 8 heads of 128, bf16 to E4M3: a prompt of 8192 tokens 12.5 us (50 MB, 4.0 TB/s), one token of 64 requests 5.0 us.
// All of an item's loads are issued before the first value is used (before that 15.2 us): the table entry and the old codes
// and scale wait behind them.
#include "kv8.hpp"

namespace slhip {

struct Kv8WriteArgs {
    Kv8Dev c;
    const void* x[2];
    int64_t st[2], sh[2];
    int64_t tile, extra;  // items by blocks (block_size, 2) or by tokens (1, 0)
    int64_t items;        // thread blocks behind them look for requests that do not fit
    int32_t chunks;       // D / 8, and its reciprocal: n / chunks = n * inverse >> 16 for n < 512
    int32_t inverse;
};

constexpr int kLeastExp = -40, kMostExp = 40;

template <int FMT> struct Code8;

template <> struct Code8<SLHIP_KV8_E4M3> {
    static constexpr uint32_t kLead = 0x600000u;  // fraction bits of 1.75
    static constexpr int kTop = 8;
    // |v * inv| <= 448 by the choice of the scale, so nothing is clamped; + 0 turns -0 into +0.
    __device__ static __forceinline__ uint32_t pack(const float* v, float inv)
    {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(fmaf(v[0], inv, 0.0f), fmaf(v[1], inv, 0.0f), 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(fmaf(v[2], inv, 0.0f), fmaf(v[3], inv, 0.0f), w, true);
        return static_cast<uint32_t>(w);
    }
    __device__ static __forceinline__ void unpack(uint32_t w, float* f)
    {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
    }
};

template <> struct Code8<SLHIP_KV8_I8> {
    static constexpr uint32_t kLead = 0x7E0000u;  // fraction bits of 1.984375
    static constexpr int kTop = 6;
    __device__ static __forceinline__ uint32_t pack(const float* v, float inv)
    {
        // 1.5 * 2^23 + code: the sum rounds to a whole number, ties to even, whose low byte is the code
        uint32_t u[4];
        for (int i = 0; i < 4; i++) u[i] = __float_as_uint(fmaf(v[i], inv, 12582912.0f));
        const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000C0Cu);
        return lo | hi;
    }
    __device__ static __forceinline__ void unpack(uint32_t w, float* f)
    {
        for (int i = 0; i < 4; i++) f[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
    }
};

// The scale of a largest value given as its bits (sign cleared; above 0x7F800000 where a NaN is among the values).
template <int FMT> __device__ __forceinline__ float scale_of(uint32_t amax)
{
    int e = static_cast<int>(amax >> 23) - 127 - Code8<FMT>::kTop + ((amax & 0x7FFFFFu) > Code8<FMT>::kLead);
    e = max(e, kLeastExp);
    return e > kMostExp ? __uint_as_float(0x7FC00000u) : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// 1 / s of a power of two.
__device__ __forceinline__ float inverse(float s) { return __uint_as_float(0x7F000000u - __float_as_uint(s)); }

// Largest of the wave, in lane 63's view made wave-uniform: within rows of 16 lanes, then row by row.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v)
{
    v = dpp_umax_step<0xB1>(v);   // quad_perm [1,0,3,2]
    v = dpp_umax_step<0x4E>(v);   // quad_perm [2,3,0,1]
    v = dpp_umax_step<0x141>(v);  // row_half_mirror
    v = dpp_umax_step<0x140>(v);  // row_mirror
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x142, 0xA, 0xF, false)));  // row_bcast:15
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x143, 0xC, 0xF, false)));  // row_bcast:31
    return __builtin_amdgcn_readlane(static_cast<int>(v), 63);
}

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// The bytes of dword j (tokens 4j .. 4j+3 of a wave's 16) that lie in tokens [a, b).
__device__ __forceinline__ uint32_t byte_mask(int j, int a, int b)
{
    const int lo = min(max(a - 4 * j, 0), 4), hi = min(max(b - 4 * j, 0), 4);
    const uint32_t upto_hi = hi == 4 ? 0xFFFFFFFFu : (1u << (8 * hi)) - 1, upto_lo = lo == 4 ? 0xFFFFFFFFu : (1u << (8 * lo)) - 1;
    return upto_hi & ~upto_lo;
}

// 16 bytes of values from element i on; VEC: they may be loaded at once.
template <int DT, bool VEC> __device__ __forceinline__ uint4 load_word(const void* p, int64_t i)
{
    if constexpr (VEC) return *reinterpret_cast<const uint4*>(static_cast<const char*>(p) + i * Vec<DT>::BYTES);
    float f[Vec<DT>::N];
#pragma unroll
    for (int j = 0; j < Vec<DT>::N; j++) f[j] = Vec<DT>::load1(p, i + j);
    return Vec<DT>::pack(f);  // the same bits again (a NaN's may change: it stays one)
}

// Two values next to each other.
template <int DT> struct Pair;
template <> struct Pair<SLHIP_F32> {
    typedef float2 T;
    template <bool VEC> __device__ static __forceinline__ T load(const void* p, int64_t i)
    {
        const float* f = static_cast<const float*>(p) + i;
        if constexpr (VEC) return *reinterpret_cast<const float2*>(f);
        return make_float2(f[0], f[1]);
    }
    __device__ static __forceinline__ float2 unpack(T v) { return v; }
};
template <> struct Pair<SLHIP_BF16> {
    typedef uint32_t T;
    template <bool VEC> __device__ static __forceinline__ T load(const void* p, int64_t i)
    {
        const uint16_t* f = static_cast<const uint16_t*>(p) + i;
        if constexpr (VEC) return *reinterpret_cast<const uint32_t*>(f);
        return f[0] | static_cast<uint32_t>(f[1]) << 16;
    }
    __device__ static __forceinline__ float2 unpack(T v) { return make_float2(bf16_lo(v), bf16_hi(v)); }
};

// DP: head dims up to 64, 128 or 256; VEC: rows that 16-byte (K) and pair (V) loads can read.
template <int DT, int FMT, int DP, bool VEC>
__global__ __launch_bounds__(1024) void kv8_write(Kv8WriteArgs a)
{
    const Kv8Dev& c = a.c;
    __shared__ uint32_t s_max[16];
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int bs = 1 << c.shift, wpi = bs >> 4;  // waves per item
    // A request that does not fit may have no item: one that begins behind the last row, or brings none. So each is looked at here,
    // by a thread.
    if (blockIdx.x >= a.items) {
        const int64_t i = (blockIdx.x - a.items) * blockDim.x + threadIdx.x;
        if (blockIdx.y == 0 && i < c.B) {
            const Kv8Request r = kv8_request(c, static_cast<int32_t>(i));
            if (r.bad) raise_request(c, static_cast<int32_t>(i), r);
        }
        return;
    }
    const Kv8Item it = kv8_find(c, blockIdx.x, a.tile, a.extra);
    const Kv8Request& r = it.r;
    const int pair = static_cast<int>(blockIdx.y) * (static_cast<int>(blockDim.x >> 6) / wpi) + wave / wpi, sub = wave % wpi;
    // everything above is the same for all of the thread block: nothing is left waiting at the barrier below
    const int b0 = r.past >> c.shift;
    if (r.n == 0 || it.piece < 0 || it.piece > ((r.past + r.n - 1) >> c.shift) - b0) return;
    const int tb = b0 + static_cast<int>(it.piece), p0 = tb << c.shift;  // the block's place in the table, its first position
    const int32_t block = r.table[tb];  // (on its way while the values are)
    const bool mine = pair < 2 * c.heads;
    const int kv = pair & 1, head = mine ? pair >> 1 : 0, D = c.D;
    const bool fresh = r.past <= p0;
    // the new tokens of this wave's 16, [na, nb), and the row of the first of the 16 (which may be a row before the request's)
    const int q0 = p0 + sub * 16;
    const int na = min(max(r.past - q0, 0), 16), nb = min(max(r.past + r.n - q0, 0), 16);
    const int64_t row0 = static_cast<int64_t>(r.first) + q0 - r.past;
    const void* x = a.x[kv];
    const int64_t xs = a.st[kv], xh = head * a.sh[kv];

    constexpr int KR = DP / 32, VR = (DP + 127) / 128;  // rounds of a lane: 8 values of K, 2 x 16 of V
    float f[KR * 8 > VR * 32 ? KR * 8 : VR * 32];
#pragma unroll
    for (float& v : f) v = 0.0f;
    // All loads go out before the first value is used: rows that are not the request's are read as one of its rows and dropped.
    if (mine && nb > na) {
        if (kv == 0) {
            constexpr int W = Vec<DT>::BYTES / 2;  // 16-byte words of 8 values
            uint4 raw[KR][W];
#pragma unroll
            for (int o = 0; o < KR; o++) {
                const int i = lane + 64 * o, row = i * a.inverse >> 16, t = min(max(row, na), nb - 1);  // 16 tokens of a.chunks
                const int64_t e = (row0 + t) * xs + xh + (i - row * a.chunks) * 8;
#pragma unroll
                for (int w = 0; w < W; w++) raw[o][w] = load_word<DT, VEC>(x, e + w * Vec<DT>::N);
            }
#pragma unroll
            for (int o = 0; o < KR; o++) {
                const int t = (lane + 64 * o) * a.inverse >> 16;
#pragma unroll
                for (int w = 0; w < W; w++) Vec<DT>::unpack(raw[o][w], f + 8 * o + w * Vec<DT>::N);
#pragma unroll
                for (int j = 0; j < 8; j++) f[8 * o + j] = t >= na && t < nb ? f[8 * o + j] : 0.0f;
            }
        } else {
            typename Pair<DT>::T raw[VR][16];
#pragma unroll
            for (int o = 0; o < VR; o++) {
                const int d = min(2 * (lane + 64 * o), D - 2);
#pragma unroll
                for (int t = 0; t < 16; t++) raw[o][t] = Pair<DT>::template load<VEC>(x, (row0 + min(max(t, na), nb - 1)) * xs + xh + d);
            }
#pragma unroll
            for (int o = 0; o < VR; o++)
#pragma unroll
                for (int t = 0; t < 16; t++) {
                    const float2 w = Pair<DT>::unpack(raw[o][t]);
                    f[32 * o + t] = t >= na && t < nb ? w.x : 0.0f;
                    f[32 * o + 16 + t] = t >= na && t < nb ? w.y : 0.0f;
                }
        }
    }
    uint32_t top = 0;
    if (block < 0 || block >= c.blocks) {  // the same for all of the thread block
        if (threadIdx.x == 0 && blockIdx.y == 0) raise_block(c, r.first, r.slot, max(p0, r.past), block);
        return;
    }
    float* sp = (kv ? c.vs : c.ks) + static_cast<int64_t>(block) * c.heads + head;
    const float s0 = fresh ? 0.0f : *sp;
    uint8_t* base = (kv ? c.v : c.k) + ((static_cast<int64_t>(block) * c.heads + head) * bs + sub * 16) * D;
    uint4 was[VR][2];  // V's codes that are there already
    if (mine && kv == 1 && !fresh) {
#pragma unroll
        for (int o = 0; o < VR; o++)
#pragma unroll
            for (int e = 0; e < 2; e++) was[o][e] = *reinterpret_cast<const uint4*>(base + (2 * (lane + 64 * o) < D ? 2 * (lane + 64 * o) + e : 0) * 16);
    }
    if (mine && nb > na) {
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof f / sizeof f[0]); j++)
            if (j < (kv == 0 ? KR * 8 : VR * 32)) top = max(top, abs_bits(f[j]));
        top = wave_umax(top);
    }
    if (wpi > 1) {
        if (lane == 0) s_max[wave] = top;
        __syncthreads();
        for (int w = 0; w < wpi; w++) top = max(top, s_max[wave - sub + w]);
    }
    if (!mine) return;
    const float sn = scale_of<FMT>(top);
    const bool lost = sn != sn || s0 != s0;  // a value that no scale holds, now or earlier
    const float s1 = lost ? __uint_as_float(0x7FC00000u) : fmaxf(s0, sn);
    const bool grew = !fresh && !lost && s1 > s0;
    const float inv = lost ? 0.0f : inverse(s1), shrink = grew ? s0 * inv : 1.0f;
    if (sub == 0 && lane == 0) *sp = s1;
    if (!fresh && !grew && nb <= na) return;
    if (lost)
        for (float& v : f) v = 0.0f;
    if (kv == 0) {
#pragma unroll
        for (int o = 0; o < KR; o++) {
            const int at = (lane + 64 * o) * 8, t = (lane + 64 * o) * a.inverse >> 16;
            if (t >= 16) continue;
            uint2* p = reinterpret_cast<uint2*>(base + at);
            if (t >= na && t < nb) {
                *p = make_uint2(Code8<FMT>::pack(f + 8 * o, inv), Code8<FMT>::pack(f + 8 * o + 4, inv));
            } else if (fresh) {
                *p = make_uint2(0, 0);
            } else if (grew) {
                const uint2 w = *p;
                float g[8];
                Code8<FMT>::unpack(w.x, g);
                Code8<FMT>::unpack(w.y, g + 4);
                *p = make_uint2(Code8<FMT>::pack(g, shrink), Code8<FMT>::pack(g + 4, shrink));
            }
        }
    } else {
#pragma unroll
        for (int o = 0; o < VR; o++) {
            const int d = 2 * (lane + 64 * o);
            if (d >= D) continue;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                uint4* p = reinterpret_cast<uint4*>(base + (d + e) * 16);
                uint32_t w[4] = {0, 0, 0, 0};
                if (!fresh) {
                    w[0] = was[o][e].x; w[1] = was[o][e].y; w[2] = was[o][e].z; w[3] = was[o][e].w;
                }
                for (int j = 0; j < 4; j++) {
                    if (grew) {
                        float g[4];
                        Code8<FMT>::unpack(w[j], g);
                        w[j] = Code8<FMT>::pack(g, shrink);
                    }
                    const uint32_t m = byte_mask(j, na, nb);
                    w[j] = (nb > na ? Code8<FMT>::pack(f + 32 * o + 16 * e + 4 * j, inv) & m : 0) | (w[j] & ~m);
                }
                *p = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

int make_kv8(const char* op, const slhip_kv8_cache* c, const slhip_kv8_batch* b, Kv8Dev* out)
{
    if (!c || !b) return fail(SLHIP_ERR_INVALID, "%s: cache and batch are required", op);
    if (c->format != SLHIP_KV8_I8 && c->format != SLHIP_KV8_E4M3) return fail(SLHIP_ERR_UNSUPPORTED, "%s: cache format %d not supported", op, c->format);
    if (c->blocks < 0 || c->heads < 1 || c->head_dim < 1 || b->requests < 0 || b->tokens < 0 || b->page_slots < 0 || b->blocks_per_slot < 0)
        return fail(SLHIP_ERR_INVALID, "%s: bad size", op);
    if (c->head_dim % 16 != 0 || c->head_dim > 256)
        return fail(SLHIP_ERR_UNSUPPORTED, "%s: head dim %lld is not a multiple of 16 up to 256", op, static_cast<long long>(c->head_dim));
    int shift = 4;
    while (shift < 8 && (1 << shift) != c->block_size) shift++;
    if ((1 << shift) != c->block_size)
        return fail(SLHIP_ERR_UNSUPPORTED, "%s: block size %lld is not 16, 32, 64, 128 or 256", op, static_cast<long long>(c->block_size));
    // positions are 32-bit, and tiles reach past a request's last one
    if (b->blocks_per_slot > (0x7FFFFFFFll - 65536) >> shift || b->tokens > 0x7FFFFFFFll - 65536 || c->blocks > 0x7FFFFFFFll ||
        b->requests > 65536 || c->heads > 4096)
        return fail(SLHIP_ERR_UNSUPPORTED, "%s: too many tokens, blocks, requests or heads", op);
    if (b->requests > 0 && b->tokens > 0) {
        if (!b->starts || !b->past || !b->pages) return fail(SLHIP_ERR_INVALID, "%s: starts, past and pages are required", op);
        if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(SLHIP_ERR_INVALID, "%s: the cache's codes and scales are required", op);
        if (!aligned16(c->k) || !aligned16(c->v)) return fail(SLHIP_ERR_INVALID, "%s: codes must be 16-byte aligned", op);
        if (c->blocks == 0) return fail(SLHIP_ERR_INVALID, "%s: the cache has no blocks", op);
    }
    *out = Kv8Dev{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale, static_cast<int32_t>(c->blocks), shift,
                  static_cast<int32_t>(c->heads), static_cast<int32_t>(c->head_dim), static_cast<int32_t>(b->requests), b->tokens,
                  b->starts, b->past, b->slots, b->pages, b->page_slots, b->blocks_per_slot, nullptr};
    return SLHIP_OK;
}

template <int DT, int FMT, int DP> static int launch(const Kv8WriteArgs& a, bool vec, dim3 grid, unsigned threads, hipStream_t st)
{
    if (vec) kv8_write<DT, FMT, DP, true><<<grid, threads, 0, st>>>(a);
    else kv8_write<DT, FMT, DP, false><<<grid, threads, 0, st>>>(a);
    return check_launch("kv8_write");
}

template <int DT, int FMT> static int by_dim(const Kv8WriteArgs& a, bool vec, dim3 grid, unsigned threads, hipStream_t st)
{
    if (a.c.D <= 64) return launch<DT, FMT, 64>(a, vec, grid, threads, st);
    if (a.c.D <= 128) return launch<DT, FMT, 128>(a, vec, grid, threads, st);
    return launch<DT, FMT, 256>(a, vec, grid, threads, st);
}

}  // namespace slhip

using namespace slhip;

extern "C" SLHIP_API int slhip_kv8_write(int dtype, const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v,
                                         int64_t v_stride_t, int64_t v_stride_h, const slhip_kv8_cache* cache,
                                         const slhip_kv8_batch* batch, slhip_stream stream)
{
    Kv8WriteArgs a{};
    const int e = make_kv8("kv8_write", cache, batch, &a.c);
    if (e) return e;
    if (dtype != SLHIP_F32 && dtype != SLHIP_BF16) return fail(SLHIP_ERR_UNSUPPORTED, "kv8_write: dtype %d not supported", dtype);
    if (a.c.B == 0 || a.c.T == 0) return SLHIP_OK;
    if (!k || !v) return fail(SLHIP_ERR_INVALID, "kv8_write: k and v are required");
    const int64_t size = dtype == SLHIP_F32 ? 4 : 2, D = a.c.D;
    if (k_stride_h < D || v_stride_h < D || k_stride_t < 0 || v_stride_t < 0) return fail(SLHIP_ERR_INVALID, "kv8_write: a head stride is smaller than the head, or a stride is negative");
    a.chunks = a.c.D / 8;
    a.inverse = (65536 + a.chunks - 1) / a.chunks;  // off by less than chunks / 65536 each: 512 * 32 of them stay below one
    a.x[0] = k;
    a.x[1] = v;
    a.st[0] = k_stride_t;
    a.st[1] = v_stride_t;
    a.sh[0] = k_stride_h;
    a.sh[1] = v_stride_h;
    const int64_t n16 = 16 / size;  // values of 16 bytes
    const bool vec = aligned16(k) && reinterpret_cast<uintptr_t>(v) % (2 * size) == 0 && k_stride_t % n16 == 0 &&
                     k_stride_h % n16 == 0 && v_stride_t % 2 == 0 && v_stride_h % 2 == 0;
    // Items by blocks, or by rows where that is fewer: a decode step has one row and one block a request.
    const int64_t bs = int64_t{1} << a.c.shift;
    const bool by_block = item_count(a.c.T, a.c.B, bs, 2) < a.c.T;
    a.tile = by_block ? bs : 1;
    a.extra = by_block ? 2 : 0;
    const int64_t items = by_block ? item_count(a.c.T, a.c.B, bs, 2) : a.c.T;
    const unsigned wpi = static_cast<unsigned>(bs >> 4), threads = 64 * (wpi < 4 ? 4 : wpi), per = threads / 64 / wpi;
    a.items = items;
    const int64_t blocks = items + (a.c.B + threads - 1) / threads;
    if (blocks * threads > 0xFFFFFFFFll) return fail(SLHIP_ERR_UNSUPPORTED, "kv8_write: too many rows");  // a launch's threads
    const dim3 grid(static_cast<unsigned>(blocks), (2 * a.c.heads + per - 1) / per);
    const int w = error_word(&a.c.err);
    if (w) return w;
    hipStream_t st = to_stream(stream);
    if (dtype == SLHIP_F32) {
        if (cache->format == SLHIP_KV8_I8) return by_dim<SLHIP_F32, SLHIP_KV8_I8>(a, vec, grid, threads, st);
        return by_dim<SLHIP_F32, SLHIP_KV8_E4M3>(a, vec, grid, threads, st);
    }
    if (cache->format == SLHIP_KV8_I8) return by_dim<SLHIP_BF16, SLHIP_KV8_I8>(a, vec, grid, threads, st);
    return by_dim<SLHIP_BF16, SLHIP_KV8_E4M3>(a, vec, grid, threads, st);
}
