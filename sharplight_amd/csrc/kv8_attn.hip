// Entry points of the attention over the 8-bit paged cache: checks, and what a call launches (kernels: kv8_attn.hpp).
#include "kv8_attn.hpp"

namespace slhip {

template <> int kv8_attn_launch<SLHIP_F32, SLHIP_KV8_I8>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_F32, SLHIP_KV8_E4M3>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_I8>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_E4M3>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);

constexpr int64_t kWaveUnits = 1024;  // key ranges of a few-row launch, over all heads
constexpr int64_t kBlockUnits = 512;  // row tiles and key ranges of a many-row launch, over all heads
constexpr int64_t kMaxSplits = 64;

// The launches of a call over T rows of B requests. Few-row waves take a request whose rows fit one or two matrix tiles
// (16 or 32 rows a K/V head): its keys are then read once by single waves. Everything else goes to thread blocks that share
// key tiles among 64 or 128 rows. Where the host cannot tell (max_new unknown or large, several requests) both are launched
// and each leaves the other's requests alone.
static Kv8AttnPlan make_plan(int dtype, const Kv8Dev& c, int64_t G, int64_t max_new)
{
    Kv8AttnPlan p{};
    const int64_t T = c.T, B = c.B, heads = c.heads, most = max_new > 0 && max_new < T ? max_new : T, rows = most * G;
    const int64_t dp = c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256;
    if (rows <= 16) {
        p.wave_rows = 16;
    } else if (rows <= 32 && dp <= 128) {  // 256 dims of two row tiles do not fit the registers
        p.wave_rows = 32;
    } else {
        p.blocks = true;
        p.wave_rows = G <= 16 && B > 1 ? 16 : 0;
    }
    if (p.wave_rows) {
        p.units = static_cast<int32_t>((kWaveUnits + heads - 1) / heads);
        p.wave_grid = (p.units + B) * heads;
        p.work_bytes = 2 * p.units * heads * (p.wave_rows * dp + p.wave_rows * 2) * 4;
    }
    p.splits = 1;
    if (p.blocks) {
        p.block_rows = dtype == SLHIP_F32 || dp == 256 ? 64 : 128;
        p.tile_tokens = static_cast<int32_t>(p.block_rows / G);
        p.block_items = item_count(T, B, p.tile_tokens, 1);
        const int64_t pairs = p.block_items * heads, longest = (c.bps << c.shift) / (4 * kTile) + 1;
        int64_t s = pairs < kBlockUnits ? (kBlockUnits + pairs - 1) / pairs : 1;
        if (s > kMaxSplits) s = kMaxSplits;
        if (s > longest) s = longest;
        p.splits = static_cast<int32_t>(s);
        const int64_t bytes = s > 1 ? pairs * s * (p.block_rows * dp + p.block_rows * 2) * 4 : 0;
        if (bytes > p.work_bytes) p.work_bytes = bytes;
    }
    return p;
}

static int check_heads(int64_t q_heads, const Kv8Dev& c)
{
    if (q_heads < 1 || q_heads % c.heads != 0)
        return fail(SLHIP_ERR_INVALID, "kv8_attention: %lld query heads are not a multiple of %d K/V heads", static_cast<long long>(q_heads), c.heads);
    if (q_heads / c.heads > 64) return fail(SLHIP_ERR_UNSUPPORTED, "kv8_attention: more than 64 query heads for a K/V head");
    return SLHIP_OK;
}

}  // namespace slhip

using namespace slhip;

extern "C" SLHIP_API int64_t slhip_kv8_attention_work_bytes(int64_t q_heads, const slhip_kv8_cache* cache,
                                                            const slhip_kv8_batch* batch, int64_t max_new)
{
    Kv8Dev c;
    if (make_kv8("kv8_attention", cache, batch, &c) || check_heads(q_heads, c)) return -1;
    if (c.B == 0 || c.T == 0) return 0;
    const int64_t a = make_plan(SLHIP_F32, c, q_heads / c.heads, max_new).work_bytes;
    const int64_t b = make_plan(SLHIP_BF16, c, q_heads / c.heads, max_new).work_bytes;
    return a > b ? a : b;
}

extern "C" SLHIP_API int slhip_kv8_attention(int dtype, const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t q_heads,
                                             void* y, int64_t y_stride_t, int64_t y_stride_h, const slhip_kv8_cache* cache,
                                             const slhip_kv8_batch* batch, const slhip_kv8_attn* cfg, void* work,
                                             int64_t work_bytes, slhip_stream stream)
{
    Kv8AttnArgs a{};
    int e = make_kv8("kv8_attention", cache, batch, &a.c);
    if (e) return e;
    if (dtype != SLHIP_F32 && dtype != SLHIP_BF16) return fail(SLHIP_ERR_UNSUPPORTED, "kv8_attention: dtype %d not supported", dtype);
    if (!cfg) return fail(SLHIP_ERR_INVALID, "kv8_attention: cfg is required");
    e = check_heads(q_heads, a.c);
    if (e) return e;
    if (!(cfg->softcap >= 0.0f) || cfg->window < 0 || cfg->max_new < 0 || !(cfg->scale - cfg->scale == 0.0f) || !(cfg->softcap - cfg->softcap == 0.0f))
        return fail(SLHIP_ERR_INVALID, "kv8_attention: scale and softcap must be finite, softcap, window and max_new not negative");
    if (a.c.B == 0 || a.c.T == 0) return SLHIP_OK;
    if (!q || !y) return fail(SLHIP_ERR_INVALID, "kv8_attention: q and y are required");
    if (q_stride_h < a.c.D || y_stride_h < a.c.D || q_stride_t < 0 || y_stride_t < 0)
        return fail(SLHIP_ERR_INVALID, "kv8_attention: a head stride is smaller than the head, or a stride is negative");
    a.q = q;
    a.y = y;
    a.qt = q_stride_t;
    a.qh = q_stride_h;
    a.yt = y_stride_t;
    a.yh = y_stride_h;
    a.G = static_cast<int32_t>(q_heads / a.c.heads);
    a.scale = cfg->scale;
    a.cap = cfg->softcap;
    a.window = cfg->window > 0x7FFFFFFF ? 0 : static_cast<int32_t>(cfg->window);  // no context is that long
    a.slopes = cfg->slopes;
    a.part = static_cast<float*>(work);
    const int64_t most = cfg->max_new > 0 && cfg->max_new < a.c.T ? cfg->max_new : a.c.T;
    if (most * a.G > 0x7FFFFFFF) return fail(SLHIP_ERR_UNSUPPORTED, "kv8_attention: too many query rows");
    a.max_rows = static_cast<int32_t>(most * a.G);
    a.strict = true;
    const Kv8AttnPlan p = make_plan(dtype, a.c, a.G, cfg->max_new);
    if (p.work_bytes > 0 && (!work || !aligned16(work) || work_bytes < p.work_bytes))
        return fail(SLHIP_ERR_INVALID, "kv8_attention: the workspace has %lld bytes, %lld are needed (16-byte aligned)",
                    static_cast<long long>(work ? work_bytes : 0), static_cast<long long>(p.work_bytes));
    if (p.wave_grid > 0x7FFFFFFF || p.block_items * p.splits * a.c.heads > 0x7FFFFFFF)
        return fail(SLHIP_ERR_UNSUPPORTED, "kv8_attention: too many tiles");
    e = error_word(&a.c.err);
    if (e) return e;
    hipStream_t st = to_stream(stream);
    if (dtype == SLHIP_F32) {
        if (cache->format == SLHIP_KV8_I8) return kv8_attn_launch<SLHIP_F32, SLHIP_KV8_I8>(a, p, st);
        return kv8_attn_launch<SLHIP_F32, SLHIP_KV8_E4M3>(a, p, st);
    }
    if (cache->format == SLHIP_KV8_I8) return kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_I8>(a, p, st);
    return kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_E4M3>(a, p, st);
}
