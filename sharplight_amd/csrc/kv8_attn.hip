// Entry points of the attention over the 8-bit paged cache: checks, and what a call launches (kernels: kv8_attn.hpp).
#include <float.h>
#include <math.h>

#include "kv8_attn.hpp"

namespace slhip {

template <> int kv8_attn_launch<SLHIP_F32, SLHIP_KV8_I8, kPlain>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_F32, SLHIP_KV8_E4M3, kPlain>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_I8, kPlain>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_E4M3, kPlain>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_F32, SLHIP_KV8_I8, kReshaped>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_F32, SLHIP_KV8_E4M3, kReshaped>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_I8, kReshaped>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_E4M3, kReshaped>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_I8, kFarCap>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);
template <> int kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_E4M3, kFarCap>(const Kv8AttnArgs&, const Kv8AttnPlan&, hipStream_t);

template <int DT, int FMT> static int launch(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st)
{
    if constexpr (DT == SLHIP_BF16) {
        if (a.cap > kFastCap) return kv8_attn_launch<DT, FMT, kFarCap>(a, p, st);
    }
    const bool reshaped = a.cap > 0.0f || a.slopes || !(a.factor > 0.0f);
    return reshaped ? kv8_attn_launch<DT, FMT, kReshaped>(a, p, st) : kv8_attn_launch<DT, FMT, kPlain>(a, p, st);
}

// Two thread blocks a CU: the registers of the line's kernels leave places for so many. Those of 256 dims have one, and half the
// workers; those of 32 rows (296 to 430 registers) have one too, and take the line's pieces in two rounds.
constexpr int64_t kWorkers = 512;
// Row tiles and key ranges of the many-row work, over all heads. With 256, 512, 1024: 5 requests of 77 to 611 new tokens and
// up to 1500 older ones, 12 heads of 64, f32 67, 54, 52 us; a prompt of 1024, 32 query heads of 128 on 8, bf16 34, 32, 42 us;
// 128 tokens on 30000, the same heads 118, 99, 111 us.
constexpr int64_t kBlockUnits = 512;
// Up to here (and up to 64 requests) the cuts go by the lengths, whose scan costs some 3 us in the kernel and in the join: 128
// tokens on 30000, as above, 103 us with equal cuts and 95 so, 7 requests of up to 74700 82 and 65 us; but the prompt of 1024 33
// and 37 us, the 5 requests 53 and 60.
constexpr int64_t kFewTiles = kBlockUnits / 4;

// Floats of the sums of `rows` rows; workers of the line; rows of a row tile; ranges of a head besides its tiles, and of a tile (cut
// into no ranges of less than 8 key tiles, see below).
static int64_t part_floats(int64_t dp, int64_t rows) { return rows * dp + rows * 2; }
static int64_t workers_of(int64_t dp) { return dp == 256 ? kWorkers / 2 : kWorkers; }
static int64_t tile_rows(int dtype, int64_t dp)
{
    return 16 * block_waves(static_cast<int>(dp)) * block_tiles(dtype == SLHIP_F32, static_cast<int>(dp));
}
static int64_t share_of(int64_t heads) { return (kBlockUnits + heads - 1) / heads; }
static int64_t splits_of(int64_t pairs, int64_t seen)
{
    const int64_t s = (kBlockUnits + pairs - 1) / pairs, most = seen / (8 * kTile);
    return s < most ? s : most;
}

// What a call over T rows of B requests launches. Few-row work takes a request whose rows fit one or two matrix tiles (16
// or 32 rows a K/V head): its keys are then read once by single waves. Everything else goes to thread blocks that share
// key tiles among 64 or 128 rows. Where the host cannot tell (max_new unknown or large, several requests) one launch holds
// both (of 256 dims two do) and each leaves the other's requests alone. Fills what of `a` the kernels go by; returns the workspace's bytes.
static int64_t make_plan(int dtype, int64_t G, int64_t max_new, Kv8AttnArgs* a, Kv8AttnPlan* p)
{
    const Kv8Dev& c = a->c;
    const int64_t T = c.T, B = c.B, heads = c.heads, most = max_new > 0 && max_new < T ? max_new : T, rows = most * G;
    const int64_t dp = c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256;
    *p = Kv8AttnPlan{};
    if (rows <= 16) p->wave_tiles = 1;
    else if (rows <= 32 && dp <= 128) p->wave_tiles = 2;  // 256 dims of two tiles do not fit the registers
    else p->blocks = true;
    if (p->blocks && G <= 16 && B > 1) p->wave_tiles = 1;
    const int64_t limit = rows < 0x7FFFFFFF ? rows : 0x7FFFFFFF, few = 16 * p->wave_tiles;
    a->max_rows = static_cast<int32_t>(p->blocks && few < limit ? few : limit);
    a->strict = !p->blocks;
    a->block_min = static_cast<int32_t>(few);
    a->block_max = static_cast<int32_t>(limit);
    // tokens that a row can see at most, and the others of its tile or request
    const int64_t tokens = c.bps << c.shift, seen = a->window > 0 && a->window + most + kTile < tokens ? a->window + most + kTile : tokens;
    int64_t bytes = 0;
    a->direct = false;
    if (p->wave_tiles) {
        // Each head gets a thread block of its own, and no second launch, where no row can see far: up to 4 rounds (1024
        // tokens), and the more the more heads there are to fill the machine while the longest run. (8 K/V heads of 128, on
        // the line and so: 8 requests of up to 2001 tokens 15 and 16 us, 64 of them 34 and 30, 256 of up to 4001 208 and 198, of
        // up to 8001 367 and 394.)
        const int64_t rounds = p->blocks || B * heads < kWorkers ? 4 : B * heads < 2 * kWorkers ? 8 : 16;
        a->direct = seen <= rounds * 4 * kTile;
        p->few_heads = B * heads <= kWorkers;
        a->workers = static_cast<int32_t>(a->direct ? B * heads : workers_of(dp));
        p->by_part = B * heads < 256;
        if (!a->direct) bytes += 2 * a->workers * part_floats(dp, few) * 4;
    }
    a->splits = 1;
    a->share = 0;
    if (p->blocks) {
        const int64_t tile = tile_rows(dtype, dp), floats = part_floats(dp, tile);
        a->tile_tokens = static_cast<int32_t>(tile / G);
        a->items = item_count(T, B, a->tile_tokens, 1);
        a->part2 = a->part + bytes / 4;
        // A range of less than 8 key tiles does not earn its partial sums and the join (a prompt of 400, 32 query heads of 128 on
        // 8, bf16: whole 20 us, in two 22; of 700 27 and 25; 5 requests of 250 to 433, 16 heads of 96 on 2: 22 and 34).
        const int64_t pairs = a->items * heads, most_cuts = seen / (8 * kTile);
        if (most_cuts >= 2 && pairs <= kFewTiles && B <= 64 && a->items * tokens / kTile < 1 << 28) {
            a->share = static_cast<int32_t>(share_of(heads));
            bytes += (a->items + a->share) * heads * floats * 4;
        } else if (most_cuts >= 2 && pairs < kBlockUnits) {
            a->splits = static_cast<int32_t>(splits_of(pairs, seen));
            bytes += pairs * a->splits * floats * 4;
        }
    }
    return bytes;
}

// The most that a call needs whose requests, rows, new tokens and table rows are no more than these: a long prompt fills the machine
// and needs nothing, its shorter end is cut along the keys. Every kind of plan that make_plan may choose, each at its largest.
static int64_t most_work(int dtype, int64_t G, int64_t max_new, const Kv8Dev& c)
{
    const int64_t heads = c.heads, rows = (max_new > 0 && max_new < c.T ? max_new : c.T) * G, tokens = c.bps << c.shift;
    const int64_t dp = c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256;
    const auto few = [&](int64_t tiles) { return tokens <= 4 * 4 * kTile ? 0 : 2 * workers_of(dp) * part_floats(dp, 16 * tiles) * 4; };
    int64_t most = G <= 16 ? few(1) : 0;
    if (dp <= 128 && G <= 32 && rows > 16 && few(2) > most) most = few(2);
    if (rows <= (dp <= 128 ? 32 : 16)) return most;
    const int64_t tile = tile_rows(dtype, dp), all = item_count(c.T, c.B, tile / G, 1);
    const int64_t beside = G <= 16 && c.B > 1 ? few(1) : 0;
    for (int64_t items = 1; items <= all && items * heads < kBlockUnits; items++) {
        const int64_t pairs = items * heads, whole = pairs <= kFewTiles ? pairs + share_of(heads) * heads : 0, cut = pairs * splits_of(pairs, tokens);
        const int64_t bytes = tokens / (8 * kTile) < 2 ? 0 : (whole > cut ? whole : cut) * part_floats(dp, tile) * 4;
        if (bytes + beside > most) most = bytes + beside;
    }
    return most > beside ? most : beside;
}

static int check_sizes(int64_t q_heads, const Kv8Dev& c)
{
    if (q_heads < 1 || q_heads % c.heads != 0)
        return fail(SLHIP_ERR_INVALID, "kv8_attention: %lld query heads are not a multiple of %d K/V heads", static_cast<long long>(q_heads), c.heads);
    if (q_heads / c.heads > 64) return fail(SLHIP_ERR_UNSUPPORTED, "kv8_attention: more than 64 query heads for a K/V head");
    if (c.B * ((c.bps << c.shift) / (4 * kTile) + 1 + kStart) > 0x7FFFFFFF)  // the line's sums are 32-bit (find_line)
        return fail(SLHIP_ERR_UNSUPPORTED, "kv8_attention: %d requests of up to %lld tokens are too many", c.B, static_cast<long long>(c.bps << c.shift));
    return SLHIP_OK;
}

}  // namespace slhip

using namespace slhip;

extern "C" SLHIP_API int64_t slhip_kv8_attention_work_bytes(int64_t q_heads, const slhip_kv8_cache* cache,
                                                            const slhip_kv8_batch* batch, int64_t max_new)
{
    Kv8Dev c;
    if (make_kv8("kv8_attention", cache, batch, &c) || check_sizes(q_heads, c)) return -1;
    if (c.B == 0 || c.T == 0) return 0;
    const int64_t f32 = most_work(SLHIP_F32, q_heads / c.heads, max_new, c), bf16 = most_work(SLHIP_BF16, q_heads / c.heads, max_new, c);
    return f32 > bf16 ? f32 : bf16;
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
    e = check_sizes(q_heads, a.c);
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
    // A cap above 2^60 counts as none: scores below 2^49 differ by less than 2^-24 of themselves from capped ones, and above that
    // (up to the cap) the largest is alone either way. Of a cap below 2^-60 its inverse counts as 2^60: all scores are 0 to 2^-60.
    // In between 1 / cap times a score's factor stays a normal number.
    a.cap = cfg->softcap > 0x1p60f ? 0.0f : cfg->softcap;
    a.window = cfg->window > 0x7FFFFFFF ? 0 : static_cast<int32_t>(cfg->window);  // no context is that long
    a.slopes = cfg->slopes;
    a.part = static_cast<float*>(work);
    const bool capped = a.cap > 0.0f;
    a.factor = cfg->scale * (!capped ? 1.0f : a.cap < 0x1p-60f ? 0x1p60f : 1.0f / a.cap);
    a.most = capped ? 0x1p86f : FLT_MAX;
    a.lost = capped ? 0x1p-113f : NAN;  // under a cap an infinity is more than the largest number, which is multiplied by that
    Kv8AttnPlan p;
    const int64_t need = make_plan(dtype, a.G, cfg->max_new, &a, &p);
    if (need > 0 && (!work || !aligned16(work) || work_bytes < need))
        return fail(SLHIP_ERR_INVALID, "kv8_attention: the workspace has %lld bytes, %lld are needed (16-byte aligned)",
                    static_cast<long long>(work ? work_bytes : 0), static_cast<long long>(need));
    // A launch has less than 2^32 threads. Row tiles and few-row work are one launch, of 256 dims two (of different thread blocks); the
    // join has two thread blocks a head, or up to 16 for each of fewer than 256 heads and of fewer than kBlockUnits row tiles.
    const int64_t tiles = p.blocks ? (a.items * a.splits + a.share) * a.c.heads : 0, few = p.wave_tiles ? a.workers : 0;
    const bool apart = a.c.D > 128;
    const int64_t threads = tiles * block_threads(apart ? 256 : 128, p.blocks ? 1 : 0) + (apart ? 0 : few * 256);
    const int64_t joins = static_cast<int64_t>(a.c.B) * a.c.heads * 2 + kBlockUnits * 32;
    if (threads > 0xFFFFFFFFll || few * 256 > 0xFFFFFFFFll || joins * 256 > 0xFFFFFFFFll)
        return fail(SLHIP_ERR_UNSUPPORTED, "kv8_attention: too many tiles");
    e = error_word(&a.c.err);
    if (e) return e;
    hipStream_t st = to_stream(stream);
    if (dtype == SLHIP_F32) {
        if (cache->format == SLHIP_KV8_I8) return launch<SLHIP_F32, SLHIP_KV8_I8>(a, p, st);
        return launch<SLHIP_F32, SLHIP_KV8_E4M3>(a, p, st);
    }
    if (cache->format == SLHIP_KV8_I8) return launch<SLHIP_BF16, SLHIP_KV8_I8>(a, p, st);
    return launch<SLHIP_BF16, SLHIP_KV8_E4M3>(a, p, st);
}
