// Host check of the work-item map (sharplight_amd/csrc/kv8_map.hpp): over random steps, every token of every request is
// in exactly one row piece, and every block that a request's tokens touch is exactly one block item, all below item_count.
#include <stdio.h>
#include <stdlib.h>

#include <set>
#include <utility>
#include <vector>

#include "../sharplight_amd/csrc/kv8_map.hpp"

using namespace slhip;

static uint64_t state = 88172645463325252ull;
static uint32_t rnd(uint32_t n) { state ^= state << 13; state ^= state >> 7; state ^= state << 17; return static_cast<uint32_t>(state >> 33) % n; }

int main()
{
    long cases = 0;
    for (int rep = 0; rep < 4000; rep++) {
        const int B = 1 + rnd(rep % 5 == 0 ? 200 : 6);
        const int64_t tile = 1 + rnd(40), bs = 16 << rnd(3);
        std::vector<int64_t> starts{0}, past;
        for (int i = 0; i < B; i++) {
            const uint32_t kind = rnd(4);
            starts.push_back(starts.back() + (kind == 0 ? 0 : kind == 1 ? 1 : rnd(90)));
            past.push_back(rnd(3) ? rnd(200) : bs * rnd(4));
        }
        const int64_t T = starts[B] + rnd(50);  // padding rows
        const auto at = [&](int64_t i) { return starts[i]; };
        std::vector<int> seen(T + 1, 0);
        std::set<std::pair<int64_t, int64_t>> blocks;
        for (int64_t item = 0; item < item_count(T, B, tile, 1); item++) {
            const int64_t i = item_request(at, B, item, tile, 1), n = starts[i + 1] - starts[i];
            const int64_t t0 = (item - item_base(starts[i], i, tile, 1)) * tile;
            if (t0 < 0) return printf("piece before its request\n"), 1;
            for (int64_t t = t0; t < n && t < t0 + tile; t++) seen[starts[i] + t]++;
        }
        for (int64_t t = 0; t < T; t++)
            if (seen[t] != (t < starts[B])) return printf("row %ld in %d pieces\n", long(t), seen[t]), 1;
        for (int by_row = 0; by_row < 2; by_row++) {
            const int64_t tl = by_row ? 1 : bs, ex = by_row ? 0 : 2;
            blocks.clear();
            for (int64_t item = 0; item < (by_row ? T : item_count(T, B, tl, ex)); item++) {
                const int64_t i = item_request(at, B, item, tl, ex), n = starts[i + 1] - starts[i];
                const int64_t piece = item - item_base(starts[i], i, tl, ex), b0 = past[i] / bs;
                if (n == 0 || piece < 0 || piece > (past[i] + n - 1) / bs - b0) continue;
                if (!blocks.insert({i, b0 + piece}).second) return printf("a block twice\n"), 1;
            }
            size_t want = 0;
            for (int i = 0; i < B; i++) {
                const int64_t n = starts[i + 1] - starts[i];
                if (n) want += (past[i] + n - 1) / bs - past[i] / bs + 1;
            }
            if (blocks.size() != want) return printf("%zu blocks of %zu\n", blocks.size(), want), 1;
        }
        cases++;
    }
    // a request that does not fit is seen as such
    if (request_fits(0, 5, 4, 0, 0, 1, 64) || request_fits(-1, 5, 8, 0, 0, 1, 64) || request_fits(5, 4, 8, 0, 0, 1, 64) ||
        request_fits(0, 5, 8, -1, 0, 1, 64) || request_fits(0, 5, 8, 60, 0, 1, 64) || request_fits(0, 5, 8, 0, 1, 1, 64) ||
        request_fits(0, 5, 8, 0, -1, 1, 64) || request_fits(0, 2147483647, 8, 2147483647, 0, 1, 64) || !request_fits(3, 8, 8, 59, 0, 1, 64))
        return printf("request_fits\n"), 1;
    printf("cases %ld\n", cases);
    return 0;
}
