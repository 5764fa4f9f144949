// csrc/kv_visible.h against a count of the keys one by one: which tiles a launch visits, that none is listed
// twice or missed, and which pool rows a block-table entry may stand for.
#include <cstdio>
#include <set>

#include "kv_visible.h"

using namespace ghip;

static int failures = 0;
#define EXPECT(cond, ...)                                  \
    do {                                                   \
        if (!(cond)) {                                     \
            if (failures++ < 20) {                         \
                std::printf("line %d: %s: ", __LINE__, #cond); \
                std::printf(__VA_ARGS__);                  \
                std::printf("\n");                         \
            }                                              \
        }                                                  \
    } while (0)

template <uint32_t kTile>
static void check_tiles(uint32_t len, uint32_t first_pos, uint32_t queries, uint32_t window, uint32_t sinks) {
    const uint32_t last_pos = first_pos + queries - 1;
    const uint32_t end = len < last_pos + 1 ? len : last_pos + 1;
    const VisibleTiles v = visible_tiles<kTile>(first_pos, end, window, sinks);
    std::set<uint32_t> want, got;
    for (uint32_t k = 0; k < len; k++)
        for (uint32_t q = first_pos; q <= last_pos; q++)
            if (key_visible(k, q, len, true, window, sinks)) want.insert(k / kTile);
    for (uint32_t i = 0; i < v.count; i++) {
        EXPECT(got.insert(v.tile(i)).second, "tile %u twice", v.tile(i));
        EXPECT(v.tile(i) * kTile < len, "tile %u behind the cache of %u", v.tile(i), len);
        EXPECT(i == 0 || v.tile(i) > v.tile(i - 1), "order");
    }
    for (uint32_t t : want) EXPECT(got.count(t), "len %u pos %u+%u window %u sinks %u: tile %u missed", len, first_pos, queries, window, sinks, t);
    // every key any query sees lies in [0, sinks) or [lo, end): what the scale of a run of rows goes by
    for (uint32_t k = 0; k < len; k++)
        for (uint32_t q = first_pos; q <= last_pos; q++)
            if (key_visible(k, q, len, true, window, sinks))
                EXPECT(k < v.end && (k >= v.lo || (window && k < sinks)), "key %u of %u not in the runs", k, len);
    // and no more tiles than the two runs touch
    EXPECT(got.size() <= want.size() + 1, "len %u pos %u+%u window %u sinks %u: %zu tiles for %zu", len, first_pos, queries, window, sinks, got.size(), want.size());
}

int main() {
    for (uint32_t len = 1; len <= 70; len += len < 20 ? 1 : 7)
        for (uint32_t first = 0; first <= 75; first += first < 10 ? 1 : 5)
            for (uint32_t queries : {1u, 2u, 9u})
                for (uint32_t window : {0u, 1u, 2u, 7u, 8u, 16u, 33u, 100u, 0xFFFFFFFFu})
                    for (uint32_t sinks : {0u, 1u, 4u, 8u, 9u, 40u, 0xFFFFFFFFu}) {
                        check_tiles<4>(len, first, queries, window, sinks);
                        check_tiles<16>(len, first, queries, window, sinks);
                    }
    // lengths near the limit of 2^31 tokens
    {
        const VisibleTiles v = visible_tiles<64>(0x7FFFFFFEu, 0x7FFFFFFFu, 4096, 4);
        EXPECT(v.sink_tiles == 1 && v.count <= 1 + 65 && v.tile(v.count - 1) == 0x7FFFFFFEu / 64, "long cache");
    }
    for (int32_t entry : {-2147483647 - 1, -7, -1, 0, 4, 5, 6, 2147483647}) {
        uint32_t row = 77;
        const bool ok = pool_row(entry, 3, 16, 5, &row);
        EXPECT(ok == (entry >= 0 && entry < 5), "entry %d", entry);
        EXPECT(row < 5 * 16, "row %u of entry %d", row, entry);
        if (ok) EXPECT(row == uint32_t(entry) * 16 + 3, "row");
    }
    std::printf(failures ? "%d FAILURES\n" : "ok\n", failures);
    return failures != 0;
}
