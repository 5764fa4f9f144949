// Calls with several queries whose windows all lie behind the cache have no tile to visit, and some of them go to the
// persistent kernel: the calls that tests/test_gpu_kv_ex_behind.py makes.
#include <algorithm>
#include <cstdio>

#include "kv_choice.h"
#include "kv_visible.h"

using namespace ghip;

int main() {
    struct Call {
        uint32_t queries, start, length, window, heads, kv_heads, dim;
        bool streamed;
    };
    int failures = 0;
    for (const Call& a : {Call{2, 2048, 1024, 1024, 32, 8, 128, true}, Call{2, 2048, 1024, 1024, 32, 8, 64, true}, Call{4, 5000, 2048, 2048, 16, 8, 128, true},
                          Call{1, 3140, 2080, 1000, 16, 16, 64, true}, Call{1, 128, 64, 20, 4, 2, 128, false}, Call{400, 2000, 1024, 700, 32, 1, 64, false}}) {
        const uint32_t end = std::min(a.length, a.start + a.queries);
        if (visible_tiles<32>(a.start, end, a.window, 0).count != 0) {
            std::printf("%u queries at %u: tiles to visit\n", a.queries, a.start);
            failures++;
        }
        for (bool wide : {false, true}) {
            KvCall c{};
            c.group = a.heads / a.kv_heads;
            c.rows = uint64_t(a.queries) * c.group;
            c.lists = a.kv_heads;
            c.queries = a.queries;
            c.head_dim = a.dim;
            c.start_pos = a.start;
            c.length = end;
            c.window_keys = a.window;
            c.causal = true;
            c.f8 = true;
            c.paged_runs = true;
            c.wide = wide;
            c.cus = 256;
            const double rows = kv_rows_cut(c).us, tiles = kv_tiles_cut(c).us, stream = kv_stream_us(c);
            if ((c.rows <= 1280 && stream < std::min(rows, tiles)) != a.streamed) {
                std::printf("%u queries at %u of %u heads: rows %f tiles %f persistent %f\n", a.queries, a.start, a.dim, rows, tiles, stream);
                failures++;
            }
        }
    }
    if (failures) return 1;
    std::printf("ok\n");
    return 0;
}
