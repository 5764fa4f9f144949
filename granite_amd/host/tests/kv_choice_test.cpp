// csrc/kv_choice.h: the estimates are finite and positive, the pieces within what the launchers take, and calls go
// where they belong: a few rows to the row kernel, a draft behind a long context to the persistent one, many rows to tiles.
#include <cstdio>

#include "kv_choice.h"

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

static KvCall call(uint32_t queries, uint32_t start, uint32_t heads, uint32_t kv_heads, uint32_t dim, bool f8, bool runs, bool wide,
                   uint64_t window_keys) {
    KvCall c{};
    c.group = heads / kv_heads;
    c.rows = uint64_t(queries) * c.group;
    c.lists = kv_heads;
    c.queries = queries;
    c.head_dim = dim;
    c.start_pos = start;
    c.length = start + queries;
    c.window_keys = window_keys;
    c.causal = true;
    c.f8 = f8;
    c.paged_runs = runs;
    c.wide = wide;
    c.cus = 256;
    return c;
}

int main() {
    for (uint32_t queries : {1u, 2u, 17u, 300u, 5000u, 70000u, 0x3FFFFFFFu})
        for (uint32_t start : {0u, 1u, 1000u, 200000u, 0x3FFFFFFFu})
            for (uint32_t group : {1u, 4u, 48u})
                for (uint32_t kv_heads : {1u, 8u, 1000u})
                    for (uint64_t window : {uint64_t(0), uint64_t(1), uint64_t(500), uint64_t(0xFFFFFFFFull) * 2})
                        for (uint32_t cus : {1u, 256u}) {
                            KvCall c = call(queries, start, group * kv_heads, kv_heads, 128, true, start % 2 == 0, group == 4, window);
                            c.cus = cus;
                            for (const KvCut& cut : {kv_rows_cut(c), kv_tiles_cut(c)}) {
                                EXPECT(cut.us > 0 && cut.us < 1e300, "%u queries at %u", queries, start);
                                EXPECT(cut.pieces >= 1 && cut.pieces <= 64, "%u pieces", cut.pieces);
                                EXPECT(cut.pieces == 1 || cut.pieces * 256.0 <= kv_keys(c, 256) + 64, "%u pieces of %f keys", cut.pieces, kv_keys(c, 256));
                            }
                            EXPECT(kv_stream_us(c) > 0 && kv_stream_us(c) < 1e300, "%u queries at %u", queries, start);
                        }
    for (int i = 0; i < 16; i++) {
        const bool f8 = i & 1, runs = i & 2, wide = i & 4;
        const uint32_t dim = i & 8 ? 128 : 64;
        for (uint32_t window : {0u, 1u, 40u, 304u, 4004u})
            EXPECT(kv_tiles_cut(call(400, 700, 96, 1, dim, f8, runs, wide, window)).us < kv_rows_cut(call(400, 700, 96, 1, dim, f8, runs, wide, window)).us,
                   "case %d window %u", i, window);
        EXPECT(kv_rows_cut(call(4, 500, 32, 8, dim, f8, runs, wide, 0)).us < kv_tiles_cut(call(4, 500, 32, 8, dim, f8, runs, wide, 0)).us, "case %d", i);
    }
    // decode steps: sequences, heads, KV heads, head size, tokens a sequence may have, window and sinks, 8-bit
    struct Step {
        uint32_t batch, heads, kv_heads, dim, capacity, window_keys;
        bool f8, streamed;
    };
    for (const Step& s : {Step{24, 32, 8, 128, 3008, 0, true, true}, Step{24, 16, 16, 64, 2944, 0, true, true}, Step{40, 28, 4, 128, 3008, 0, true, true},
                          Step{60, 48, 1, 64, 4064, 0, true, true}, Step{30, 40, 5, 128, 3008, 0, true, true}, Step{40, 34, 2, 128, 4096, 0, true, true},
                          Step{24, 32, 8, 128, 3008, 2537, true, true}, Step{24, 16, 16, 128, 3024, 2004, true, true}, Step{24, 16, 16, 64, 2528, 0, true, true},
                          Step{24, 16, 16, 64, 3024, 2504, true, true}, Step{24, 16, 16, 64, 3024, 2504, false, true}, Step{24, 16, 16, 64, 3024, 2004, false, true},
                          Step{16, 16, 8, 128, 4064, 4000, false, true}, Step{16, 16, 8, 128, 4064, 2637, false, true}, Step{16, 24, 24, 64, 4064, 2637, false, true},
                          Step{16, 24, 24, 64, 4064, 4000, false, true}, Step{1, 32, 16, 128, 16000, 9000, false, true}, Step{1, 48, 48, 64, 16000, 9000, false, true},
                          Step{1, 32, 8, 128, 512, 0, true, false}, Step{4, 32, 8, 128, 256, 0, true, false}, Step{16, 32, 8, 128, 64, 0, true, false}}) {
        KvCall c = call(1, 0, s.heads, s.kv_heads, s.dim, s.f8, true, true, s.window_keys);
        c.lists = s.batch * s.kv_heads;
        c.length = s.capacity;
        c.causal = false;
        EXPECT((kv_stream_us(c) < kv_rows_cut(c).us) == s.streamed, "%u sequences of %u, %u heads of %u, window %u: %f against %f", s.batch, s.capacity, s.kv_heads, s.dim, s.window_keys, kv_stream_us(c), kv_rows_cut(c).us);
    }
    EXPECT(kv_stream_us(call(4, 32768, 32, 8, 128, true, true, false, 0)) < kv_rows_cut(call(4, 32768, 32, 8, 128, true, true, false, 0)).us, "a draft");
    if (failures) {
        std::printf("%d failures\n", failures);
        return 1;
    }
    std::printf("ok\n");
    return 0;
}
