// Which kernel a call takes over 8-bit pools or through a window, and into how many pieces the keys are cut: estimates
// in microseconds from the sizes alone, plain arithmetic without HIP.
//
// The three candidates differ in how many query rows share what is read.  The row kernel has 16 a workgroup: little to set
// up, and every 16 rows read their keys again.  The persistent kernel has 16 a wave, a fixed number of waves and no tail.  The
// tiles kernel has 256 a workgroup and runs at the rate of the matrix cores, behind a long prologue.  The constants are
// fits to 160 calls drawn over 2 to 1500 queries, 1 to 16 KV heads, contexts up to 33000 and windows from 1 on, each timed on
// all three, and to 150 decode steps of 1 to 64 sequences on the two that take them.  What following the estimates costs over
// the best kernel of each call: 2.3 % over those 160 (the worst 1.6 times), 1.7 % over 100 others (1.3 times), 0.8 % over the steps
// (1.4 times).
#pragma once

#include <stdint.h>

#include <algorithm>
#include <cmath>

namespace ghip {

struct KvCall {
    uint64_t rows;   // per KV head and sequence: queries * heads of a group
    uint32_t lists;  // KV heads * sequences
    uint32_t queries, group, head_dim;
    uint32_t start_pos, length;  // position of the first query, keys of the cache
    uint64_t window_keys;        // window and sinks, 0: no window
    bool causal;
    bool f8, paged_runs;  // paged_runs: 16 tokens in a row lie in one block, or the cache is contiguous
    bool wide;            // float queries or results
    uint32_t cus;
};

// Keys that a workgroup of `rows` rows visits; without a window the average, where they grow with the query's position.
inline double kv_keys(const KvCall& c, uint64_t rows) {
    if (c.window_keys) return double(std::min<uint64_t>(c.length, c.window_keys + (std::min(rows, c.rows) + c.group - 1) / c.group));
    if (!c.causal || c.start_pos >= c.queries) return c.length;
    return (std::min(c.start_pos, c.length) + c.length) / 2.0;
}

struct KvCut {
    uint32_t pieces;
    double us;
};

// Rounds of workgroups over the chip, one a CU at a time; after the second the CUs no longer end together.
inline double kv_rounds(double workgroups, uint32_t cus) {
    const double x = workgroups / cus;
    return x <= 2.0 ? std::ceil(x) : x + 0.5;
}

// Partial results to memory and back at 4 TB/s, and the launch that joins them.
inline double kv_join_us(const KvCall& c, uint32_t pieces) {
    return pieces == 1 ? 0.0 : 5.0 + 8.0 * pieces * double(c.rows) * c.lists * c.head_dim / 4e6;
}

// Row kernel: eight waves take tiles of 64 tokens in turn, 3 us each (4.5 where every token has its own table entry) as long
// as memory gives 4.4 TB/s (5.2 where rows are 256 bytes), of which a CU gets at most 1/150.
inline KvCut kv_rows_cut(const KvCall& c) {
    const double workgroups = double((c.rows + 15) / 16) * c.lists, tiles = std::ceil(kv_keys(c, 16) / 64);
    const double tile_us = c.paged_runs ? 3.0 : c.f8 ? 4.5 : 3.5;
    const double row_bytes = double(c.head_dim) * (c.f8 ? 1 : 2);
    const double memory_us = workgroups * tiles * 128.0 * row_bytes / (row_bytes >= 256 ? 5.2e6 : 4.4e6);
    KvCut best{1, 0.0};
    const uint32_t most = uint32_t(std::min(std::max(tiles / 8, 1.0), 64.0));
    for (uint32_t n = 1; n <= most && (n == 1 || workgroups * n <= c.cus); n++) {
        const double busy = kv_rounds(workgroups * n, c.cus) * (1.5 + std::max(1.0, tiles / (8.0 * n)) * tile_us);
        const double us = 4.0 + std::max(memory_us * std::max(1.0, 0.6 * c.cus / (workgroups * n)), busy) + kv_join_us(c, n);
        if (n == 1 || us < best.us) best = {n, us};
    }
    return best;
}

// Tiles kernel: 2.1 us a tile of 64 keys at head size 128, 1.5 at 64, 1.6 times that with float queries or results (an
// operand in two halves), 1.3 times that with a scale per 4 keys; three tiles' time for the prologue and the end.
inline KvCut kv_tiles_cut(const KvCall& c) {
    const double workgroups = double((c.rows + 255) / 256) * c.lists, tiles = std::ceil(kv_keys(c, 256) / 64);
    const double tile_us = (c.head_dim == 128 ? 2.1 : 1.5) * (c.wide ? 1.6 : 1.0) * (c.paged_runs ? 1.0 : 1.3);
    KvCut best{1, 0.0};
    const uint32_t most = uint32_t(std::min(std::max(tiles / 4, 1.0), 64.0));
    for (uint32_t n = 1; n <= most && (n == 1 || workgroups * n <= 4.0 * c.cus); n++) {
        const double us = 5.5 + kv_rounds(workgroups * n, c.cus) * (std::ceil(tiles / n) + 3) * tile_us + kv_join_us(c, n);
        if (n == 1 || us < best.us) best = {n, us};
    }
    return best;
}

// Persistent kernel (blocks of multiples of 16 tokens, or a contiguous cache): eight waves a CU share the tiles of 16 rows
// and 32 tokens.
inline double kv_stream_us(const KvCall& c) {
    const double units = double((c.rows + 15) / 16) * c.lists * (kv_keys(c, c.rows) / 32 + 0.5) / (8.0 * c.cus);
    return 9.5 + std::max(1.0, units) * (c.f8 ? (c.head_dim == 128 ? 2.6 : 1.6) : (c.head_dim == 128 ? 6.0 : 3.3));
}

}  // namespace ghip
