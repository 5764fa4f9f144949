// Which keys a launch of the windowed / 8-bit attention entry points has to visit, as plain integer
// arithmetic: no HIP in this header, so the same functions are checked on the CPU against a count
// of the keys one by one.
//
// A query at position p sees key k of a cache of `len` tokens iff k < len, k <= p (causal) and, under a
// window, k > p - window or k < sinks.  The queries of a launch (or of a workgroup) are at positions
// first_pos .. last_pos, so the keys that any of them sees are the sinks in front and one run that
// begins where the first query's window does:
//
//     [0, sink_end)  and  [lo, end),   sink_end <= lo
//
// Keys are visited in tiles of kTile tokens numbered from key 0; the tiles of the two runs are numbered
// through without a gap (a tile that both runs touch is listed once), and tile() maps back.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define GHIP_HD __host__ __device__ __forceinline__
#else
#define GHIP_HD inline
#endif

namespace ghip {

struct VisibleTiles {
    uint32_t lo;          // first key of the window's run
    uint32_t end;         // one behind its last
    uint32_t sink_tiles;  // tiles in front that hold sinks and lie before the run's first tile
    uint32_t skipped;     // tiles between those and the run's first tile
    uint32_t count;       // tiles to visit

    GHIP_HD uint32_t tile(uint32_t i) const { return i < sink_tiles ? i : i + skipped; }
};

// First key of the window of a query at position `pos` (window 0: none).
GHIP_HD uint32_t window_begin(uint32_t pos, uint32_t window) {
    return window != 0 && pos >= window ? pos - window + 1 : 0u;
}

// `end`: one behind the last key any query sees, at most the length of the cache.
template <uint32_t kTile>
GHIP_HD VisibleTiles visible_tiles(uint32_t first_pos, uint32_t end, uint32_t window, uint32_t sinks) {
    VisibleTiles v;
    v.end = end;
    v.lo = window_begin(first_pos, window);
    const uint32_t begin = v.lo < end ? v.lo : end;  // the window may lie behind the cache's end
    uint32_t sink_end = sinks < begin ? sinks : begin;
    if (window == 0) sink_end = 0;
    const uint32_t first = begin / kTile;
    const uint32_t last = end / kTile + (end % kTile != 0);
    v.sink_tiles = sink_end / kTile + (sink_end % kTile != 0);
    if (v.sink_tiles > first) v.sink_tiles = first;
    v.skipped = first - v.sink_tiles;
    v.count = v.sink_tiles + (last - first);
    return v;
}

// Whether a query at position `pos` sees key `key` of a cache of `len` tokens.
GHIP_HD bool key_visible(uint32_t key, uint32_t pos, uint32_t len, bool causal, uint32_t window, uint32_t sinks) {
    if (key >= len || (causal && key > pos)) return false;
    return window == 0 || key >= window_begin(pos, window) || key < sinks;
}

// Row of a paged pool that holds token `tok` whose block-table entry is `entry`; false where the entry
// names no block of the pool.
GHIP_HD bool pool_row(int32_t entry, uint32_t in_block, uint32_t block_size, uint32_t num_blocks, uint32_t* row) {
    const bool valid = static_cast<uint32_t>(entry) < num_blocks;
    *row = valid ? static_cast<uint32_t>(entry) * block_size + in_block : 0u;
    return valid;
}

}  // namespace ghip
