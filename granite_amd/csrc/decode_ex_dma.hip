// The persistent decode kernel over 8-bit pools whose blocks are multiples of 16 tokens, with K and V moved global -> LDS
// without passing through registers.
//
// The list of tiles, the shares, the pieces and the merge are those of decode_ex_stream.hip, with tiles of 32 tokens.
// What differs is how a wave gets its data.  As an MFMA operand straight from memory, neighbouring lanes hold different
// rows, so a 16-byte load of K touches 64 cache lines' worth of addresses and an 8-byte load of V half a line: the
// data path of the vector cache was busy 80 % of the time and waves waited to issue loads, at 5.4 TB/s.  A wave-wide
// global_load_lds_dwordx4 reads eight whole rows of 128 bytes instead (sixteen of 64), and what lies in LDS is
// read as the operands want it:
//   K    ds_read_b128, lane (n, g): row n, bytes 64 i + 16 g (two steps of the first product)
//   V^T  ds_read_b64_tr_b8: within 16 lanes, lane 2 k + r points at 8 bytes of key k and lane j receives byte j of
//        the 16 of each of the 8 keys, which is row j of the A operand: no transposition in registers
// Rows lie one after the other; the 16-byte pieces of a row are XORed with a function of the row, so that the 16 rows
// of a K read and the 16 of half a V read fall into all 64 banks.
//
// A wave owns two buffers of one tile (16 KiB in all at head size 128): it waits for a tile, computes it, and asks for
// the tile after the next into the same buffer, so that between one and two tiles per wave, 64 to 128 KiB per CU, are in
// flight.  No barriers.  What belongs to a tile (pool rows of its two runs of 16 tokens, their scales) is worked out 32
// tiles at a time, a lane per run; its block-table entries and scales come through LDS as well, since a load the
// compiler waits for would wait for all transfers in flight.
//
// Measured (group of 4 or 8 heads over 8 KV heads of 128, half Q, whole call with the merge): 64 sequences of 256 to 8192 tokens
// 98 us for 556 MB, 5.7 TB/s; 2 of 131072 92 us for 515 MB, 5.6 TB/s.  Without the arithmetic (timing only) the kernel takes
// as long: what bounds it is the pattern of memory accesses, 7 us until the first tiles have come and waves that end
// 15 to 28 us apart.
#include "common.h"
#include "kv_attend.h"

namespace ghip {
namespace {

constexpr uint32_t kWaves = 8;
constexpr uint32_t kPlanHeader = 4;
constexpr uint32_t kTokens = 32;      // per tile
constexpr uint32_t kPlanUnits = 32;   // tiles worked out at a time: two runs each, a lane per run

typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef int int2x __attribute__((__vector_size__(2 * sizeof(int))));

// 64 x 16 (or 64 x 4) bytes from a scalar base and per-lane offsets (or per-lane addresses) into LDS: lane i's piece
// lands at lds_addr + 16 i (4 i).  Counted by vmcnt; nothing tells the compiler that LDS changes.  kOnce: nobody reads
// them again (64 sequences of 8192: 7 % quicker as non-temporal; read by ten groups of 16 rows: 8 % slower).
template <bool kOnce>
__device__ __forceinline__ void dma16(uint32_t lds_addr, const void* sbase, uint32_t lane_off) {
    if constexpr (kOnce)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" : : "s"(lds_addr), "v"(lane_off), "s"(sbase) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds_addr), "v"(lane_off), "s"(sbase) : "memory", "m0");
}
__device__ __forceinline__ void dma4(uint32_t lds_addr, const void* addr) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds_addr), "v"(addr) : "memory", "m0");
}
template <int kCount>
__device__ __forceinline__ void wait_transfers() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kCount) : "memory");
}

template <int kD>
struct Geo {
    static constexpr uint32_t kRows = 1024 / kD;                  // rows per transfer
    static constexpr uint32_t kPieces = kD / 16;                  // 16-byte pieces of a row
    static constexpr uint32_t kHalf = kTokens * kD;               // bytes of K (of V) of a tile
    static constexpr int kTransfers = 2 * int(kTokens / kRows);   // per tile
    static constexpr uint32_t kWaveBytes = 4 * kHalf;             // two tiles
    static constexpr uint32_t kSideBytes = 3 * 64 * 4;            // entries, K scales, V scales
    // what a piece index of row r is XORed with
    static __device__ __forceinline__ uint32_t swizzle(uint32_t r) {
        return kD == 128 ? ((r >> 1) & 7) ^ ((r >> 2) & 4) : ((r >> 2) & 3) ^ ((r >> 3) & 2);
    }
};

// kMulti: several queries of one sequence.  The rows of a KV head, row = query * group + head, take the place of its group's
// heads: 16 of them are a "head" of the list, which streams the KV head's tiles as any other (few rows: what they share
// they find in the L2).
template <bool kQF32, int kD, uint32_t kPer, bool kMulti>
__global__ void __launch_bounds__(kWaves* kWave, 2) kv_dma_kernel(KvParams p) {
    using G = Geo<kD>;
    constexpr int kSteps = kD / 32, kBlocks = kD / 16;
    const uint32_t lane = threadIdx.x & 63, wave = ex_uniform(threadIdx.x >> 6);
    const uint32_t n = lane & 15, g = lane >> 4;
    const uint32_t worker = blockIdx.x * (kWaves / kPer) + wave / kPer;

    extern __shared__ __attribute__((aligned(16))) unsigned char s_raw[];
    unsigned char* const s_wave = s_raw + wave * G::kWaveBytes;
    unsigned char* const s_side = s_raw + kWaves * G::kWaveBytes + wave * G::kSideBytes;
    uint32_t* const s_prefix = reinterpret_cast<uint32_t*>(s_raw + kWaves * (G::kWaveBytes + G::kSideBytes));
    uint32_t* const s_len = s_prefix + p.batch + 1;
    const uint32_t lds_wave = uint32_t(uintptr_t((lds_byte*)s_wave)), lds_side = uint32_t(uintptr_t((lds_byte*)s_side));

    // ---- tile counts and their prefix sums, as in decode_ex_stream.hip
    __shared__ uint32_t s_wave_sum[kWaves];
    const uint32_t vheads = p.num_kv_heads * p.q_groups;
    const uint32_t n_rows = kMulti ? p.seq_q * p.group : p.group;  // of a KV head
    auto seen_of = [&](uint32_t len) __attribute__((always_inline)) {
        if constexpr (kMulti) return visible_tiles<kTokens>(p.start_pos, p.causal ? min(len, p.start_pos + p.seq_q) : len, p.window, p.sinks);
        else return visible_tiles<kTokens>(len - 1, len, p.window, p.sinks);
    };
    auto count_of = [&](uint32_t len) __attribute__((always_inline)) { return len ? seen_of(len).count : 0u; };
    uint32_t tiles_total;
    {
        const uint32_t run = (p.batch + blockDim.x - 1) / blockDim.x, b0 = threadIdx.x * run;
        uint32_t mine = 0;
        for (uint32_t b = b0; b < min(b0 + run, p.batch); b++) {
            const uint32_t len = ex_seq_len(p, b);
            s_len[b] = len;
            mine += count_of(len);
        }
        uint32_t incl = mine;
#pragma unroll
        for (uint32_t off = 1; off < kWave; off <<= 1) {
            const uint32_t up = ex_lane_read(incl, lane >= off ? lane - off : lane);
            if (lane >= off) incl += up;
        }
        if (lane == kWave - 1) s_wave_sum[wave] = incl;
        __syncthreads();
        uint32_t before = 0, all = 0;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; w++) {
            const uint32_t v = s_wave_sum[w];
            if (w < wave) before += v;
            all += v;
        }
        uint32_t at = before + incl - mine;
        for (uint32_t b = b0; b < min(b0 + run, p.batch); b++) {
            s_prefix[b] = at;
            at += count_of(s_len[b]);
        }
        tiles_total = ex_uniform(all);
        if (threadIdx.x == 0) s_prefix[p.batch] = tiles_total;
        __syncthreads();
    }
    const uint32_t lists = vheads / kPer;
    const uint32_t total = tiles_total * lists;
    const uint32_t per = max((total + p.workers - 1) / p.workers, p.min_per);
    if (blockIdx.x == 0) {
        for (uint32_t i = threadIdx.x; i <= p.batch; i += blockDim.x) p.plan[kPlanHeader + i] = s_prefix[i];
        if (threadIdx.x == 0) {
            p.plan[0] = per;
            p.plan[1] = kPer;
        }
    }
    const uint32_t u0 = worker * per;
    if (u0 >= total) return;
    const uint32_t n_units = min(per, total - u0);

    // ---- what the tiles are: lane 2 u + r has run r of unit `first + u`
    struct Plan {
        uint32_t tok, len, b, lh;  // first token of the tile, sequence's length, sequence, list head | last of its segment << 31
        uint32_t row;              // pool row of the run's first token
        uint32_t valid;            // the page is one of the pool's
        float ks, vs;
    };
    uint32_t search_steps = 0;
    while ((1u << search_steps) < p.batch) search_steps++;
    auto run_token = [&](const Plan& q) __attribute__((always_inline)) { return q.tok + 16 * (lane & 1); };
    auto kv_head_of = [&](uint32_t lh) __attribute__((always_inline)) {
        const uint32_t vh = (lh & 0x7FFFFFFFu) * kPer + wave % kPer;
        return p.q_groups == 1 ? vh : vh / p.q_groups;
    };
    // step 1: which tiles; their block-table entries are requested
    auto plan_tiles = [&](uint32_t first) __attribute__((always_inline)) -> Plan {
        Plan q;
        const uint32_t u = u0 + min(first + (lane >> 1), n_units - 1);
        uint32_t lo = 0, hi = p.batch;  // prefix[lo] * lists <= u < prefix[hi] * lists
        for (uint32_t i = 0; i < search_steps; i++) {
            const uint32_t mid = (lo + hi) >> 1;
            const bool below = s_prefix[mid] * lists <= u;
            lo = below ? mid : lo;
            hi = below ? hi : mid;
        }
        q.len = s_len[lo];
        const uint32_t in_seq = u - s_prefix[lo] * lists;
        const VisibleTiles seen = seen_of(max(q.len, 1u));
        const uint32_t lh = in_seq / seen.count, t = in_seq - lh * seen.count;
        q.b = lo;
        q.lh = lh | (t + 1 == seen.count ? 0x80000000u : 0u);
        q.tok = seen.tile(t) * kTokens;
        const uint32_t tok = min(run_token(q), max(q.len, 1u) - 1);
        const uint32_t blk = p.bs_shift >= 0 ? tok >> p.bs_shift : tok / p.block_size;
        dma4(lds_side, p.tables + size_t(lo) * p.max_blocks + blk);
        return q;
    };
    // step 2, the entries being there: rows; the scales are requested
    auto plan_rows = [&](Plan& q) __attribute__((always_inline)) {
        const uint32_t tok = min(run_token(q), max(q.len, 1u) - 1);
        const uint32_t in = (p.bs_shift >= 0 ? tok & (p.block_size - 1) : tok % p.block_size) & ~15u;
        const int32_t entry = reinterpret_cast<const int32_t*>(s_side)[lane];
        q.valid = pool_row(entry, in, p.block_size, p.num_blocks, &q.row) ? 1u : 0u;
        const size_t at = size_t(q.valid ? uint32_t(entry) : 0u) * p.num_kv_heads + kv_head_of(q.lh);
        dma4(lds_side + 256, p.k_scale + at);
        dma4(lds_side + 512, p.v_scale + at);
    };
    // step 3, the scales being there.  A run that no query sees has scale 0, whatever lies in the arrays.
    auto plan_scales = [&](Plan& q) __attribute__((always_inline)) {
        const VisibleTiles seen = seen_of(max(q.len, 1u));
        const uint32_t first = run_token(q), lo = seen.lo;
        const bool used = bool(int(q.valid) & int(first < seen.end) & (int(first + 15 >= lo) | int(first < p.sinks)));
        const float ks = reinterpret_cast<const float*>(s_side)[64 + lane], vs = reinterpret_cast<const float*>(s_side)[128 + lane];
        q.ks = used ? ks : 0.0f;
        q.vs = used ? vs : 0.0f;
    };
    Plan cur, next;
    cur = plan_tiles(0);
    wait_transfers<0>();
    plan_rows(cur);

    // ---- a tile on its way: what is read from the plan when it is requested
    struct Unit {
        uint32_t tok, len, b, lh, valid;  // valid: a bit per run
        float ks[2], vs[2];
    };
    auto lane_u = [&](uint32_t v, uint32_t l) __attribute__((always_inline)) { return uint32_t(__builtin_amdgcn_readlane(int(v), int(l))); };
    auto lane_f = [&](float v, uint32_t l) __attribute__((always_inline)) { return __uint_as_float(uint32_t(__builtin_amdgcn_readlane(int(__float_as_uint(v)), int(l)))); };
    const uint32_t row_bytes = uint32_t(p.row_bytes);
    // transfer q of a tile: rows kRows q + lane / kPieces, slot lane % kPieces holds piece slot ^ swizzle(row)
    const uint32_t r_in = lane / G::kPieces;
    const uint32_t piece_a = (lane % G::kPieces) ^ G::swizzle(r_in);
    const uint32_t off_a = r_in * row_bytes + 16 * piece_a;
    const uint32_t off_b = r_in * row_bytes + 16 * (piece_a ^ (kD == 128 ? 4 : 2));
    auto request = [&](uint32_t i, uint32_t buf) __attribute__((always_inline)) -> Unit {
        const uint32_t l = 2 * (i % kPlanUnits);
        Unit u;
        u.tok = lane_u(cur.tok, l);
        u.len = lane_u(cur.len, l);
        u.b = lane_u(cur.b, l);
        u.lh = lane_u(cur.lh, l);
        u.valid = lane_u(cur.valid, l) | (lane_u(cur.valid, l + 1) << 1);
        const uint64_t head = uint64_t(kv_head_of(u.lh)) * uint64_t(p.head_bytes);
        const uint32_t dst = lds_wave + buf * 2 * G::kHalf;
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // the buffer's last reads are through
#pragma unroll
        for (uint32_t run = 0; run < 2; run++) {
            const uint64_t at = uint64_t(lane_u(cur.row, l + run)) * row_bytes + head;
#pragma unroll
            for (uint32_t q = 0; q < 16 / G::kRows; q++) {
                // which of the two lane offsets: swizzle(row + kRows q + 16 run) differs from swizzle(row) by a constant bit
                const bool other = kD == 128 ? (q ^ run) & 1 : run;
                const uint32_t to = dst + (run * (16 / G::kRows) + q) * 1024;
                dma16<!kMulti>(to, p.k + at + uint64_t(q * G::kRows) * row_bytes, other ? off_b : off_a);
                dma16<!kMulti>(to + G::kHalf, p.v + at + uint64_t(q * G::kRows) * row_bytes, other ? off_b : off_a);
            }
        }
        return u;
    };

    auto take_scales = [&](uint32_t i, Unit& u) __attribute__((always_inline)) {
        const uint32_t l = 2 * (i % kPlanUnits);
        u.ks[0] = lane_f(cur.ks, l);
        u.ks[1] = lane_f(cur.ks, l + 1);
        u.vs[0] = lane_f(cur.vs, l);
        u.vs[1] = lane_f(cur.vs, l + 1);
    };

    // ---- query rows and running state, as Rows16
    half8 bq[kSteps], bq_lo[kQF32 ? kSteps : 1];
    float q_unit = p.scale_log2;  // of a product with the row as loaded in the log2 domain, the K scale apart
    float m_run = kExNegBig, l_run = 0.0f, bound = kExNegBig;
    float4v acc[kBlocks];
    auto clear = [&]() __attribute__((always_inline)) {
        m_run = kExNegBig;
        l_run = 0.0f;
        bound = kExNegBig;
#pragma unroll
        for (int t = 0; t < kBlocks; t++) acc[t] = float4v{0, 0, 0, 0};
    };
    // what the lane's row sees: keys in front of row_hi, from row_lo on or sinks; every row of the wave sees those in front of
    // all_hi, from all_lo on
    uint32_t row_hi = 0, row_lo = 0, all_hi = 0, all_lo = 0;
    auto load_q = [&](const Unit& u) __attribute__((always_inline)) {
        const uint32_t vh = (u.lh & 0x7FFFFFFFu) * kPer + wave % kPer, kvh = vh / p.q_groups, row0 = (vh % p.q_groups) * 16;
        const bool live = row0 + n < n_rows;
        const uint32_t row = live ? row0 + n : row0;
        int64_t at = int64_t(u.b) * p.q_batch;
        if constexpr (kMulti) {
            const uint32_t query = row / p.group, last = (min(row0 + 16, n_rows) - 1) / p.group;
            at += int64_t(query) * p.q_tok + int64_t(kvh * p.group + (row - query * p.group)) * p.q_head;
            auto limit = [&](uint32_t pos) __attribute__((always_inline)) { return p.causal ? min(u.len, pos + 1) : u.len; };
            row_hi = limit(p.start_pos + query);
            row_lo = window_begin(p.start_pos + query, p.window);
            all_hi = limit(p.start_pos + row0 / p.group);
            all_lo = window_begin(p.start_pos + last, p.window);
        } else {
            at += int64_t(kvh * p.group + row) * p.q_head;
            row_hi = all_hi = u.len;
            row_lo = all_lo = window_begin(u.len - 1, p.window);
        }
        auto d_of = [&](int s) __attribute__((always_inline)) { return 64 * (s / 2) + 16 * g + 8 * (s % 2); };
        if constexpr (kQF32) {
            q_unit = p.scale_log2 * ex_load_floats<kSteps>(static_cast<const float*>(p.q) + at, d_of, [](float v) { return max_over_groups(v); }, 1.0f, live, bq, bq_lo);
        } else {
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                uint4v w = *reinterpret_cast<const uint4v*>(static_cast<const uint16_t*>(p.q) + at + d_of(s));
                if (!live) w = uint4v{0, 0, 0, 0};
                bq[s] = ex_half8(w);
            }
        }
    };
    auto flush = [&](const Unit& u) __attribute__((always_inline)) {
        float l = l_run;
        l += wave_shfl_xor(l, 16);
        l += wave_shfl_xor(l, 32);
        const uint32_t lh = u.lh & 0x7FFFFFFFu, row0 = ((lh * kPer + wave % kPer) % p.q_groups) * 16;
        if (row0 + n < n_rows) {
            const uint32_t piece = worker + u.b * lists + lh;
            const size_t at = size_t(piece) * p.part_cap + (wave % kPer) * (p.part_cap / kPer) + n;
            const float unit = ex_unit(bound);
#pragma unroll
            for (int t = 0; t < kBlocks; t++) *reinterpret_cast<float4v*>(p.part_o + at * kD + 16 * t + 4 * g) = acc[t] * unit;
            if (g == 0) {
                p.part_ml[at * 2] = m_run;
                p.part_ml[at * 2 + 1] = l;
            }
        }
        clear();
    };

    // ---- operand addresses inside a tile's K (V): row 16 sub + n; key of the V read
    uint32_t k_at[2][kSteps / 2], v_at[kBlocks];
#pragma unroll
    for (uint32_t sub = 0; sub < 2; sub++)
#pragma unroll
        for (uint32_t i = 0; i < kSteps / 2; i++) {
            const uint32_t r = 16 * sub + n;
            k_at[sub][i] = r * kD + 16 * ((4 * i + g) ^ G::swizzle(r));
        }
    {
        const uint32_t k = n >> 1;  // lane 2 k + r of its 16: key tau(g, k), bytes 8 r ..
        const uint32_t key = k < 4 ? 4 * g + k : 16 + 4 * g + (k - 4);
#pragma unroll
        for (uint32_t t = 0; t < uint32_t(kBlocks); t++) v_at[t] = key * kD + 16 * (t ^ G::swizzle(key)) + 8 * (n & 1);
    }

    auto compute = [&](const Unit& u, uint32_t buf) __attribute__((always_inline)) {
        const unsigned char* sk = s_wave + buf * 2 * G::kHalf;
        const unsigned char* sv = sk + G::kHalf;
        float s[2][4];
        uint4v kw[2][kSteps / 2];
#pragma unroll
        for (int sub = 0; sub < 2; sub++)
#pragma unroll
            for (int i = 0; i < kSteps / 2; i++) kw[sub][i] = *reinterpret_cast<const uint4v*>(sk + k_at[sub][i]);
        uint2v vw[kBlocks];
#pragma unroll
        for (int t = 0; t < kBlocks; t++)
            vw[t] = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) int2x*)(sv + v_at[t])));
        float4v c[2];
        c[0] = c[1] = float4v{0, 0, 0, 0};
#pragma unroll
        for (int step = 0; step < kSteps; step++)
#pragma unroll
            for (int sub = 0; sub < 2; sub++) {
                const uint4v w = kw[sub][step / 2];
                const half8 a = step % 2 ? f8x8_to_half8(w.z, w.w) : f8x8_to_half8(w.x, w.y);
                c[sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bq[step], c[sub], 0, 0, 0);
                if constexpr (kQF32) c[sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bq_lo[step], c[sub], 0, 0, 0);
            }
#pragma unroll
        for (int sub = 0; sub < 2; sub++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[sub][i] = c[sub][i] * ex_finite(u.ks[sub] * q_unit);
        uint32_t sees = 0xFFu;  // kMulti: bit 4 sub + i, the lane's row sees token 16 sub + 4 g + i
        const bool masked = u.tok + kTokens > all_hi || (u.tok < all_lo && u.tok + kTokens > p.sinks) || u.valid != 3;
        if (masked) {
            uint32_t keep[2];  // a byte per token
            if constexpr (kMulti) sees = 0;
            const VisibleTiles seen = seen_of(u.len);
#pragma unroll
            for (int sub = 0; sub < 2; sub++) {
                keep[sub] = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t tok = u.tok + 16 * sub + 4 * g + i, valid = (u.valid >> sub) & 1u;
                    const bool vis = bool(int(valid) & int(tok < row_hi) & (int(tok >= row_lo) | int(tok < p.sinks)));
                    const bool any = kMulti ? bool(int(valid) & int(tok < seen.end) & (int(tok >= seen.lo) | int(tok < p.sinks))) : vis;
                    s[sub][i] = vis ? s[sub][i] : -INFINITY;
                    keep[sub] |= any ? 0xFFu << (8 * i) : 0u;
                    if constexpr (kMulti) sees |= vis ? 1u << (4 * sub + i) : 0u;
                    asm volatile("" : "+v"(s[sub][i]), "+v"(keep[sub]), "+v"(sees));
                }
            }
#pragma unroll
            for (int t = 0; t < kBlocks; t++) {
                vw[t].x &= keep[0];
                vw[t].y &= keep[1];
                asm volatile("" : "+v"(vw[t]));
            }
        }
        float tops[2];
#pragma unroll
        for (int sub = 0; sub < 2; sub++) tops[sub] = fmaxf(fmaxf(s[sub][0], s[sub][1]), fmaxf(s[sub][2], s[sub][3]));
        const float top = max_over_groups(fmaxf(tops[0], tops[1])), m_new = fmaxf(m_run, top), moved = m_run - m_new;
        m_run = m_new;
        l_run *= fast_exp2(moved);
        // V scales relative to the row's largest p * (V scale), as attend_tile
        const float e0 = ex_exponent(u.vs[0]), e1 = ex_exponent(u.vs[1]);
        const float z = max_over_groups(fmaxf((tops[0] - m_new) + e0, (tops[1] - m_new) + e1));
        const float bound_new = fmaxf(bound + moved, z), whole = ceilf(bound_new);
        const float rescale = fast_exp2(moved + (ceilf(bound) - whole));
        bound = bound_new;
        if (__any(rescale != 1.0f)) {
#pragma unroll
            for (int t = 0; t < kBlocks; t++) acc[t] *= rescale;
        }
        half8 hi, rem;
#pragma unroll
        for (int sub = 0; sub < 2; sub++) {
            const float shift = (sub ? e1 : e0) - whole, f = ex_mantissa(u.vs[sub]) * kExBoost;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float d = s[sub][i] - m_new;
                l_run += fast_exp2(d);
                _Float16 half, rest;
                ex_split(fast_exp2(d + shift) * f, half, rest);
                hi[4 * sub + i] = half;
                rem[4 * sub + i] = rest;
            }
        }
        if (kMulti && masked) {
            // a NaN of V reaches the rows that see its token and no others: taken out of V, and put back through a product
            // of "is NaN" and "sees"
            half8 see;
#pragma unroll
            for (int j = 0; j < 8; j++) see[j] = (sees >> j) & 1u ? _Float16(1) : _Float16(0);
#pragma unroll
            for (int t = 0; t < kBlocks; t++) {
                uint2v nan;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    // bytes whose low seven bits are all ones: adding one carries into bit 7
                    const uint32_t hit = ((vw[t][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                    vw[t][w] &= ~((hit >> 7) * 0xFFu);
                    nan[w] = (hit >> 7) * 0x38u;  // 1.0
                }
                const float4v mark = __builtin_amdgcn_mfma_f32_16x16x32_f16(f8x8_to_half8(nan.x, nan.y), see, float4v{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) acc[t][i] = mark[i] > 0.0f ? NAN : acc[t][i];
            }
        }
#pragma unroll
        for (int t = 0; t < kBlocks; t++) {
            const half8 a = f8x8_to_half8(vw[t].x, vw[t].y);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi, acc[t], 0, 0, 0);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, rem, acc[t], 0, 0, 0);
        }
    };

    clear();
    // (the first tiles do not wait for their scales, which were requested before them)
    Unit now = request(0, 0), then = now;
    if (n_units > 1) then = request(1, 1);
    load_q(now);
    if (n_units > 1) wait_transfers<2 * G::kTransfers>();
    else wait_transfers<G::kTransfers>();
    plan_scales(cur);
    next = cur;
    take_scales(0, now);
    take_scales(min(1u, n_units - 1), then);
    for (uint32_t i = 0; i < n_units; i++) {
        if (i + 1 < n_units) wait_transfers<G::kTransfers>();  // all but the next tile's
        else wait_transfers<0>();
        compute(now, i & 1);
        const bool last = i + 1 >= n_units;
        if (last || (now.lh >> 31)) {
            flush(now);
            if (!last) load_q(then);
        }
        now = then;
        const uint32_t j = i + 2;
        if (j < n_units) {
            if (j % kPlanUnits == 0) cur = next;
            then = request(j, i & 1);
            take_scales(j, then);
            // the next 32 tiles' plan, in three steps a few tiles apart: what a step needs was requested by the one before
            // and is older than the last tile's transfers, which the loop waits for
            const uint32_t at = j % kPlanUnits;
            if (at == 4 && j - at + kPlanUnits < n_units) next = plan_tiles(j - at + kPlanUnits);
            else if (at == 12 && j - at + kPlanUnits < n_units) plan_rows(next);
            else if (at == 20 && j - at + kPlanUnits < n_units) plan_scales(next);
        }
    }
}

template <bool kQF32, int kD, uint32_t kPer, bool kMulti>
int launch_rows_of(const KvParams& p, dim3 grid, size_t lds) {
    auto kernel = kv_dma_kernel<kQF32, kD, kPer, kMulti>;
    static bool configured[kMaxDevices];
    if (int rc = raise_dynamic_lds_limit(reinterpret_cast<const void*>(kernel), kv_dma_lds_bytes(kD, kStreamMaxBatch), configured)) return rc;
    kernel<<<grid, dim3(kWaves * kWave), lds, ctx().stream>>>(p);
    return launch_status();
}
template <bool kQF32, int kD, uint32_t kPer>
int launch_per(const KvParams& p, dim3 grid, size_t lds) {
    return p.decode ? launch_rows_of<kQF32, kD, kPer, false>(p, grid, lds) : launch_rows_of<kQF32, kD, kPer, true>(p, grid, lds);
}
template <bool kQF32, int kD>
int launch_d(const KvParams& p, uint32_t per_list, dim3 grid, size_t lds) {
    if (per_list == 8) return launch_per<kQF32, kD, 8>(p, grid, lds);
    if (per_list == 4) return launch_per<kQF32, kD, 4>(p, grid, lds);
    if (per_list == 2) return launch_per<kQF32, kD, 2>(p, grid, lds);
    return launch_per<kQF32, kD, 1>(p, grid, lds);
}

}  // namespace

size_t kv_dma_lds_bytes(uint32_t D, uint32_t batch) {
    const size_t tiles = kWaves * (D == 128 ? Geo<128>::kWaveBytes + Geo<128>::kSideBytes : Geo<64>::kWaveBytes + Geo<64>::kSideBytes);
    return tiles + (2 * size_t(batch) + 1) * sizeof(uint32_t);
}

int launch_kv_dma(const KvParams& p, uint32_t D, bool q_f32, uint32_t per_list, dim3 grid) {
    const size_t lds = kv_dma_lds_bytes(D, p.batch);
    if (D == 128) return q_f32 ? launch_d<true, 128>(p, per_list, grid, lds) : launch_d<false, 128>(p, per_list, grid, lds);
    return q_f32 ? launch_d<true, 64>(p, per_list, grid, lds) : launch_d<false, 64>(p, per_list, grid, lds);
}

}  // namespace ghip
