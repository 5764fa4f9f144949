// Attention of a run of queries over 8-bit paged pools, and through a sliding window with sinks: the tiles
// kernel for gfx950 and the merge of its key splits.
//
// What it computes is written at granite_hip_attention_ex (granite_hip.h).  The arithmetic is that of
// attention_tiles_kernel (prefill.hip): S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16_f16, a wave owning 32
// query rows, K and V tiles of 64 keys in LDS as halves, a three-stage pipeline over 32-key sub-tiles (scores of
// j + 1, softmax of j, second product of j - 1 in one phase, vector work spread behind the MFMAs).  What is new:
//
// * Rows are (query, head of the KV head's group) pairs, row = query * group + head, so a workgroup's 256 rows
//   share one KV head's tiles and cover few positions: 256 / group of them.  Under a window a workgroup visits
//   window + 256 / group keys for rows that see `window` each (with a head to itself it would visit window + 256), and
//   a chunk of 37 queries in groups of 4 is one workgroup's worth of rows instead of four quarter-full ones.
// * Codes become halves once per workgroup, on the way from registers to LDS (v_cvt_scalef32_pk_f16_fp8,
//   two codes an instruction): a half holds every e4m3 value, so the products are those of the codes themselves.  Converting
//   operands as they are read would put four conversions beside every MFMA of every wave.
// * Scales never touch an element of K or V.  Where block sizes are multiples of 16 a run of 16 keys lies in one block, so
//   a sub-tile has two scales of K and two of V; where they are other multiples of 4 (kExPaged4) a run of 4 does, which
//   are the rows 8 a + 4 g .. + 3 that lane (n, g) has of its column: four scales a lane instead of two.  K's goes into the factor that takes a score to the
//   log2 domain.  V's enters the exponent: with x = score + log2(v scale) the probabilities p' = exp2(x - ref)
//   carry it, the second product takes the codes, and the sum l takes each run's p' times 1 / (v scale).  The
//   reference follows x, so a large or small V scale never pushes p' out of the range of a half.  Cost per sub-tile:
//   two subtractions and one more multiply-add than without scales.  Where a scale is beyond 2^+-48, p' may have vanished
//   that the sum should count; such a sub-tile's part of l is worked out from the scores (rare).
// * Tiles are visited by the list of kv_visible.h: those of the sinks, then those of the window.
//
// Measured (half Q and results): 512 queries of 64 heads over 8 KV heads of 128 behind 32768 keys 535 to 572 us a call, 1.0 PFLOP/s
// (a large half matrix product reaches 1.17); 4096 queries of 32 heads of 64 through a window of 4096 196 us, 0.70 PFLOP/s;
// 2048 queries of 32 heads of 128 through a window of 512 31 us.  What bounds it: a tile is 64 MFMAs on a SIMD, 2048 cycles,
// and some 370 vector instructions beside them (softmax, conversions of codes and probabilities), 6 a MFMA at head size
// 128 and 11 at 64; the matrix cores are busy 45 % (27 %) of the time.
//
// Probabilities are rounded to half: against float64 a half result is then 2.9e-4 off (root mean square, relative) where
// its own rounding alone would leave 2.1e-4, and a second product for the remainders costs a third more.  That is what float
// outputs get (kPrecise): a half and a half remainder, the second product twice (512 queries behind 32768 keys 748 us where half
// outputs take 553); float queries are two halves as well, the first product twice (897 us).  Sums and accumulators are float.
//
// V of keys that no row of the workgroup sees is stored as zeros, since 0 * NaN is NaN.  In tiles that only
// some rows see, infinities and NaNs of V are stored as zeros as well, and where there were any they are added
// at the end to the rows that see them.
#include "common.h"
#include "kv_attend.h"

namespace ghip {
namespace {

constexpr int kBM = 256;  // query rows per workgroup
constexpr int kBN = 64;   // keys per tile
constexpr int kThreads = 512;
constexpr int kKBuffers = 3, kVBuffers = 3;
constexpr uint32_t kPlan = 64;  // tiles whose rows and scales are worked out at a time
constexpr float kProbLimit = 16384.0f;  // a row's probabilities of a sub-tile may sum to this much
constexpr float kPlainScales = 48.0f;   // V scales within 2^-48 .. 2^48 take the sum's weights from the probabilities
constexpr uint32_t kFarScale = 1u << 8;   // others
constexpr float kFusedScores = 0x1p20f;  // references below this leave scores to a fused multiply-add

template <int kD, int kRows>
struct Shape {
    static constexpr uint32_t kRun = kRows == kExPaged4 ? 4 : 16;  // keys that are sure to lie in one block
    static constexpr uint32_t kTileRuns = kBN / kRun;
    static constexpr int kKPitch = kD + 8;  // halves
    static constexpr int kVPitch = kD;      // halves, 64-byte chunks swizzled with the key
    static constexpr int kKTile = kBN * kKPitch, kVTile = kBN * kVPitch;
    static constexpr size_t kTileBytes = size_t(kKBuffers * kKTile + kVBuffers * kVTile) * sizeof(uint16_t);
    static constexpr size_t kLdsBytes = kTileBytes + 2 * kPlan * kTileRuns * sizeof(float4v) + 16;
    static constexpr int kSteps = kD / 16;   // MFMAs of the scores of a sub-tile
    static constexpr int kBlocks = kD / 32;  // 32-row head-dim blocks of O^T
    static constexpr int kPhase = kSteps + 2 * kBlocks;
};

// Halves of x that are infinite or NaN become zero; whether there were any.
__device__ __forceinline__ bool drop_specials(uint4v& x) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bool lo = (x[i] & 0x7C00u) == 0x7C00u, hi = (x[i] & 0x7C000000u) == 0x7C000000u;
        if (lo) x[i] &= 0xFFFF0000u;
        if (hi) x[i] &= 0x0000FFFFu;
        any = any || lo || hi;
    }
    return any;
}

template <bool kQF32, bool kPrecise, bool kF8, int kRows, int kD>
__global__ void __launch_bounds__(kThreads, 2) kv_tiles_kernel(KvParams p) {
    using S = Shape<kD, kRows>;
    constexpr bool kFine = kRows == kExPaged4;
    constexpr uint32_t kTileRuns = S::kTileRuns;
    constexpr int kLaneRuns = kFine ? 4 : 2, kRunShift = kFine ? 2 : 3;  // of the 16 scores a lane has of a sub-tile
    constexpr int kKPitch = S::kKPitch, kVPitch = S::kVPitch, kKTile = S::kKTile, kVTile = S::kVTile, kSteps = S::kSteps,
                  kBlocks = S::kBlocks, kPhase = S::kPhase;
    extern __shared__ __attribute__((aligned(16))) uint16_t s_mem[];
    uint16_t* const s_k0 = s_mem;
    uint16_t* const s_v0 = s_mem + kKBuffers * kKTile;
    // of run i of the workgroup's j-th tile, at (j mod 128) * kTileRuns + i: scale of the scores, log2 of the V scale, its inverse,
    // bits (the place of the run among those of a lane's 16 scores, where its page is one of the pool's; kFarScale)
    float4v* const s_run = reinterpret_cast<float4v*>(reinterpret_cast<unsigned char*>(s_mem) + S::kTileBytes);
    uint32_t* const s_special = reinterpret_cast<uint32_t*>(s_run + 2 * kPlan * kTileRuns);

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = ex_uniform(tid >> 6);
    const uint32_t n = lane & 31, g = lane >> 5;

    // ---- which (KV head, key split, row tile): ids are handed to the 8 XCDs round-robin, so they are remapped
    // for the workgroups that stream the same keys to share an L2
    uint32_t job = blockIdx.x;
    {
        constexpr uint32_t kXcds = 8;
        if (gridDim.x % kXcds == 0) job = (job % kXcds) * (gridDim.x / kXcds) + job / kXcds;
    }
    const uint32_t slot = job % p.q_tiles, rest = job / p.q_tiles;
    const uint32_t split = rest % p.n_splits, kvh = rest / p.n_splits;

    // ---- rows.  Two runs of 128, four waves each, one wave of each on a SIMD.  Where the keys a row sees grow with
    // its position (causal, no window, few keys in front), the k-th run from the end is paired with the k-th from
    // the start, so that every workgroup has the same work (p.paired, set by the launcher).
    constexpr uint32_t kHalf = kBM / 2;
    const uint32_t n_rows = p.seq_q * p.group;
    const uint32_t halves = (n_rows + kHalf - 1) / kHalf;
    const uint32_t late_half = p.paired ? halves - 1 - slot : 2 * slot + 1;
    const uint32_t early_half = p.paired ? slot : 2 * slot;
    const bool second_run = wave >= kThreads / 128;
    const bool run_live = !second_run || early_half < late_half;
    const uint32_t my_half = (p.paired != 0) == second_run ? early_half : late_half;
    const uint32_t r0 = run_live ? my_half * kHalf + 32 * (wave & 3) : n_rows;
    const bool wave_active = r0 < n_rows;
    const uint32_t row = min(r0 + n, n_rows - 1);
    const bool row_live = r0 + n < n_rows;
    const uint32_t query = row / p.group, head = kvh * p.group + (row - query * p.group);

    // ---- keys: of the workgroup, of this wave, of this lane's row
    auto pos_of = [&](uint32_t r) __attribute__((always_inline)) { return p.start_pos + min(r, n_rows - 1) / p.group; };
    const uint32_t wg_first = pos_of(early_half * kHalf), wg_last = pos_of((late_half + 1) * kHalf - 1);
    const uint32_t len = p.max_tokens;
    auto limit_of = [&](uint32_t pos) __attribute__((always_inline)) { return p.causal ? min(len, pos + 1) : len; };
    const VisibleTiles seen = visible_tiles<kBN>(wg_first, limit_of(wg_last), p.window, p.sinks);
    const uint32_t all_hi = limit_of(wg_first), all_lo = window_begin(wg_last, p.window);  // seen by every row
    const uint32_t t_begin = uint32_t(uint64_t(seen.count) * split / p.n_splits);
    const uint32_t n_tiles = uint32_t(uint64_t(seen.count) * (split + 1) / p.n_splits);
    const uint32_t wave_first = pos_of(r0), wave_last = pos_of(r0 + 31);
    const uint32_t wave_hi = limit_of(wave_last);  // behind the last key any row of the wave sees
    const uint32_t every_hi = limit_of(wave_first), every_lo = window_begin(wave_last, p.window);  // every row sees
    const uint32_t row_hi = limit_of(p.start_pos + query), row_lo = window_begin(p.start_pos + query, p.window);

    // ---- Q^T as B operand: lane (n, g), step s holds Q[row][16 s + 8 g .. + 7]
    half8 bq[kSteps];
    half8 bq_lo[kQF32 ? kSteps : 1];
    float q_unit = p.scale_log2;  // kQF32: of a product with the row as loaded in the log2 domain, the K scale apart; positive
    {
        const int64_t off = int64_t(query) * p.q_tok + int64_t(head) * p.q_head + 8 * g;
        if constexpr (kQF32) {
            auto both_lanes = [](float v) {
                const LanePair both = half_wave_pair(v);
                return fmaxf(both.lo, both.hi);
            };
            q_unit = p.scale_log2 * ex_load_floats<kSteps>(static_cast<const float*>(p.q) + off, [](int s) { return 16 * s; }, both_lanes, p.q_sign, true, bq, bq_lo);
        } else {
#pragma unroll
            for (int s = 0; s < kSteps; s++)
                bq[s] = ex_half8(*reinterpret_cast<const uint4v*>(static_cast<const uint16_t*>(p.q) + off + 16 * s)) * _Float16(p.q_sign);
        }
    }

    float m_ref = kExNegBig, l_run = 0.0f, limit = kProbLimit;
    float16v oacc[kBlocks];
#pragma unroll
    for (int t = 0; t < kBlocks; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) oacc[t][r] = 0.0f;

    // ---- staging: a thread moves a piece of key ld_r of K and of V; the eight threads of a key cover its row.
    // The keys of a wave's pieces (8 of them) lie in one run.
    const uint32_t ld_c = tid & 7, ld_r = tid >> 3;
    constexpr uint32_t kPieceHalves = kD / 8;                 // per thread and row
    constexpr bool kTwo = kD == 128;                          // two 16-byte stores
    constexpr uint32_t kRegs = (kF8 ? kD / 8 : kD / 4) / 4;   // registers of a piece as loaded: 2, 4 or 8
    constexpr uint32_t kSwz = kBlocks - 1;
    // 8 bits: 16 (8) consecutive elements from kPieceHalves * ld_c on.  Half: 8 from 8 ld_c on and, of 128, 8 from 64 on.
    const uint32_t e0 = kF8 ? kPieceHalves * ld_c : 8 * ld_c, e1 = kF8 ? e0 + 8 : e0 + 64;
    auto v_at = [&](uint32_t e) __attribute__((always_inline)) { return ld_r * kVPitch + ((((e >> 5) ^ (ld_r & kSwz)) << 5) | (e & 31)); };
    const uint32_t k_st0 = ld_r * kKPitch + e0, k_st1 = ld_r * kKPitch + e1, v_st0 = v_at(e0), v_st1 = v_at(e1);
    const uint8_t* const k_base = p.k + int64_t(kvh) * p.head_bytes + (kF8 ? e0 : 2 * e0);
    const uint8_t* const v_base = p.v + int64_t(kvh) * p.head_bytes + (kF8 ? e0 : 2 * e0);

    // The 8 keys of a wave's pieces lie in one run of 16 (in two of 4), so the address of a run's first row is the wave's; a
    // lane adds its row's and column's offset.  Rows and scales are worked out for 64 tiles at a time, a lane per tile,
    // and read back lane by lane: per tile that left two scalar reads of what had been lookups, divisions and
    // conversions in the shadow of too few MFMAs (512 queries at 32768: 559 us before, 538 with it; a window of 4096 at
    // head size 64: 217 and 204).
    constexpr int kPieceRuns = kFine ? 2 : 1;
    const uint32_t wave_key = 8 * wave;
    const uint32_t lane_off = (ld_r & (kFine ? 3 : 7)) * uint32_t(p.row_bytes);
    auto key_of = [&](uint32_t it) __attribute__((always_inline)) { return seen.tile(it) * kBN; };  // first key of the it-th tile
    // lane u: first key of run f of the wave's keys in tile t_begin + 64 block + u (the last one again behind it)
    auto plan_key = [&](uint32_t block, int f) __attribute__((always_inline)) {
        const uint32_t it = min(t_begin + kPlan * block + lane, n_tiles - 1);
        return min(seen.tile(it) * kBN + wave_key + 4 * f, (seen.end - 1) & (kFine ? ~3u : ~7u));
    };
    // the block-table entries
    struct Entries {
        int32_t e[kPieceRuns];
    };
    auto plan_entries = [&](uint32_t block) __attribute__((always_inline)) -> Entries {
        Entries r;
#pragma unroll
        for (int f = 0; f < kPieceRuns; f++) r.e[f] = kRows == kExContiguous ? 0 : p.tables[plan_key(block, f) / p.block_size];
        return r;
    };
    // pool row of the first key, bit 31: the page is one of the pool's; and the scales of its run
    struct Plan {
        uint32_t row[kPieceRuns];
        float ks[kPieceRuns], vs[kPieceRuns];
    };
    auto plan_rows = [&](uint32_t block, const Entries& entries) __attribute__((always_inline)) -> Plan {
        Plan r;
#pragma unroll
        for (int f = 0; f < kPieceRuns; f++) {
            const uint32_t key = plan_key(block, f);
            r.ks[f] = r.vs[f] = 1.0f;
            if constexpr (kRows == kExContiguous) {
                r.row[f] = key | 0x80000000u;
            } else {
                const int32_t entry = entries.e[f];
                const bool valid = pool_row(entry, key % p.block_size, p.block_size, p.num_blocks, &r.row[f]);
                if constexpr (kF8) {
                    const uint64_t at = uint64_t(valid ? uint32_t(entry) : 0u) * p.num_kv_heads + kvh;
                    r.ks[f] = p.k_scale[at];
                    r.vs[f] = p.v_scale[at];
                }
                r.row[f] |= valid ? 0x80000000u : 0u;
            }
        }
        return r;
    };
    // what the softmax takes from the scales, for every wave.  A run that nobody sees may have anything for
    // scales; a masked score, minus infinity, must come through the factor and the shift as what it is: a positive
    // factor, a finite shift.
    auto plan_runs = [&](const Plan& r, uint32_t half) __attribute__((always_inline)) {
        if (kRows == kExContiguous || (!kFine && (wave & 1))) return;  // (waves 2 i and 2 i + 1 have the same run of 16)
#pragma unroll
        for (int f = 0; f < kPieceRuns; f++) {
            const bool valid = r.row[f] >> 31;
            const float vs = kF8 && valid ? fminf(fmaxf(r.vs[f], 0x1p-100f), 0x1p+126f) : 1.0f;
            float4v info;
            // (float queries: the K scale alone, each row has a factor of its own)
            if constexpr (kQF32) info.x = kF8 && valid ? fmaxf(r.ks[f], 0x1p-126f) : 1.0f;
            else info.x = kF8 && valid ? fmaxf(fmaxf(r.ks[f], 0.0f) * p.scale_log2, 0x1p-126f) : p.scale_log2;
            info.y = kF8 ? __builtin_amdgcn_logf(vs) : 0.0f;
            info.z = 1.0f / vs;
            const uint32_t run = kFine ? 2 * wave + f : wave >> 1, place = kFine ? (run >> 1) & 3 : run & 1;
            info.w = __uint_as_float(!valid ? 0u : (1u << place) | (fabsf(info.y) > kPlainScales ? kFarScale : 0u));
            s_run[(half * kPlan + lane) * kTileRuns + run] = info;
        }
    };
    // a tile's planned rows: one value for the wave, or one for its first four keys and one for the others
    struct At {
        uint32_t row[kPieceRuns];
    };
    struct Piece {
        uint32_t k[kRegs], v[kRegs];
    };
    auto fetch = [&](uint32_t (&dst)[kRegs], const uint8_t* src) __attribute__((always_inline)) {
        if constexpr (kRegs == 2) {
            const uint2v w = *reinterpret_cast<const uint2v*>(src);
            dst[0] = w.x;
            dst[1] = w.y;
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kRegs / 4; i++) {
                const uint4v w = *reinterpret_cast<const uint4v*>(src + 128 * i);
#pragma unroll
                for (int j = 0; j < 4; j++) dst[4 * i + j] = w[j];
            }
        }
    };
    auto of_lane = [&](const At& at) __attribute__((always_inline)) -> uint32_t {
        if constexpr (kFine) return ld_r & 4 ? at.row[1] : at.row[0];
        else return at.row[0];
    };
    auto piece_at = [&](const uint8_t* base, const At& at) __attribute__((always_inline)) -> const uint8_t* {
        const uint32_t row = of_lane(at) & 0x7FFFFFFFu;
        if constexpr (kRows == kExContiguous) {
            // (rows behind the last key may lie behind the cache's end: the last one instead)
            return base + uint64_t(min(row + (ld_r & 7), len - 1)) * uint64_t(p.row_bytes);
        } else {
            return base + uint64_t(row) * uint64_t(p.row_bytes) + lane_off;
        }
    };
    auto load_k = [&](const At& at, Piece& piece) __attribute__((always_inline)) { fetch(piece.k, piece_at(k_base, at)); };
    auto load_v = [&](const At& at, Piece& piece) __attribute__((always_inline)) { fetch(piece.v, piece_at(v_base, at)); };
    auto halves_of = [&](const uint32_t (&src)[kRegs], int half) __attribute__((always_inline)) -> uint4v {
        if constexpr (kF8) {
            return __builtin_bit_cast(uint4v, f8x8_to_half8(src[2 * half], src[2 * half + 1]));
        } else {
            return uint4v{src[4 * half], src[4 * half + 1], src[4 * half + 2], src[4 * half + 3]};
        }
    };
    auto store_k = [&](uint32_t buf, const Piece& piece) __attribute__((always_inline)) {
        uint16_t* s = s_k0 + buf * kKTile;
        *reinterpret_cast<uint4v*>(s + k_st0) = halves_of(piece.k, 0);
        if constexpr (kTwo) *reinterpret_cast<uint4v*>(s + k_st1) = halves_of(piece.k, 1);
    };
    // Whether some row of the workgroup does not see some key of the tile that begins at key0.
    auto partial = [&](uint32_t key0) __attribute__((always_inline)) {
        return key0 + kBN > all_hi || (key0 < all_lo && key0 + kBN > p.sinks);
    };
    auto store_v = [&](uint32_t buf, uint32_t it, const At& at, const Piece& piece) __attribute__((always_inline)) {
        const uint32_t valid = of_lane(at) >> 31;
        uint16_t* s = s_v0 + buf * kVTile;
        uint4v x0 = halves_of(piece.v, 0), x1 = {0, 0, 0, 0};
        if constexpr (kTwo) x1 = halves_of(piece.v, 1);
        const uint32_t key0 = key_of(min(it, n_tiles - 1));
        if (partial(key0) || (kRows != kExContiguous && !valid)) {
            const uint32_t key = key0 + ld_r;
            bool special = drop_specials(x0);
            if constexpr (kTwo) special = drop_specials(x1) || special;
            if (!valid || key >= seen.end || (key < seen.lo && key >= p.sinks)) {
                x0 = x1 = uint4v{0, 0, 0, 0};
                special = false;
            }
            if (special) *s_special = 1;
        }
        *reinterpret_cast<uint4v*>(s + v_st0) = x0;
        if constexpr (kTwo) *reinterpret_cast<uint4v*>(s + v_st1) = x1;
    };

    // ---- V^T operand reads through ds_read_b64_tr_b16 (see prefill.hip): 16-lane group q4, lane 4 k4 + r4 of it points
    // at key 4 g + k4, head-dim elements 32 t + 16 (q4 & 1) + 8 (r4 & 1) + 4 (r4 >> 1) .. + 3
    uint32_t vt_off[kBlocks];
    {
        const uint32_t q4 = lane >> 4, i16 = lane & 15, k4 = i16 >> 2, r4 = i16 & 3, key = 4 * g + k4;
        const uint32_t in_chunk = 16 * (q4 & 1) + 8 * (r4 & 1) + 4 * (r4 >> 1);
#pragma unroll
        for (uint32_t t = 0; t < uint32_t(kBlocks); t++) vt_off[t] = key * kVPitch + (((t ^ (k4 & kSwz)) << 5) | in_chunk);
    }
    auto v_pair = [&](const uint16_t* vp) __attribute__((always_inline)) -> half8 {
        const uint2v lo = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4v __attribute__((address_space(3)))*)(vp)));
        const uint2v hi = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4v __attribute__((address_space(3)))*)(vp + 8 * kVPitch)));
        return ex_half8(uint4v{lo.x, lo.y, hi.x, hi.y});
    };

    // ---- per-tile pieces of a wave
    struct Run {
        float scale, lvs, inv;
    };
    struct Runs {
        Run r[kLaneRuns];
        uint32_t bits;  // of those whose page is one of the pool's; kFarScale
    };
    constexpr uint32_t kAllRuns = (1u << kLaneRuns) - 1;
    // positive and finite, so that a masked score stays minus infinity and a product of zero stays zero
    auto factor_of = [&](float ks) __attribute__((always_inline)) {
        return kQF32 ? __builtin_amdgcn_fmed3f(ks * q_unit, 0x1p-126f, FLT_MAX) : q_unit;
    };
    auto runs_of = [&](uint32_t it, int sub) __attribute__((always_inline)) -> Runs {
        Runs x;
        x.bits = kAllRuns;
        if constexpr (kRows == kExContiguous) {
            x.r[0] = x.r[1] = Run{factor_of(1.0f), 0.0f, 1.0f};
        } else {
            const uint32_t at = (it - t_begin) % (2 * kPlan) * kTileRuns + (kTileRuns / 2) * sub + (kFine ? g : 0);
            x.bits = 0;
#pragma unroll
            for (int a = 0; a < kLaneRuns; a++) {
                const float4v r = s_run[at + (kFine ? 2 * a : a)];
                x.bits |= __float_as_uint(r.w);
                x.r[a] = kF8 ? Run{kQF32 ? factor_of(r.x) : r.x, r.y, r.z} : Run{factor_of(1.0f), 0.0f, 1.0f};
            }
            if constexpr (!kFine) x.bits = ex_uniform(x.bits);
        }
        return x;
    };
    // keys of the sub-tile at key0 that the lane's row does not see become minus infinity
    auto apply_mask = [&](uint32_t key0, uint32_t bits, float16v& s) __attribute__((always_inline)) {
        if (key0 + 32 <= every_hi && (key0 >= every_lo || key0 + 32 <= p.sinks) && (kFine ? __all((bits & kAllRuns) == kAllRuns) : (bits & kAllRuns) == kAllRuns)) return;
        // what depends on the lane goes into three numbers, the rest is a constant per element; no short-circuit logic,
        // so that it stays compares and selects
        const int32_t base = int32_t(key0 + 4 * g), lo = int32_t(row_lo) - base, sink = int32_t(p.sinks) - base;
        int32_t hi[kLaneRuns];
#pragma unroll
        for (int a = 0; a < kLaneRuns; a++) hi[a] = (bits >> a) & 1u ? int32_t(row_hi) - base : -1;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int32_t in = 8 * (r >> 2) + (r & 3);
            const bool vis = bool(int(in < hi[r >> kRunShift]) & (int(in >= lo) | int(in < sink)));
            s[r] = vis ? s[r] : -INFINITY;
        }
    };
    auto scores = [&](uint32_t kbuf, int sub, float16v& out) __attribute__((always_inline)) {
        const uint16_t* krow = s_k0 + kbuf * kKTile + (32 * sub + n) * kKPitch + 8 * g;
        float16v c = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
            const half8 a = ex_half8(*reinterpret_cast<const uint4v*>(krow + 16 * s));
            c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, bq[s], c, 0, 0, 0);
            if constexpr (kQF32) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, bq_lo[s], c, 0, 0, 0);
        }
        out = c;
    };
    struct Probs {
        half8 hi[2];
        half8 lo[kPrecise ? 2 : 1];
    };
    // Probabilities are relative to a reference that moves only when those of a sub-tile sum to kProbLimit or more
    // (or to infinity, as in the first), see prefill.hip.  In front of the exponential a score is fused with its
    // factor and the reference.  What the reference's own rounding leaves there, up to half its last place, is nothing while
    // it is below 2^20 but beyond a float's exponents from 2^30 on: a row whose reference is that large has every sub-tile done
    // again with rounded scores (limit 0), whose difference to the reference is exact.
    auto rounded_score = [&](float s, float scale) __attribute__((always_inline)) {
#pragma clang fp contract(off)
        return s * scale;
    };
    auto rebase = [&](const float16v& s, const Runs& runs) __attribute__((always_inline)) {
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; r++) top = fmaxf(top, rounded_score(s[r], runs.r[r >> kRunShift].scale) + runs.r[r >> kRunShift].lvs);
        const LanePair both = half_wave_pair(top);
        const float m_new = fmaxf(m_ref, fmaxf(both.lo, both.hi));
        // (in two steps for the sum, which can be 2^100 times larger than the probabilities)
        const float root = fast_exp2(0.5f * (m_ref - m_new)), alpha = root * root;
        m_ref = m_new;
        if (!(fabsf(m_ref) < kFusedScores) && m_ref != kExNegBig) limit = 0.0f;
        l_run = l_run * root * root;
#pragma unroll
        for (int t = 0; t < kBlocks; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) oacc[t][r] *= alpha;
    };
    auto pack = [&](const float* pe, half8& hi, half8* lo) __attribute__((always_inline)) {  // 8 probabilities
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const _Float16 h = static_cast<_Float16>(pe[j]);
            hi[j] = h;
            if constexpr (kPrecise) (*lo)[j] = static_cast<_Float16>(pe[j] - static_cast<float>(h));
        }
    };
    // sum[a]: of the probabilities of run a
    auto probabilities_once = [&](const float16v& s, const Runs& runs, Probs& out, float (&sum)[kLaneRuns]) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < kLaneRuns; a++) sum[a] = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float pe[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int a = (8 * u + j) >> kRunShift;
                pe[j] = fast_exp2((rounded_score(s[8 * u + j], runs.r[a].scale) - m_ref) + runs.r[a].lvs);
                sum[a] += pe[j];
            }
            pack(pe, out.hi[u], &out.lo[kPrecise ? u : 0]);
        }
    };
    auto total_of = [&](const float (&sum)[kLaneRuns]) __attribute__((always_inline)) {
        float t = sum[0] + sum[1];
        if constexpr (kFine) t += sum[2] + sum[3];
        return t;
    };
    // The sum's weights of a sub-tile some of whose V scales are beyond 2^+-kPlainScales, and of every one behind a scale above
    // 2^kPlainScales, from which the reference may come: probabilities times 1 / (V scale) would have vanished where the
    // reference comes from a scale 2^102 larger (blocks of zeros, with the append's 2^-96, beside values of 1e4).  Taken from
    // the scores; the power of two is room towards the smallest float, and 2^100, the inverse of the smallest scale, times it
    // is in range.
    auto far_weights = [&](const float16v& s, const Runs& runs, float (&sum)[kLaneRuns]) __attribute__((always_inline)) {
        float t = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; r++) t += fast_exp2((rounded_score(s[r], runs.r[r >> kRunShift].scale) - m_ref) + 20.0f);
        l_run += t * 0x1p-20f;
#pragma unroll
        for (int a = 0; a < kLaneRuns; a++) sum[a] = 0.0f;
    };
    auto accumulate = [&](uint32_t vbuf, int sub, const Probs& pr) __attribute__((always_inline)) {
        const uint16_t* sv = s_v0 + vbuf * kVTile + 32 * sub * kVPitch;
#pragma unroll
        for (int t = 0; t < kBlocks; t++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const half8 a = v_pair(sv + vt_off[t] + 16 * u * kVPitch);
                oacc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pr.hi[u], oacc[t], 0, 0, 0);
                if constexpr (kPrecise) oacc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pr.lo[u], oacc[t], 0, 0, 0);
            }
    };
    // One phase of the pipeline: scores of sub-tile j + 1 (key0_q, buffer kbuf), softmax of j (s_in, runs_in), second
    // product of j - 1.  `side(step)` is the caller's work in the shadow of the MFMAs.
    auto fused_phase = [&](uint32_t it_q, uint32_t key0_q, uint32_t kbuf, int sub_q, float16v& s_out, const float16v& s_in, const Runs& runs_in,
                           Probs& p_out, uint32_t vbuf, int sub_v, const Probs& p_prev, auto&& side) __attribute__((always_inline)) {
        const uint16_t* krow = s_k0 + kbuf * kKTile + (32 * sub_q + n) * kKPitch + 8 * g;
        const uint16_t* sv = s_v0 + vbuf * kVTile + 32 * sub_v * kVPitch;
        auto k_operand = [&](int s) __attribute__((always_inline)) { return ex_half8(*reinterpret_cast<const uint4v*>(krow + 16 * s)); };
        auto v_operand = [&](int i) __attribute__((always_inline)) { return v_pair(sv + vt_off[i % kBlocks] + 16 * (i / kBlocks) * kVPitch); };
        constexpr int kRing = 3;
        half8 ring[kRing];
#pragma unroll
        for (int i = 0; i < kRing - 1; i++) ring[i] = k_operand(i);
        float16v c = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        float shift[kLaneRuns], psum[kLaneRuns];
#pragma unroll
        for (int a = 0; a < kLaneRuns; a++) {
            shift[a] = runs_in.r[a].lvs - m_ref;
            psum[a] = 0.0f;
        }
        float pe[16];
        uint32_t pw[8], pl[kPrecise ? 8 : 1];
        float tn = __builtin_fmaf(s_in[0], runs_in.r[0].scale, shift[0]);
        auto finish = [&](int i) __attribute__((always_inline)) {  // elements 2 i, 2 i + 1
            pw[i] = pack_f16x2(pe[2 * i], pe[2 * i + 1]);
            if constexpr (kPrecise) {
                const half2v h = __builtin_bit_cast(half2v, pw[i]);
                pl[i] = pack_f16x2(pe[2 * i] - static_cast<float>(h.x), pe[2 * i + 1] - static_cast<float>(h.y));
                asm volatile("" : "+v"(pl[i]));
            }
            asm volatile("" : "+v"(pw[i]));
        };
        auto softmax_step = [&](int e) __attribute__((always_inline)) {
            pe[e] = fast_exp2(tn);
            if (e < 15) tn = __builtin_fmaf(s_in[e + 1], runs_in.r[(e + 1) >> kRunShift].scale, shift[(e + 1) >> kRunShift]);
            if (e > 0) psum[(e - 1) >> kRunShift] += pe[e - 1];
            if (e > 0 && (e & 1) == 0) finish(e / 2 - 1);
            asm volatile("" : "+v"(pe[e]), "+v"(tn), "+v"(psum[e >> kRunShift]));
            if (e > 0) asm volatile("" : "+v"(psum[(e - 1) >> kRunShift]));
        };
        constexpr int kPer = 16 / kPhase;
        auto vector_work = [&](int step) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < kPer; j++) softmax_step(step * kPer + j);
            side(step);
        };
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
            if (s + kRing - 1 < kSteps) ring[(s + kRing - 1) % kRing] = k_operand(s + kRing - 1);
            c = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[s % kRing], bq[s], c, 0, 0, 0);
            if constexpr (kQF32) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[s % kRing], bq_lo[s], c, 0, 0, 0);
            vector_work(s);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < kRing - 1; i++) ring[i] = v_operand(i);
        apply_mask(key0_q, kRows == kExContiguous ? kAllRuns : runs_of(it_q, sub_q).bits, c);  // rare
#pragma unroll
        for (int i = 0; i < 2 * kBlocks; i++) {
            if (i + kRing - 1 < 2 * kBlocks) ring[(i + kRing - 1) % kRing] = v_operand(i + kRing - 1);
            oacc[i % kBlocks] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % kRing], p_prev.hi[i / kBlocks], oacc[i % kBlocks], 0, 0, 0);
            if constexpr (kPrecise)
                oacc[i % kBlocks] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % kRing], p_prev.lo[i / kBlocks], oacc[i % kBlocks], 0, 0, 0);
            vector_work(kSteps + i);
            __builtin_amdgcn_sched_barrier(0);
        }
        psum[kLaneRuns - 1] += pe[15];
        finish(7);
        p_out.hi[0] = ex_half8(uint4v{pw[0], pw[1], pw[2], pw[3]});
        p_out.hi[1] = ex_half8(uint4v{pw[4], pw[5], pw[6], pw[7]});
        if constexpr (kPrecise) {
            p_out.lo[0] = ex_half8(uint4v{pl[0], pl[1], pl[2], pl[3]});
            p_out.lo[1] = ex_half8(uint4v{pl[4], pl[5], pl[6], pl[7]});
        }
        if (__any(!(total_of(psum) < limit) || (kF8 && (runs_in.bits & kFarScale)))) {  // rare: the reference has to move, redo the sub-tile
            rebase(s_in, runs_in);
            probabilities_once(s_in, runs_in, p_out, psum);
            if constexpr (kF8) {
                bool high = false;
#pragma unroll
                for (int a = 0; a < kLaneRuns; a++) high = high || runs_in.r[a].lvs > kPlainScales;
                if (__any(high)) limit = 0.0f;  // this way from here on
                if (__any((runs_in.bits & kFarScale) || limit == 0.0f)) far_weights(s_in, runs_in, psum);
            }
        }
#pragma unroll
        for (int a = 0; a < kLaneRuns; a++) l_run += psum[a] * runs_in.r[a].inv;
        s_out = c;
    };

    if (tid == 0) *s_special = 0;
    __syncthreads();
    if (t_begin < n_tiles) {  // uniform; an empty share writes a neutral partial
        // Tiles this wave computes: up to the last one that holds a key some row of it sees (one in front of a later
        // window's first is masked whole).  There is one code path: both
        // phases run in every iteration, and where a stage does not apply yet it works on zero probabilities.
        uint32_t my_end = t_begin;
        if (wave_active)
            for (uint32_t it = n_tiles; it > t_begin; it--)
                if (key_of(it - 1) < wave_hi) {
                    my_end = it;
                    break;
                }

        // ---- prologue: in LDS K of the first two tiles and V of the first, in flight K of the third and V of the second, and
        // the rows of the first 64.  An iteration is long enough for what is loaded in one to be there in the next (a second
        // piece in flight gained nothing and cost registers: 935 us for 512 queries with float results at 32768, 895 without).
        Piece a;
        Plan cur = plan_rows(0, plan_entries(0));
        Plan next = cur;
        auto row_of = [&](uint32_t j) __attribute__((always_inline)) -> At {
            At at;
#pragma unroll
            for (int f = 0; f < kPieceRuns; f++) at.row[f] = uint32_t(__builtin_amdgcn_readlane(int(cur.row[f]), int(j % kPlan)));
            return at;
        };
        const At o0 = row_of(0), o1 = row_of(1), o2 = row_of(2);
        {
            Piece b;
            load_k(o0, a);
            load_v(o0, a);
            load_k(o1, b);
            plan_runs(cur, 0);
            plan_runs(cur, 1);  // (tiles behind the last, whose scores nobody takes, find numbers)
            store_k(0, a);
            store_v(0, t_begin, o0, a);
            store_k(1, b);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(o2, a);
        load_v(o1, a);
        __builtin_amdgcn_sched_barrier(0);
        At at_v = o2, at_v1 = o1;  // of the tile whose V is loaded next, and of the one whose V is in flight
        __syncthreads();

        float16v s0, s1;
        Probs p_old, p_new;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            p_old.hi[u] = half8{0, 0, 0, 0, 0, 0, 0, 0};
            if constexpr (kPrecise) p_old.lo[u] = p_old.hi[u];
        }
        if (my_end > t_begin) {
            scores(0, 0, s0);
            apply_mask(key_of(t_begin), runs_of(t_begin, 0).bits, s0);
        }
        uint32_t kb_cur = 0, kb_next = 1, kb_store = 2;
        // (the first iteration's second product, of nothing, reads the first tile's V: whatever it holds, every row sees it)
        uint32_t vb_prev = 0, vb_cur = 0, vb_store = 1;
        auto staging = [&](uint32_t it, int part) __attribute__((always_inline)) {
            if (part == 0) store_k(kb_store, a);                  // K of tile it + 2
            if (part == 2) store_v(vb_store, it + 1, at_v1, a);  // V of tile it + 1
            if (part == 4) {  // K of it + 3, V of it + 2
                const uint32_t j = it + 3 - t_begin;
                if (j % kPlan == 0) cur = next;
                const At at_k = row_of(j);
                load_k(at_k, a);
                load_v(at_v, a);
                at_v1 = at_v;
                at_v = at_k;
            }
            if (part == 5) {
                // the next 64 tiles.  In one go, with two waits for memory: what three steps a few tiles apart would carry from
                // one to the next costs more in registers (512 at 32768: 541 us, so 534; with float queries and results over
                // blocks of 8 tokens, 24407 keys, 1353 and 1148)
                const uint32_t j = it + 3 - t_begin, block = j / kPlan + 1;
                if (j % kPlan == 40 && t_begin + block * kPlan < n_tiles) {
                    next = plan_rows(block, plan_entries(block));
                    plan_runs(next, block & 1);
                }
            }
        };
        auto rotate_buffers = [&]() __attribute__((always_inline)) {
            __syncthreads();
            const uint32_t kf = kb_cur;
            kb_cur = kb_next;
            kb_next = kb_store;
            kb_store = kf;
            vb_prev = vb_cur;
            vb_cur = vb_store;
            vb_store = 3 - vb_prev - vb_cur;
        };
        // At head size 64 a phase has too few MFMAs to cover all of the staging: it is spread over both (196 us against
        // 204 for 4096 queries with a window of 4096; at 128 the second phase covers nothing more: 550 against 538 for 512 at 32768).
        constexpr bool kSpread = kD == 64;
        auto iteration = [&](uint32_t it) __attribute__((always_inline)) {
            const uint32_t key_cur = key_of(it), key_nxt = key_of(it + 1);
            const Runs ra = runs_of(it, 0);
            fused_phase(it, key_cur + 32, kb_cur, 1, s1, s0, ra, p_new, vb_prev, 1, p_old, [&](int step) {
                const int part = step - (kPhase - 8);
                if (!kSpread || part == 0) staging(it, part);
            });
            const Runs rb = runs_of(it, 1);
            fused_phase(it + 1, key_nxt, kb_next, 0, s0, s1, rb, p_old, vb_cur, 0, p_new, [&](int step) {
                const int part = step - (kPhase - 8) + 2;
                if (kSpread && part >= 2) staging(it, part);
            });
            rotate_buffers();
        };
        auto stage_only = [&](uint32_t it) __attribute__((always_inline)) {
#pragma unroll
            for (int part = 0; part < 6; part++) staging(it, part);
            rotate_buffers();
        };
        uint32_t it = t_begin;
        for (; it < my_end; it++) iteration(it);
        if (my_end > t_begin) accumulate(vb_prev, 1, p_old);
        for (; it < n_tiles; it++) stage_only(it);
    }

    if (!wave_active) return;
    {
        const LanePair both = half_wave_pair(l_run);
        l_run = both.lo + both.hi;
    }
    if (!row_live) return;
    // Accumulator [t][4 a + b] is head-dim element 32 t + 16 (a >> 1) + 8 g + 4 (a & 1) + b: 8 consecutive per (t, a >> 1).
    bool nan = false;  // infinities of V may have come out as NaN, through a probability's remainder or an underflow to zero
    if constexpr (!kF8) {
#pragma unroll
        for (int t = 0; t < kBlocks; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) nan = nan || oacc[t][r] != oacc[t][r];
        nan = nan && l_run < INFINITY;
        if (nan) {
#pragma unroll
            for (int t = 0; t < kBlocks; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) oacc[t][r] = oacc[t][r] != oacc[t][r] ? 0.0f : oacc[t][r];
        }
    }
    if (t_begin < n_tiles && (*s_special || nan)) {
        // the infinities and NaNs of V that were left out in tiles that not every row sees, or all of them (rare)
        for (uint32_t it = t_begin; it < n_tiles; it++) {
            const uint32_t key0 = key_of(it);
            if (!nan && !partial(key0)) continue;
            for (uint32_t key = key0; key < min(key0 + kBN, row_hi); key++) {
                if (key < row_lo && key >= p.sinks) continue;
                uint32_t at = key;
                if constexpr (kRows != kExContiguous) {
                    const uint32_t blk = key / p.block_size;
                    if (!pool_row(p.tables[blk], key - blk * p.block_size, p.block_size, p.num_blocks, &at)) continue;
                }
                const uint8_t* v = p.v + int64_t(kvh) * p.head_bytes + int64_t(at) * p.row_bytes;
#pragma unroll
                for (int t = 0; t < kBlocks; t++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const uint32_t d = 32 * t + 16 * (r >> 3) + 8 * g + (r & 7);
                        if constexpr (kF8) {
                            if ((v[d] & 0x7Fu) == 0x7Fu) oacc[t][r] = NAN;
                        } else {
                            const float x = static_cast<float>(reinterpret_cast<const _Float16*>(v)[d]);
                            if (!(fabsf(x) < INFINITY)) oacc[t][r] += x;
                        }
                    }
            }
        }
    }
    if (p.n_splits > 1) {
        const size_t at = (size_t(split) * p.num_kv_heads + kvh) * n_rows + row;
        float* po = p.part_o + at * kD;
#pragma unroll
        for (int t = 0; t < kBlocks; t++)
#pragma unroll
            for (int ah = 0; ah < 2; ah++) {
                float* op = po + 32 * t + 16 * ah + 8 * g;
                *reinterpret_cast<float4v*>(op) = float4v{oacc[t][8 * ah], oacc[t][8 * ah + 1], oacc[t][8 * ah + 2], oacc[t][8 * ah + 3]};
                *reinterpret_cast<float4v*>(op + 4) = float4v{oacc[t][8 * ah + 4], oacc[t][8 * ah + 5], oacc[t][8 * ah + 6], oacc[t][8 * ah + 7]};
            }
        if (g == 0) {
            p.part_ml[at * 2] = m_ref;
            p.part_ml[at * 2 + 1] = l_run;
        }
        return;
    }
    const bool none = l_run == 0.0f;  // the row sees no key
    const float inv_l = none ? 0.0f : 1.0f / l_run;
    const int64_t off = int64_t(query) * p.out_tok + int64_t(head) * p.out_head;
#pragma unroll
    for (int t = 0; t < kBlocks; t++)
#pragma unroll
        for (int ah = 0; ah < 2; ah++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = oacc[t][8 * ah + e] * inv_l;
            const uint32_t d = 32 * t + 16 * ah + 8 * g;
            if constexpr (kPrecise) {
                float* op = static_cast<float*>(p.out) + off + d;
                *reinterpret_cast<float4v*>(op) = float4v{x[0], x[1], x[2], x[3]};
                *reinterpret_cast<float4v*>(op + 4) = float4v{x[4], x[5], x[6], x[7]};
            } else {
                uint4v w;
                w.x = pack_f16x2(x[0], x[1]);
                w.y = pack_f16x2(x[2], x[3]);
                w.z = pack_f16x2(x[4], x[5]);
                w.w = pack_f16x2(x[6], x[7]);
                *reinterpret_cast<uint4v*>(static_cast<uint16_t*>(p.out) + off + d) = w;
            }
        }
    if (p.lse && g == 0)
        p.lse[int64_t(head) * p.lse_head + query] = none ? -INFINITY : (m_ref + __builtin_amdgcn_logf(l_run)) * kExLn2;
}

// Joins the key splits of 2048 / D rows of one KV head: a thread per eight head-dim elements.
template <bool kOutF32, int kD>
__global__ void __launch_bounds__(256) kv_tiles_merge_kernel(KvParams p) {
    constexpr uint32_t kLanes = kD / 8;
    const uint32_t n_rows = p.seq_q * p.group, kvh = blockIdx.y;
    const uint32_t row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes, dc = threadIdx.x % kLanes;
    if (row >= n_rows) return;
    float mx = kExNegBig, l = 0.0f;
    float o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (uint32_t s0 = 0; s0 < p.n_splits; s0 += 4) {  // four at a time: their loads are in flight together
        float m[4], ls[4];
        float4v a[4], b[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const size_t at = (size_t(min(s0 + i, p.n_splits - 1)) * p.num_kv_heads + kvh) * n_rows + row;
            m[i] = p.part_ml[at * 2];
            ls[i] = p.part_ml[at * 2 + 1];
            a[i] = *reinterpret_cast<const float4v*>(p.part_o + at * kD + 8 * dc);
            b[i] = *reinterpret_cast<const float4v*>(p.part_o + at * kD + 8 * dc + 4);
        }
        float m_new = mx;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) m_new = fmaxf(m_new, s0 + i < p.n_splits ? m[i] : kExNegBig);
        const float keep_root = fast_exp2(0.5f * (mx - m_new)), keep = keep_root * keep_root;  // two steps as in rebase
        l = l * keep_root * keep_root;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] *= keep;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            if (s0 + i >= p.n_splits) continue;
            const float root = fast_exp2(0.5f * (m[i] - m_new)), f = root * root;
            l += ls[i] * root * root;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                o[e] += a[i][e] * f;
                o[4 + e] += b[i][e] * f;
            }
        }
        mx = m_new;
    }
    const bool none = l == 0.0f;
    const float inv_l = none ? 0.0f : 1.0f / l;
    const uint32_t query = row / p.group, head = kvh * p.group + row % p.group;
    const int64_t off = int64_t(query) * p.out_tok + int64_t(head) * p.out_head + 8 * dc;
    float x[8];
    // (a piece's infinity times a weight that has vanished is NaN here, as in the other kernels' sums)
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = settle_nan(p, o[e] * inv_l, l, 0, kvh, p.start_pos + query, p.max_tokens, 8 * dc + e);
    if constexpr (kOutF32) {
        float* op = static_cast<float*>(p.out) + off;
        *reinterpret_cast<float4v*>(op) = float4v{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<float4v*>(op + 4) = float4v{x[4], x[5], x[6], x[7]};
    } else {
        uint4v w;
        w.x = pack_f16x2(x[0], x[1]);
        w.y = pack_f16x2(x[2], x[3]);
        w.z = pack_f16x2(x[4], x[5]);
        w.w = pack_f16x2(x[6], x[7]);
        *reinterpret_cast<uint4v*>(static_cast<uint16_t*>(p.out) + off) = w;
    }
    if (p.lse && dc == 0) p.lse[int64_t(head) * p.lse_head + query] = none ? -INFINITY : (mx + __builtin_amdgcn_logf(l)) * kExLn2;
}

template <bool kQF32, bool kPrecise, bool kF8, int kRows, int kD>
int launch_one(const KvParams& p, dim3 grid) {
    auto kernel = kv_tiles_kernel<kQF32, kPrecise, kF8, kRows, kD>;
    static bool configured[kMaxDevices];
    if (int rc = raise_dynamic_lds_limit(reinterpret_cast<const void*>(kernel), Shape<kD, kRows>::kLdsBytes, configured)) return rc;
    kernel<<<grid, dim3(kThreads), Shape<kD, kRows>::kLdsBytes, ctx().stream>>>(p);
    return launch_status();
}
template <bool kQF32, bool kPrecise, int kD>
int launch_cache(const KvParams& p, dim3 grid, bool f8, int rows) {
    if (f8 && rows == kExPaged16) return launch_one<kQF32, kPrecise, true, kExPaged16, kD>(p, grid);
    if (f8) return launch_one<kQF32, kPrecise, true, kExPaged4, kD>(p, grid);
    if (rows == kExPaged4) return launch_one<kQF32, kPrecise, false, kExPaged4, kD>(p, grid);
    if (rows == kExPaged16) return launch_one<kQF32, kPrecise, false, kExPaged16, kD>(p, grid);
    return launch_one<kQF32, kPrecise, false, kExContiguous, kD>(p, grid);
}
template <int kD>
int launch_types(const KvParams& p, dim3 grid, bool q_f32, bool f8, int rows) {
    if (q_f32 && p.out_f32) return launch_cache<true, true, kD>(p, grid, f8, rows);
    if (q_f32) return launch_cache<true, false, kD>(p, grid, f8, rows);
    if (p.out_f32) return launch_cache<false, true, kD>(p, grid, f8, rows);
    return launch_cache<false, false, kD>(p, grid, f8, rows);
}

}  // namespace

int launch_kv_tiles(KvParams p, const KvCall& call, bool q_f32, int rows, const ScratchSource& scratch) {
    const uint32_t D = call.head_dim;
    const bool f8 = call.f8;
    const uint64_t n_rows = uint64_t(p.seq_q) * p.group;
    p.q_tiles = uint32_t((n_rows + kBM - 1) / kBM);
    // With a window every row sees about as many keys, and behind a long prefix nearly as many.
    p.paired = p.causal && p.window == 0 && p.start_pos < 4 * uint64_t(p.seq_q);
    // the factor of the scores is positive in the kernel (see the runs' scales there): a negative one's sign, and the
    // zero of a zero one, go to Q
    p.q_sign = p.scale_log2 > 0.0f ? 1.0f : p.scale_log2 < 0.0f ? -1.0f : 0.0f;
    p.scale_log2 = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2);
    const uint64_t wgs = uint64_t(p.q_tiles) * p.num_kv_heads;
    p.n_splits = kv_tiles_cut(call).pieces;
    const size_t slots = p.n_splits > 1 ? size_t(p.n_splits) * p.num_kv_heads * n_rows : 0;
    const size_t need = slots * (D + 2) * sizeof(float);
    if (scratch.query) {
        *scratch.query = need;
        return GRANITE_HIP_OK;
    }
    if (wgs * p.n_splits > 0x7FFFFFFFull || p.num_kv_heads > 65535u) return GRANITE_HIP_EINVAL;
    if (need > 0) {
        void* ws = nullptr;
        if (int rc = take_scratch(scratch, need, &ws)) return rc;
        p.part_o = static_cast<float*>(ws);
        p.part_ml = p.part_o + slots * D;
    }
    int rc;
    {
        KernelTimerScope timer("attention_ex");
        const dim3 grid(uint32_t(wgs * p.n_splits));
        rc = D == 128 ? launch_types<128>(p, grid, q_f32, f8, rows) : launch_types<64>(p, grid, q_f32, f8, rows);
    }
    if (rc != GRANITE_HIP_OK || p.n_splits == 1) return rc;
    {
        KernelTimerScope timer("attention_ex_merge");
        const dim3 grid(uint32_t((n_rows + 2048 / D - 1) / (2048 / D)), p.num_kv_heads), block(256);
        hipStream_t st = ctx().stream;
        if (D == 128) {
            if (p.out_f32) kv_tiles_merge_kernel<true, 128><<<grid, block, 0, st>>>(p);
            else kv_tiles_merge_kernel<false, 128><<<grid, block, 0, st>>>(p);
        } else {
            if (p.out_f32) kv_tiles_merge_kernel<true, 64><<<grid, block, 0, st>>>(p);
            else kv_tiles_merge_kernel<false, 64><<<grid, block, 0, st>>>(p);
        }
    }
    return launch_status();
}

}  // namespace ghip
