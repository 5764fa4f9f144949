// Building blocks of the attention kernels over 8-bit pools and windowed caches (decode_ex.hip,
// attention_ex.hip): the launch parameters and the work of one wave on one key tile.
#pragma once

#include <cfloat>

#include "common.h"
#include "kv_choice.h"
#include "kv_visible.h"

namespace ghip {

constexpr float kExLog2e = 1.4426950408889634f;
constexpr float kExLn2 = 0.6931471805599453f;
constexpr float kExNegBig = -FLT_MAX;  // what a running maximum starts from: at or below any finite score

// How token positions map to rows.  Runs of 16 consecutive tokens that start at a multiple of 16 lie in
// one block when the block size is a multiple of 16: one table entry, one scale and one base address
// then serve 16 tokens and stay in scalar registers.  kExPaged4, runs of 4, is the tiles kernel's only.
enum : int { kExContiguous = 0, kExPaged16 = 1, kExPagedAny = 2, kExPaged4 = 3 };

struct KvParams {
    const void* q;
    int64_t q_batch, q_tok, q_head;  // element strides
    const uint8_t* k;
    const uint8_t* v;
    const float* k_scale;  // 8-bit pools: [num_blocks, num_kv_heads]
    const float* v_scale;
    const int32_t* tables;
    const int32_t* seq_lens;
    void* out;
    int64_t out_batch, out_tok, out_head;
    float* lse;
    int64_t lse_batch, lse_tok, lse_head;
    float* part_o;  // split launches: unnormalised partial outputs
    float* part_ml;
    uint32_t* plan;
    uint32_t batch, seq_q, num_heads, num_kv_heads, group;
    uint32_t q_groups;  // runs of 16 query heads that share a KV head
    uint32_t block_size, max_blocks, num_blocks;
    int bs_shift;        // log2(block_size), -1 where it is no power of two
    int64_t row_bytes;   // between consecutive rows of one KV head
    int64_t head_bytes;  // between KV heads of one row
    uint32_t max_tokens; // bound on any length
    int decode;          // one query per sequence, at the sequence's last position
    int causal;
    int out_f32;
    uint32_t start_pos, window, sinks;
    uint32_t n_splits, q_tiles;
    uint32_t paired;     // tiles kernel: late and early runs of rows share a workgroup
    uint32_t workers, min_per, part_cap;
    float scale_log2;
    float q_sign;  // tiles kernel: 1, -1 or 0, taken into Q
};

// decode_ex_stream.hip: the persistent kernels, tiles of 32 tokens.  tiles_per_seq: most tiles a sequence can have to visit.
constexpr uint32_t kStreamMaxBatch = 2560;  // sequences of a launch: larger batches go in parts
bool kv_stream_supports(const KvParams& p, bool f8, int rows, uint32_t tiles_per_seq);
int launch_kv_stream(KvParams p, uint32_t D, bool q_f32, bool f8, int rows, uint32_t tiles_per_seq, const ScratchSource& scratch);
// decode_ex_dma.hip: the one over 8-bit pools, through LDS; p as launch_kv_stream has it.
size_t kv_dma_lds_bytes(uint32_t D, uint32_t batch);
int launch_kv_dma(const KvParams& p, uint32_t D, bool q_f32, uint32_t per_list, dim3 grid);
// attention_ex.hip: the tiles kernel.  Block sizes are multiples of 4, or the cache is contiguous.
int launch_kv_tiles(KvParams p, const KvCall& call, bool q_f32, int rows, const ScratchSource& scratch);

#if defined(__HIPCC__)

__device__ __forceinline__ half8 ex_half8(uint4v x) { return __builtin_bit_cast(half8, x); }

__device__ __forceinline__ uint32_t ex_lane_read(uint32_t v, uint32_t src_lane) {
    return uint32_t(__builtin_amdgcn_ds_bpermute(int(src_lane << 2), int(v)));
}
__device__ __forceinline__ uint32_t ex_uniform(uint32_t v) {
    return uint32_t(__builtin_amdgcn_readfirstlane(int(v)));
}

// Two e4m3 codes (the low or the high half of `w`) as two halves.  Exact: a half holds every e4m3 value.
template <bool kHigh>
__device__ __forceinline__ uint32_t f8x2_to_f16x2(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(int(w), 1.0f, kHigh));
}
__device__ __forceinline__ half8 f8x8_to_half8(uint32_t a, uint32_t b) {
    return ex_half8(uint4v{f8x2_to_f16x2<false>(a), f8x2_to_f16x2<true>(a), f8x2_to_f16x2<false>(b), f8x2_to_f16x2<true>(b)});
}

// Probabilities enter the second product times this, and over 8-bit pools times the V scale over 2^bound, where 2^bound is the
// largest p * (V scale) among the keys that the row itself has seen: it is then near 2^14, 65504 being out of reach, and what is
// up to 2^28 times smaller keeps 22 bits in a half and its remainder.  The scale goes into the exponent of the
// probability, which by itself might vanish.  (The bound has to follow the probabilities: taken from the scales alone, a
// block of next to no probability whose scale is 2^40 times the others' left nothing of these.  One for the wave with a
// change to one for every row where scales lie 2^7 apart is as quick.)
constexpr float kExBoost = 16384.0f;

__device__ __forceinline__ float ex_power(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }
// A V scale as mantissa (0.5 <= . < 1) and exponent.
__device__ __forceinline__ float ex_exponent(float vs) { return float(__builtin_amdgcn_frexp_expf(vs)); }
__device__ __forceinline__ float ex_mantissa(float vs) { return __builtin_amdgcn_frexp_mantf(vs); }
// A product as a half and the half remainder of it.  The product is pinned as the float it rounds to: where the compiler
// may fuse it, it took the half of the exact product for the remainder and that of the rounded one for the operand, and where
// the two lie either side of a tie the pair was half a step of a half, 2^-11, off.
__device__ __forceinline__ void ex_split(float product, _Float16& half, _Float16& rest) {
    asm volatile("" : "+v"(product));
    half = static_cast<_Float16>(product);
    rest = static_cast<_Float16>(product - static_cast<float>(half));
}

// What an accumulator relative to `bound` (log2, see Rows16) counts.
__device__ __forceinline__ float ex_unit(float bound) { return __builtin_ldexpf(1.0f / kExBoost, int(fmaxf(ceilf(bound), -200.0f))); }

__device__ __forceinline__ uint32_t ex_seq_len(const KvParams& p, uint32_t b) {
    const uint32_t len = p.seq_lens ? uint32_t(max(p.seq_lens[b], 0)) : p.max_tokens;
    return min(len, p.max_tokens);
}

// The work of one wave on one key tile, for up to 16 query rows (MFMA columns) of one KV head.
//
//   S^T[tok, row] = K[tok, :] . Q[row, :]     v_mfma_f32_16x16x32_f16 per 16 tokens and 32 elements
//   softmax in the result layout: lane (n, g) holds row n, tokens 16 sub + 4 g + i
//   O^T[d, row]  += V^T[d, tok] . P^T[tok, row]
//
// A tile is 64 tokens of an 8-bit cache or 32 of a half one: 64 registers of K and V per lane either
// way.  K is the A operand as it lies in memory; the head-dim elements a lane holds for step s are
// d_of(s, g) .. + 7, an order that only Q has to share: the four lanes of a row read 64 consecutive bytes per
// instruction in either type.  V^T takes the tokens of a step in the order 4 g + j, 16 + 4 g + j, which is how the first
// product leaves the probabilities, and is put together from 4 x 4 byte (8 x 2 half) transposes with
// v_perm_b32; row m of output tile t is d = 8 m + t, so a lane ends with 32 consecutive elements.
// At head size 64 lanes 8 .. 15 of a group repeat the V loads of lanes 0 .. 7 and what they compute is dropped.
template <bool kF8, int kRows, int kD>
struct Tile {
    static constexpr int kSubs = kF8 ? 4 : 2;
    static constexpr uint32_t kTokens = 16 * kSubs;
    static constexpr int kSteps = kD / 32;
    static constexpr int kPairs = kSubs / 2;  // MFMA contractions (32 tokens) of the second product
    static constexpr int kKLoads = kF8 ? kD / 64 : kSteps;
    static constexpr int kVWords = kF8 ? 2 : 4;

    static __device__ __forceinline__ uint32_t d_of(int s, uint32_t g) {
        return kF8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
    }

    // Rows of a tile.  Paged16: lane l holds the row of token 16 (l & 3) of the tile (its 16-token
    // run) and the run's scales; else: of token l & (kTokens - 1).
    struct Rows {
        uint32_t row;
        float ks, vs;
        uint32_t valid;
    };
    // tok0: first token of the tile.  `seen`: what the launch's or workgroup's queries see between
    // them; the block table is not looked up beyond its end, and rows none of them sees have scale 0
    // (whatever lies in the scale array there must not count as the largest).
    // In two steps, so that the table entry can be in flight while other loads are issued.
    // needs_mask: whether some row that sees [lo, hi) and the sinks does not see some token of the tile,
    // invalid pages included (uniform).
    static __device__ __forceinline__ bool needs_mask(const KvParams& p, const Rows& r, uint32_t tok0, uint32_t lo, uint32_t hi) {
        bool m = tok0 + kTokens > hi || (tok0 < lo && tok0 + kTokens > p.sinks);
        if constexpr (kRows != kExContiguous) m = m || __any(r.valid == 0);
        return m;
    }
    struct Entry {
        int32_t entry;
        uint32_t in;  // row in the block; contiguous: the row
    };
    static __device__ __forceinline__ uint32_t first_of(uint32_t tok0, uint32_t lane) {
        return kRows == kExPaged16 ? tok0 + 16 * (lane & (kSubs - 1)) : tok0 + (lane & (kTokens - 1));
    }
    static __device__ __forceinline__ Entry entry_of(const KvParams& p, const int32_t* table, uint32_t tok0,
                                                     const VisibleTiles& seen, uint32_t lane) {
        Entry e;
        const uint32_t tok = min(first_of(tok0, lane), seen.end - 1);
        if constexpr (kRows == kExContiguous) {
            e.entry = 0;
            e.in = tok;
        } else {
            uint32_t blk;
            if (p.bs_shift >= 0) {
                blk = tok >> p.bs_shift;
                e.in = tok & (p.block_size - 1);
            } else {
                blk = tok / p.block_size;
                e.in = tok - blk * p.block_size;
            }
            // (a run whose first token is clamped is addressed from its start all the same)
            if constexpr (kRows == kExPaged16) e.in &= ~15u;
            e.entry = table[blk];
        }
        return e;
    }
    static __device__ __forceinline__ Rows rows_from(const KvParams& p, const Entry& e, uint32_t kvh, uint32_t tok0,
                                                     const VisibleTiles& seen, uint32_t lane) {
        Rows r;
        r.ks = r.vs = 1.0f;
        r.valid = 1;
        if constexpr (kRows == kExContiguous) {
            r.row = e.in;
        } else {
            r.valid = pool_row(e.entry, e.in, p.block_size, p.num_blocks, &r.row) ? 1u : 0u;
            if constexpr (kF8) {
                const uint32_t first = first_of(tok0, lane);
                const size_t at = size_t(r.valid ? uint32_t(e.entry) : 0u) * p.num_kv_heads + kvh;
                const bool used = bool(int(r.valid) & int(first < seen.end) &
                                       (int(first + (kRows == kExPaged16 ? 15 : 0) >= seen.lo) | int(first < p.sinks)));
                const float ks = p.k_scale[at], vs = p.v_scale[at];
                r.ks = used ? ks : 0.0f;
                r.vs = used ? vs : 0.0f;
            }
        }
        return r;
    }

    uint4v ka[kSubs][kKLoads];
    uint32_t vr[kSubs * 4][kVWords];  // token 16 (j / 4) + 4 g + j % 4 at d = 8 n

    // Paged16: a run of 16 rows is a buffer of its own whose base is scalar (pools may exceed the 4 GiB an offset
    // reaches, a run cannot), so a load needs no vector arithmetic: the lane's offset inside the run, the same for every
    // run, plus a scalar for the row of four (V) or an immediate (K).
    __device__ __forceinline__ void load(const KvParams& p, const Rows& r, uint32_t kvh, uint32_t lane) {
        const uint32_t n = lane & 15, g = lane >> 4;
        const uint8_t* kb = p.k + int64_t(kvh) * p.head_bytes;
        const uint8_t* vb = p.v + int64_t(kvh) * p.head_bytes;
        constexpr uint32_t kElem = kF8 ? 1 : 2;
        const uint32_t k_in = kElem * d_of(0, g), v_in = kElem * 8 * (n & (kD / 8 - 1));
        if constexpr (kRows == kExPaged16) {
            const uint32_t row_bytes = uint32_t(p.row_bytes);
            const int k_off = int(n * row_bytes + k_in), v_off = int(4 * g * row_bytes + v_in);
#pragma unroll
            for (int sub = 0; sub < kSubs; sub++) {
                const uint64_t at = uint64_t(uint32_t(__builtin_amdgcn_readlane(int(r.row), sub))) * row_bytes;
                const auto run = run_of(kb + at, row_bytes);
#pragma unroll
                for (int i = 0; i < kKLoads; i++)
                    ka[sub][i] = __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(run, k_off, 64 * i, 0));
            }
#pragma unroll
            for (int sub = 0; sub < kSubs; sub++) {
                const uint64_t at = uint64_t(uint32_t(__builtin_amdgcn_readlane(int(r.row), sub))) * row_bytes;
                const auto run = run_of(vb + at, row_bytes);
                // every byte of V is used once: streaming loads (bit 1 of the last operand)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (kF8) {
                        const uint2v w = __builtin_bit_cast(uint2v, __builtin_amdgcn_raw_buffer_load_b64(run, v_off, int(j * row_bytes), 2));
                        vr[4 * sub + j][0] = w.x;
                        vr[4 * sub + j][1] = w.y;
                    } else {
                        const uint4v w = __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(run, v_off, int(j * row_bytes), 2));
#pragma unroll
                        for (int i = 0; i < 4; i++) vr[4 * sub + j][i] = w[i];
                    }
                }
            }
            return;
        }
#pragma unroll
        for (int sub = 0; sub < kSubs; sub++) {
            const uint8_t* kp = kb + uint64_t(ex_lane_read(r.row, 16 * sub + n)) * uint64_t(p.row_bytes) + k_in;
#pragma unroll
            for (int i = 0; i < kKLoads; i++) ka[sub][i] = *reinterpret_cast<const uint4v*>(kp + 64 * i);
        }
#pragma unroll
        for (int j = 0; j < kSubs * 4; j++) {
            const uint8_t* vp = vb + uint64_t(ex_lane_read(r.row, 16 * (j / 4) + 4 * g + j % 4)) * uint64_t(p.row_bytes) + v_in;
            if constexpr (kF8) {
                const uint2v w = __builtin_nontemporal_load(reinterpret_cast<const uint2v*>(vp));
                vr[j][0] = w.x;
                vr[j][1] = w.y;
            } else {
                const uint4v w = __builtin_nontemporal_load(reinterpret_cast<const uint4v*>(vp));
#pragma unroll
                for (int i = 0; i < 4; i++) vr[j][i] = w[i];
            }
        }
    }
    // The 16 rows from `first` on as a buffer: raw 32-bit elements, reads behind its end give zero.
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t run_of(const uint8_t* first, uint32_t row_bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(first), 0, int(16 * row_bytes), 0x00020000);
    }

    // A operand of the first product: step s of sub-tile `sub`
    __device__ __forceinline__ half8 k_operand(int sub, int s) const {
        if constexpr (kF8) {
            const uint4v w = ka[sub][s / 2];
            return s % 2 ? f8x8_to_half8(w.z, w.w) : f8x8_to_half8(w.x, w.y);
        } else {
            return ex_half8(ka[sub][s]);
        }
    }
    // A operands t = 4 w .. 4 w + 3 (8-bit) or 2 w, 2 w + 1 (half) of contraction `pair`
    template <typename F>
    __device__ __forceinline__ void v_operands(int pair, int w, F&& use) const {
        const int j0 = 8 * pair;
        if constexpr (kF8) {
            // 4 x 4 byte transposes: tokens j0 .. j0 + 3 and j0 + 4 .. j0 + 7
            uint32_t b[2][4];
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const uint32_t a0 = vr[j0 + 4 * q][w], a1 = vr[j0 + 4 * q + 1][w], a2 = vr[j0 + 4 * q + 2][w],
                               a3 = vr[j0 + 4 * q + 3][w];
                const uint32_t l01 = __builtin_amdgcn_perm(a1, a0, 0x05010400u);  // a0.0 a1.0 a0.1 a1.1
                const uint32_t h01 = __builtin_amdgcn_perm(a1, a0, 0x07030602u);  // a0.2 a1.2 a0.3 a1.3
                const uint32_t l23 = __builtin_amdgcn_perm(a3, a2, 0x05010400u);
                const uint32_t h23 = __builtin_amdgcn_perm(a3, a2, 0x07030602u);
                b[q][0] = __builtin_amdgcn_perm(l23, l01, 0x05040100u);
                b[q][1] = __builtin_amdgcn_perm(l23, l01, 0x07060302u);
                b[q][2] = __builtin_amdgcn_perm(h23, h01, 0x05040100u);
                b[q][3] = __builtin_amdgcn_perm(h23, h01, 0x07060302u);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) use(4 * w + i, f8x8_to_half8(b[0][i], b[1][i]));
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t sel = i ? 0x07060302u : 0x05040100u;
                uint4v a;
                a.x = __builtin_amdgcn_perm(vr[j0 + 1][w], vr[j0][w], sel);
                a.y = __builtin_amdgcn_perm(vr[j0 + 3][w], vr[j0 + 2][w], sel);
                a.z = __builtin_amdgcn_perm(vr[j0 + 5][w], vr[j0 + 4][w], sel);
                a.w = __builtin_amdgcn_perm(vr[j0 + 7][w], vr[j0 + 6][w], sel);
                use(2 * w + i, ex_half8(a));
            }
        }
    }
};

// The maximum over the four lanes n, n + 16, n + 32, n + 48, in all of them: two register swaps, no LDS round trip
// (v_permlane16_swap exchanges the odd rows of 16 lanes of one register with the even rows of the other).
__device__ __forceinline__ float max_over_groups(float v) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    const LanePair both = half_wave_pair(fmaxf(a, b));
    return fmaxf(both.lo, both.hi);
}

// Float queries are taken times a power of two, the same for a whole row, that brings the row's largest element to
// 2^14 .. 2^15, and then as a half and a half remainder: an element is off by at most 2^-23 of itself or 2^-40 of the largest,
// whatever the row's magnitude (2^-97 and more).  The scores' factor takes the power back.  Infinities and NaN stay what they are.
// A lane loads the eight elements from d_of(s) on of step s; row_max: the maximum over the lanes that share the row; `sign` is
// 1, -1 or 0.  Returns what a product with the row is to be multiplied with.  (The row is held in registers from the maximum to
// the halves: read twice, 37 queries at 4096 took 30.4 us, so 28.9.)
template <int kSteps, typename DOf, typename RowMax>
__device__ __forceinline__ float ex_load_floats(const float* row, DOf&& d_of, RowMax&& row_max, float sign, bool live, half8* hi, half8* lo) {
    float x[kSteps][8], top = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
        const float4v x0 = *reinterpret_cast<const float4v*>(row + d_of(s)), x1 = *reinterpret_cast<const float4v*>(row + d_of(s) + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[s][i] = x0[i];
            x[s][4 + i] = x1[i];
        }
    }
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[s][i]));
    const int shift = max(-113, min(112, 15 - __builtin_amdgcn_frexp_expf(row_max(top))));
    const float power = ex_power(shift) * sign;
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float xs = live ? x[s][i] * power : 0.0f;  // (exact: one rounding either way, see ex_split)
            const _Float16 h = static_cast<_Float16>(xs);
            hi[s][i] = h;
            lo[s][i] = static_cast<_Float16>(xs - static_cast<float>(h));
        }
    return ex_power(-shift);
}
// A factor of scores as a finite number: a code of zero times it is zero.
__device__ __forceinline__ float ex_finite(float x) { return fminf(fmaxf(x, -FLT_MAX), FLT_MAX); }

// Query rows of a wave as B operands, and the running softmax state of those rows.
template <bool kQF32, bool kF8, int kD>
struct Rows16 {
    static constexpr int kSteps = kD / 32;
    half8 bq[kSteps];
    half8 bq_lo[kQF32 ? kSteps : 1];
    float unit;   // of a product with the row as loaded in the log2 domain, the K scale apart
    float m, l;   // running maximum (log2 domain) and this lane's part of the sum
    float bound;  // 8 bits: log2 of the largest p * 2^(exponent of the V scale), p relative to m; acc counts in units of
                  // 2^ceil(bound) / kExBoost: whole powers of two, which are taken off an exponent without a rounding
    float4v acc[8];

    __device__ __forceinline__ void clear() {
        m = kExNegBig;
        l = 0.0f;
        bound = kF8 ? kExNegBig : 0.0f;
#pragma unroll
        for (int t = 0; t < 8; t++) acc[t] = float4v{0, 0, 0, 0};
    }
    // src: element offset of the lane's row; dead rows are zeros
    __device__ __forceinline__ void load_q(const KvParams& p, int64_t at, bool live, uint32_t g) {
        if constexpr (kQF32) {
            unit = p.scale_log2 * ex_load_floats<kSteps>(
                                      static_cast<const float*>(p.q) + at, [g](int s) { return Tile<kF8, kExContiguous, kD>::d_of(s, g); },
                                      [](float v) { return max_over_groups(v); }, 1.0f, live, bq, bq_lo);
        } else {
            unit = p.scale_log2;
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                uint4v w = *reinterpret_cast<const uint4v*>(static_cast<const uint16_t*>(p.q) + at + Tile<kF8, kExContiguous, kD>::d_of(s, g));
                if (!live) w = uint4v{0, 0, 0, 0};
                bq[s] = ex_half8(w);
            }
        }
    }
};

// The output element d of a row whose sum came out as NaN although its probabilities did not: with infinities among the V it
// sees of a half cache the products of a probability's half and remainder may cancel (inf - inf) or vanish (inf * 0) where the
// sum is infinite.  It is the sum of the infinities and NaNs the row sees.  (Not for 8-bit pools, whose only special is NaN.)
__device__ __forceinline__ float settle_nan(const KvParams& p, float result, float l, uint32_t b, uint32_t kvh, uint32_t pos, uint32_t len, uint32_t d) {
    if (result == result || p.k_scale || !(l < INFINITY)) return result;
    const uint32_t lo = window_begin(pos, p.window), hi = p.causal ? min(len, pos + 1) : len;
    float sum = 0.0f;
    for (uint32_t key = 0; key < hi; key++) {
        if (key < lo && key >= p.sinks) {
            key = lo - 1;
            continue;
        }
        uint32_t row = key;
        if (p.tables) {
            const uint32_t blk = key / p.block_size;
            if (!pool_row(p.tables[size_t(b) * p.max_blocks + blk], key - blk * p.block_size, p.block_size, p.num_blocks, &row)) continue;
        }
        const float x = static_cast<float>(reinterpret_cast<const _Float16*>(p.v + int64_t(kvh) * p.head_bytes + int64_t(row) * p.row_bytes)[d]);
        if (!(fabsf(x) < INFINITY)) sum += x;
    }
    return sum != 0.0f ? sum : result;
}

// One tile's contribution to the rows of `st`.  `seen` is what all rows see between them, [lo, hi) and
// the first `sinks` tokens what the lane's own row sees.  `masked` (uniform): some row does not see some
// token of the tile.  kPerRow: the rows differ in what they see.
//
// V of a token that no row sees is zeroed, since 0 * NaN is NaN.  Where rows differ, a masked tile's V is
// taken with its infinities and NaNs replaced by zeros, and two products with the indicators of
// (+inf or NaN) and (-inf or NaN) in place of V and of visibility in place of P put them back into the
// rows that do see them.
template <bool kQF32, bool kF8, int kRows, int kD, bool kPerRow>
__device__ __forceinline__ void attend_tile(const KvParams& p, Tile<kF8, kRows, kD>& tile,
                                            const typename Tile<kF8, kRows, kD>::Rows& rows, uint32_t tok0,
                                            const VisibleTiles& seen, uint32_t lo, uint32_t hi, bool masked,
                                            Rows16<kQF32, kF8, kD>& st, uint32_t lane) {
    using T = Tile<kF8, kRows, kD>;
    constexpr int kSubs = T::kSubs;
    const uint32_t g = lane >> 4;
    // a value of the lane that holds token 16 sub + 4 g + i (Paged16: its run)
    auto of_token = [&](float x, int sub, int i) __attribute__((always_inline)) -> float {
        if constexpr (kRows == kExPaged16) return __uint_as_float(uint32_t(__builtin_amdgcn_readlane(int(__float_as_uint(x)), sub)));
        else return __uint_as_float(ex_lane_read(__float_as_uint(x), 16 * sub + 4 * g + i));
    };
    float s[kSubs][4];
#pragma unroll
    for (int sub = 0; sub < kSubs; sub++) {
        float4v c = {0, 0, 0, 0};
#pragma unroll
        for (int step = 0; step < T::kSteps; step++) {
            const half8 a = tile.k_operand(sub, step);
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, st.bq[step], c, 0, 0, 0);
            if constexpr (kQF32) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, st.bq_lo[step], c, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[sub][i] = c[i] * ex_finite(kF8 ? of_token(rows.ks, sub, i) * st.unit : st.unit);
    }
    bool special = false;  // kPerRow, masked: some V of the tile is infinite or NaN
    uint32_t visible = 0xFFFFu;  // bit 4 sub + i: the lane's row sees token 16 sub + 4 g + i
    if (masked) {
        if constexpr (kPerRow) visible = 0;
#pragma unroll
        for (int sub = 0; sub < kSubs; sub++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t in = 16 * sub + 4 * g + i, tok = tok0 + in;
                const uint32_t valid = kRows == kExContiguous ? 1u
                                       : kRows == kExPaged16  ? uint32_t(__builtin_amdgcn_readlane(int(rows.valid), sub))
                                                              : ex_lane_read(rows.valid, in);
                const bool vis = bool(int(valid) & int(tok < hi) & (int(tok >= lo) | int(tok < p.sinks)));
                if constexpr (kPerRow) visible |= vis ? 1u << (4 * sub + i) : 0u;
                s[sub][i] = vis ? s[sub][i] : -INFINITY;
                const bool any = kPerRow ? bool(int(valid) & int(tok < seen.end) & (int(tok >= seen.lo) | int(tok < p.sinks))) : vis;
                // (pinned here: moved behind the branch, the selects and the conditions they need would be paid for by
                // every tile)
                asm volatile("" : "+v"(s[sub][i]));
#pragma unroll
                for (int w = 0; w < T::kVWords; w++) {
                    tile.vr[4 * sub + i][w] = any ? tile.vr[4 * sub + i][w] : 0u;
                    asm volatile("" : "+v"(tile.vr[4 * sub + i][w]));
                }
            }
        if constexpr (kPerRow) {
            uint32_t hit = 0;
#pragma unroll
            for (int j = 0; j < 4 * kSubs; j++)
#pragma unroll
                for (int w = 0; w < T::kVWords; w++) {
                    // 8 bits: a byte's low seven bits are all ones; half: its exponent's five are.  Adding one in the lowest
                    // place of those carries into the bit above.
                    const uint32_t x = tile.vr[j][w];
                    hit |= kF8 ? ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u : ((x & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
                }
            special = __any(hit != 0);
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 4 * kSubs; i++) top = fmaxf(top, s[i / 4][i % 4]);
    top = max_over_groups(top);
    const float m_new = fmaxf(st.m, top), moved = st.m - m_new;
    float rescale = fast_exp2(moved), whole = 0.0f;  // of O, of l; ceil(bound)
    st.l *= rescale;
    if constexpr (kF8) {
        float z = -INFINITY;
#pragma unroll
        for (int sub = 0; sub < kSubs; sub++) {
            if constexpr (kRows == kExPaged16) {
                const float t = fmaxf(fmaxf(s[sub][0], s[sub][1]), fmaxf(s[sub][2], s[sub][3]));
                z = fmaxf(z, (t - m_new) + ex_exponent(of_token(rows.vs, sub, 0)));
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) z = fmaxf(z, (s[sub][i] - m_new) + ex_exponent(of_token(rows.vs, sub, i)));
            }
        }
        const float bound = fmaxf(st.bound + moved, max_over_groups(z));
        whole = ceilf(bound);
        rescale = fast_exp2(moved + (ceilf(st.bound) - whole));
        st.bound = bound;
    }
    if (__any(rescale != 1.0f)) {
#pragma unroll
        for (int t = 0; t < 8; t++) st.acc[t] *= rescale;
    }
    st.m = m_new;
    half8 hi8[T::kPairs], lo8[T::kPairs];
#pragma unroll
    for (int sub = 0; sub < kSubs; sub++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float d = s[sub][i] - m_new, e = fast_exp2(d);
            st.l += e;
            float scaled = e * kExBoost;
            if constexpr (kF8) {
                const float vs = of_token(rows.vs, sub, i);
                scaled = fast_exp2(d + (ex_exponent(vs) - whole)) * (ex_mantissa(vs) * kExBoost);
            }
            _Float16 half, rest;
            ex_split(scaled, half, rest);
            hi8[sub / 2][4 * (sub % 2) + i] = half;
            lo8[sub / 2][4 * (sub % 2) + i] = rest;
        }
#pragma unroll
    for (int pair = 0; pair < T::kPairs; pair++)
#pragma unroll
        for (int w = 0; w < T::kVWords; w++)
            tile.v_operands(pair, w, [&](int t, half8 a) __attribute__((always_inline)) {
                if (kPerRow && special) {
                    half8 plus, minus, sees;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint16_t bits = __builtin_bit_cast(uint16_t, _Float16(a[j]));
                        const bool special = (bits & 0x7C00u) == 0x7C00u, nan = special && (bits & 0x3FFu);
                        plus[j] = special && (nan || !(bits & 0x8000u)) ? _Float16(1) : _Float16(0);
                        minus[j] = special && (nan || (bits & 0x8000u)) ? _Float16(1) : _Float16(0);
                        if (special) a[j] = _Float16(0);
                        sees[j] = (visible >> (8 * pair + j)) & 1u ? _Float16(1) : _Float16(0);
                    }
                    const float4v zero = {0, 0, 0, 0};
                    const float4v up = __builtin_amdgcn_mfma_f32_16x16x32_f16(plus, sees, zero, 0, 0, 0);
                    const float4v down = __builtin_amdgcn_mfma_f32_16x16x32_f16(minus, sees, zero, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (up[i] > 0.0f) st.acc[t][i] += INFINITY;
                        if (down[i] > 0.0f) st.acc[t][i] -= INFINITY;
                    }
                }
                st.acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi8[pair], st.acc[t], 0, 0, 0);
                st.acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, lo8[pair], st.acc[t], 0, 0, 0);
            });
}

#endif  // __HIPCC__

}  // namespace ghip
