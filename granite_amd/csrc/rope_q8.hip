// Rotary position embedding of Q and K fused with the append of K and V to 8-bit paged pools (HBM bound).
//
// The half-precision form is rope.hip; the rotation is the same, with every product and sum rounded on its own
// (RoPECache::apply, src/llm/rope.cpp:24-92, bit for bit where its tables are given).  The pools hold e4m3 codes
// and a power-of-two scale for each (block, KV head) of K and of V:
//
//   top   = max |x| over the new, finite elements of the block and head
//   need  = 2^e, the smallest e in [-96, 120] with top <= 448 * 2^e   (448: the largest e4m3 value)
//   scale = need where the call writes row 0 of the block, else max(old scale, need)
//   code  = e4m3(x / scale), to nearest even; the rows in front become e4m3(code * old / scale) where it grew
//
// A code has three bits of mantissa wherever its scale puts it (above 2^-6), so a power of two loses nothing
// against top / 448, x / scale is exact, and growing a scale is exact as well for codes that stay above 2^-6.
//
// One launch of up to three kinds of workgroups:
//   * run of tokens of one sequence: one to sixteen waves per (block the run touches, KV head), by the block
//     size.  They take the block's new rows in turn and keep them in registers between the maximum and the
//     codes (8 rows of 128 or 16 of 64 elements a wave; what sixteen waves cannot hold is read twice),
//   * one token per sequence: a wave per (token, KV head), K in its lower half and V in its upper,
//   * Q: a thread per eight elements of a token's row in one or kQHeads heads, cos and sin loaded once for all.
//
// Measured (32 query heads over 8 KV heads of 128): 8187 tokens, half in and float Q out, 59.9 us a call for 256 MB, 4.3 TB/s,
// where a large copy reaches 4.9 (66 us with one head a thread and a wave a block); 64 tokens of 64 sequences, each the first of its
// block, 3.2 us of kernel in a call of 7.8 us: the launch; 512 tokens (64 heads) 8.5 us a call, 3.7 TB/s.  A scale that grows late
// in a block costs a step more: a wave walks the rows in front one after the other.  The kernel on its own, at the clocks of a few
// calls: 5.5 us for tokens that start a block or leave its scale, 7.9 where every scale grows at row 15 of 16, 32 at row 127 of 128.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "kv_visible.h"

namespace ghip {
namespace {

constexpr uint32_t kWaves = 4;      // of a workgroup, but for blocks of so many tokens that four waves do not hold them
constexpr uint32_t kMaxWaves = 16;
constexpr int kHold = 2;         // passes of a wave over new rows that stay in registers
constexpr uint32_t kQHeads = 2;  // heads per thread of the Q part of a large launch
constexpr float kF8Max = 448.0f;

struct RopeQ8Params {
    const void* q;
    void* q_out;
    const void* k;
    const void* v;
    uint8_t* k_cache;
    uint8_t* v_cache;
    float* k_scale;
    float* v_scale;
    const int32_t* table;
    const int32_t* positions;
    int64_t table_stride;
    const float* cos_t;
    const float* sin_t;
    uint32_t table_positions;
    float freq_base;
    uint32_t num_heads_q, num_heads_k, seq_len, start_pos;
    uint32_t block_size, num_blocks, max_blocks;
    uint32_t kv_groups;  // workgroups of the K/V part, in front of those of the Q part
    uint32_t q_heads;    // heads per thread of the Q part
    uint32_t kv_units, unit_waves;  // run form: (block, head) pairs, and how many of a workgroup's waves share one
    int q_out_f32;
};

struct Quad {
    float x[4];
};
struct Oct {
    Quad lo, hi;
};

template <bool kF16>
__device__ __forceinline__ Quad load_quad(const void* base, size_t at) {  // read once: streaming
    Quad r;
    if constexpr (kF16) {
        const half4 h = __builtin_nontemporal_load(reinterpret_cast<const half4*>(static_cast<const _Float16*>(base) + at));
#pragma unroll
        for (int i = 0; i < 4; i++) r.x[i] = static_cast<float>(h[i]);
    } else {
        const float4v f = __builtin_nontemporal_load(reinterpret_cast<const float4v*>(static_cast<const float*>(base) + at));
#pragma unroll
        for (int i = 0; i < 4; i++) r.x[i] = f[i];
    }
    return r;
}

template <bool kF16>
__device__ __forceinline__ void load_oct(const void* base, size_t at, Quad& lo, Quad& hi) {
    if constexpr (kF16) {
        const half8 h = __builtin_nontemporal_load(reinterpret_cast<const half8*>(static_cast<const _Float16*>(base) + at));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            lo.x[i] = static_cast<float>(h[i]);
            hi.x[i] = static_cast<float>(h[4 + i]);
        }
    } else {
        lo = load_quad<false>(base, at);
        hi = load_quad<false>(base, at + 4);
    }
}

struct Angles {
    float c0, s0, c1, s1;  // of pairs 2 j and 2 j + 1
};
__device__ __forceinline__ Angles angles_of(const RopeQ8Params& p, uint32_t pos, uint32_t j, uint32_t D) {
    Angles a;
    if (p.cos_t) {
        const size_t at = size_t(pos) * (D / 2) + 2 * j;
        const float2v c = *reinterpret_cast<const float2v*>(p.cos_t + at), s = *reinterpret_cast<const float2v*>(p.sin_t + at);
        a.c0 = c.x; a.c1 = c.y; a.s0 = s.x; a.s1 = s.y;
    } else {  // as rope.hip: freq = 1 / pow(base, 2 i / D)
        const float a0 = float(pos) * (1.0f / powf(p.freq_base, float(4 * j) / float(D)));
        const float a1 = float(pos) * (1.0f / powf(p.freq_base, float(4 * j + 2) / float(D)));
        a.c0 = cosf(a0); a.s0 = sinf(a0);
        a.c1 = cosf(a1); a.s1 = sinf(a1);
    }
    return a;
}
__device__ __forceinline__ Quad rotate(const Quad& q, const Angles& a) {
#pragma clang fp contract(off)
    Quad r;
    const float e0 = q.x[0] * a.c0, f0 = q.x[1] * a.s0, g0 = q.x[0] * a.s0, h0 = q.x[1] * a.c0;
    const float e1 = q.x[2] * a.c1, f1 = q.x[3] * a.s1, g1 = q.x[2] * a.s1, h1 = q.x[3] * a.c1;
    r.x[0] = e0 - f0;
    r.x[1] = g0 + h0;
    r.x[2] = e1 - f1;
    r.x[3] = g1 + h1;
    return r;
}

__device__ __forceinline__ float finite_top(const Quad& q, float top) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t mag = __float_as_uint(q.x[i]) & 0x7FFFFFFFu;
        top = fmaxf(top, mag < 0x7F800000u ? __uint_as_float(mag) : 0.0f);
    }
    return top;
}

// Smallest power of two s, 2^-96 <= s <= 2^120, with top <= 448 s.  448 = 1.75 * 2^8, so the exponent of
// `top` less 8, and one more where its mantissa is above 1.75.
__device__ __forceinline__ float scale_for(float top) {
    const uint32_t bits = __float_as_uint(top);
    int e = int(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    e = max(-96, min(120, e));  // (zero and the smallest magnitudes have exponent field 0: the floor)
    return __uint_as_float(uint32_t(e + 127) << 23);
}

__device__ __forceinline__ float to_f8_range(float x) {  // NaN stays NaN
    return x != x ? x : fminf(fmaxf(x, -kF8Max), kF8Max);
}
__device__ __forceinline__ uint32_t encode(const Quad& q, float inv) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(to_f8_range(q.x[0] * inv), to_f8_range(q.x[1] * inv), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(to_f8_range(q.x[2] * inv), to_f8_range(q.x[3] * inv), w, true);
    return uint32_t(w);
}
// The four codes of `w` times `ratio` (at most 1), rounded again.
__device__ __forceinline__ uint32_t recode(uint32_t w, float ratio) {
    const float2v lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    return encode(Quad{{lo.x, lo.y, hi.x, hi.y}}, ratio);
}

__device__ __forceinline__ float wave_max(float v, int from) {
    for (int off = from; off > 0; off >>= 1) v = fmaxf(v, wave_shfl_xor(v, off));
    return v;
}

template <bool kSrcF16, int kD>
__device__ void append_run(const RopeQ8Params& p) {
    constexpr uint32_t kOcts = kD / 8, kRowsPerPass = 64 / kOcts;
    __shared__ float s_top[kMaxWaves][2];
    const uint32_t n_waves = blockDim.x / 64;
    const uint32_t lane = threadIdx.x & 63, wave = uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
    const uint32_t part = wave % p.unit_waves;  // of the waves that share a unit
    const uint32_t unit = min(blockIdx.x * (n_waves / p.unit_waves) + wave / p.unit_waves, p.kv_units - 1);
    const bool spare = blockIdx.x * (n_waves / p.unit_waves) + wave / p.unit_waves >= p.kv_units;
    const uint32_t head = unit % p.num_heads_k, blk = p.start_pos / p.block_size + unit / p.num_heads_k;
    const uint32_t end = p.start_pos + p.seq_len;
    const uint32_t lo = max(p.start_pos, blk * p.block_size), hi = min(end, (blk + 1) * p.block_size);  // positions
    const int32_t entry = p.table[blk];
    const uint32_t j = lane % kOcts, sub = lane / kOcts;
    const uint32_t n_rows = hi - lo;

    auto fetch = [&](uint32_t i, Oct& k, Oct& v) {  // new row i of the block
        const uint32_t s = lo + i - p.start_pos;
        const size_t at = (size_t(s) * p.num_heads_k + head) * kD + 8 * j;
        load_oct<kSrcF16>(p.k, at, k.lo, k.hi);
        load_oct<kSrcF16>(p.v, at, v.lo, v.hi);
    };
    auto turn = [&](uint32_t i, Oct& k) {
        k.lo = rotate(k.lo, angles_of(p, lo + i, 2 * j, kD));
        k.hi = rotate(k.hi, angles_of(p, lo + i, 2 * j + 1, kD));
    };
    Oct kq[kHold], vq[kHold];
    float k_top = 0.0f, v_top = 0.0f;
    const uint32_t stride = p.unit_waves * kRowsPerPass, first = part * kRowsPerPass + sub;
#pragma unroll
    for (int h = 0; h < kHold; h++)
        if (h * stride + first < n_rows) fetch(h * stride + first, kq[h], vq[h]);
    const size_t scale_at = size_t(uint32_t(entry) < p.num_blocks ? uint32_t(entry) : 0u) * p.num_heads_k + head;
    const uint32_t kept = lo - blk * p.block_size;  // rows in front of the new ones
    const float k_old = kept ? p.k_scale[scale_at] : 0.0f, v_old = kept ? p.v_scale[scale_at] : 0.0f;
#pragma unroll
    for (int h = 0; h < kHold; h++) {
        if (h * stride + first < n_rows) {
            turn(h * stride + first, kq[h]);
            k_top = finite_top(kq[h].hi, finite_top(kq[h].lo, k_top));
            v_top = finite_top(vq[h].hi, finite_top(vq[h].lo, v_top));
        }
    }
    for (uint32_t i = kHold * stride + first; i < n_rows; i += stride) {
        Oct k, v;
        fetch(i, k, v);
        turn(i, k);
        k_top = finite_top(k.hi, finite_top(k.lo, k_top));
        v_top = finite_top(v.hi, finite_top(v.lo, v_top));
    }
    k_top = wave_max(k_top, 32);
    v_top = wave_max(v_top, 32);
    if (p.unit_waves > 1) {  // uniform over the launch
        if (lane == 0) {
            s_top[wave][0] = k_top;
            s_top[wave][1] = v_top;
        }
        __syncthreads();
        for (uint32_t w = wave - part; w < wave - part + p.unit_waves; w++) {
            k_top = fmaxf(k_top, s_top[w][0]);
            v_top = fmaxf(v_top, s_top[w][1]);
        }
    }
    uint32_t row0;  // pool row of position lo; the block's first row is row0 - kept
    if (!pool_row(entry, kept, p.block_size, p.num_blocks, &row0) || spare) return;
    const float k_new = fmaxf(k_old, scale_for(k_top)), v_new = fmaxf(v_old, scale_for(v_top));
    const float k_inv = 1.0f / k_new, v_inv = 1.0f / v_new;
    auto store = [&](uint32_t i, const Oct& k, const Oct& v) {
        const size_t at = (size_t(row0 + i) * p.num_heads_k + head) * kD + 8 * j;
        *reinterpret_cast<uint2v*>(p.k_cache + at) = uint2v{encode(k.lo, k_inv), encode(k.hi, k_inv)};
        *reinterpret_cast<uint2v*>(p.v_cache + at) = uint2v{encode(v.lo, v_inv), encode(v.hi, v_inv)};
    };
#pragma unroll
    for (int h = 0; h < kHold; h++)
        if (h * stride + first < n_rows) store(h * stride + first, kq[h], vq[h]);
    for (uint32_t i = kHold * stride + first; i < n_rows; i += stride) {
        Oct k, v;
        fetch(i, k, v);
        turn(i, k);
        store(i, k, v);
    }
    if (k_new > k_old || v_new > v_old) {
        for (uint32_t i = first; i < kept; i += stride) {
            const size_t at = (size_t(row0 - kept + i) * p.num_heads_k + head) * kD + 8 * j;
            if (k_new > k_old) {
                uint2v* w = reinterpret_cast<uint2v*>(p.k_cache + at);
                *w = uint2v{recode(w->x, k_old * k_inv), recode(w->y, k_old * k_inv)};
            }
            if (v_new > v_old) {
                uint2v* w = reinterpret_cast<uint2v*>(p.v_cache + at);
                *w = uint2v{recode(w->x, v_old * v_inv), recode(w->y, v_old * v_inv)};
            }
        }
        if (part == 0 && lane == 0) {
            p.k_scale[scale_at] = k_new;
            p.v_scale[scale_at] = v_new;
        }
    }
}

// Position of token s; false where it is negative or beyond the tables.
__device__ __forceinline__ bool position_of(const RopeQ8Params& p, uint32_t s, uint32_t* pos) {
    if (!p.positions) {
        *pos = p.start_pos + s;
        return true;
    }
    const int32_t given = p.positions[s];
    *pos = given < 0 ? 0u : uint32_t(given);
    return given >= 0 && !(p.cos_t && *pos >= p.table_positions);
}

template <bool kSrcF16, int kD>
__device__ void append_step(const RopeQ8Params& p) {
    constexpr uint32_t kQuads = kD / 4;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * kWaves + uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
    if (unit >= p.seq_len * p.num_heads_k) return;
    const uint32_t s = unit / p.num_heads_k, head = unit % p.num_heads_k;
    uint32_t pos;
    if (!position_of(p, s, &pos)) return;
    const uint32_t blk = pos / p.block_size, kept = pos - blk * p.block_size;
    if (blk >= p.max_blocks) return;
    const int32_t entry = p.table[int64_t(s) * p.table_stride + blk];
    uint32_t row;
    if (!pool_row(entry, kept, p.block_size, p.num_blocks, &row)) return;
    // the lower half of the wave has K, the upper V
    const bool is_v = lane >= 32;
    const uint32_t j = lane & 31;
    const bool live = j < kQuads;
    const size_t at = (size_t(s) * p.num_heads_k + head) * kD + 4 * min(j, kQuads - 1);
    const Angles ang = angles_of(p, pos, min(j, kQuads - 1), kD);
    float* scales = is_v ? p.v_scale : p.k_scale;
    const size_t scale_at = size_t(uint32_t(entry)) * p.num_heads_k + head;
    const float old_scale = kept ? scales[scale_at] : 0.0f;
    Quad x = load_quad<kSrcF16>(is_v ? p.v : p.k, at);
    if (!is_v) x = rotate(x, ang);
    const float top = wave_max(finite_top(x, 0.0f), 16);  // of the lane's half of the wave
    const float scale = fmaxf(old_scale, scale_for(top)), inv = 1.0f / scale;
    uint8_t* cache = is_v ? p.v_cache : p.k_cache;
    if (live)
        *reinterpret_cast<uint32_t*>(cache + (size_t(row) * p.num_heads_k + head) * kD + 4 * j) = encode(x, inv);
    if (scale > old_scale) {
        if (live) {
            for (uint32_t i = 0; i < kept; i++) {
                uint32_t* w = reinterpret_cast<uint32_t*>(cache + (size_t(row - kept + i) * p.num_heads_k + head) * kD + 4 * j);
                *w = recode(*w, old_scale * inv);
            }
        }
        if (j == 0) scales[scale_at] = scale;
    }
}

// A thread has eight consecutive elements of a row, 16 bytes of halves, in q_heads heads; the loads of all of them and
// of their angles are in flight together.
template <bool kSrcF16, int kD>
__device__ void rotate_q(const RopeQ8Params& p) {
    constexpr uint32_t kOcts = kD / 8;
    const uint32_t runs = (p.num_heads_q + p.q_heads - 1) / p.q_heads;
    const uint64_t idx = uint64_t(blockIdx.x - p.kv_groups) * blockDim.x + threadIdx.x;
    const uint32_t j = uint32_t(idx % kOcts);
    const uint64_t rest = idx / kOcts;
    if (rest >= uint64_t(runs) * p.seq_len) return;
    const uint32_t s = uint32_t(rest / runs), run = uint32_t(rest - uint64_t(s) * runs);
    uint32_t pos;
    if (!position_of(p, s, &pos)) return;
    const uint32_t h0 = run * p.q_heads;
    const size_t at0 = (size_t(s) * p.num_heads_q + h0) * kD + 8 * j;
    Quad lo[kQHeads], hi[kQHeads];
#pragma unroll
    for (uint32_t i = 0; i < kQHeads; i++) {
        if (i < p.q_heads && h0 + i < p.num_heads_q) load_oct<kSrcF16>(p.q, at0 + i * kD, lo[i], hi[i]);
    }
    const Angles a0 = angles_of(p, pos, 2 * j, kD), a1 = angles_of(p, pos, 2 * j + 1, kD);
#pragma unroll
    for (uint32_t i = 0; i < kQHeads; i++) {
        if (i >= p.q_heads || h0 + i >= p.num_heads_q) continue;
        const Quad r0 = rotate(lo[i], a0), r1 = rotate(hi[i], a1);
        const size_t at = at0 + i * kD;
        if (p.q_out_f32) {
            float4v* out = reinterpret_cast<float4v*>(static_cast<float*>(p.q_out) + at);
            out[0] = float4v{r0.x[0], r0.x[1], r0.x[2], r0.x[3]};
            out[1] = float4v{r1.x[0], r1.x[1], r1.x[2], r1.x[3]};
        } else {
            *reinterpret_cast<uint4v*>(static_cast<uint16_t*>(p.q_out) + at) =
                uint4v{pack_f16x2(r0.x[0], r0.x[1]), pack_f16x2(r0.x[2], r0.x[3]), pack_f16x2(r1.x[0], r1.x[1]), pack_f16x2(r1.x[2], r1.x[3])};
        }
    }
}

template <bool kSrcF16, int kD>
__global__ void __launch_bounds__(kMaxWaves* kWave) rope_q8_kernel(RopeQ8Params p) {
    if (blockIdx.x >= p.kv_groups) rotate_q<kSrcF16, kD>(p);
    else if (p.positions) append_step<kSrcF16, kD>(p);
    else append_run<kSrcF16, kD>(p);
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

}  // namespace

int launch_rope_append_q8(const granite_hip_rope_q8_args& a) {
    if (!a.q && !a.k) return GRANITE_HIP_ENULL;
    if ((a.q == nullptr) != (a.q_out == nullptr) || (a.k == nullptr) != (a.v == nullptr)) return GRANITE_HIP_ENULL;
    if (a.head_dim != 128 && a.head_dim != 64) return GRANITE_HIP_EUNSUPPORTED;
    if (a.src_dtype != GRANITE_HIP_F32 && a.src_dtype != GRANITE_HIP_F16) return GRANITE_HIP_EINVAL;
    if (a.q && a.q_out_dtype != GRANITE_HIP_F32 && a.q_out_dtype != GRANITE_HIP_F16) return GRANITE_HIP_EINVAL;
    if ((a.q && a.num_heads_q == 0) || (a.k && a.num_heads_k == 0)) return GRANITE_HIP_EINVAL;
    if (a.q && a.q_out == a.q && a.src_dtype != a.q_out_dtype) return GRANITE_HIP_EINVAL;
    if ((a.cos_table == nullptr) != (a.sin_table == nullptr)) return GRANITE_HIP_ENULL;
    if (!a.cos_table && !(a.freq_base > 0.0f)) return GRANITE_HIP_EINVAL;
    const uint64_t end = uint64_t(a.start_pos) + a.seq_len;
    if (end >= (1ull << 31)) return GRANITE_HIP_EINVAL;
    if (a.cos_table && !a.positions && end > a.table_positions) return GRANITE_HIP_EOVERFLOW;
    if (a.k) {
        if (!a.k_cache || !a.v_cache || !a.k_scale || !a.v_scale || !a.block_table) return GRANITE_HIP_ENULL;
        if (a.block_size == 0 || a.num_blocks == 0 || a.max_blocks_per_seq == 0) return GRANITE_HIP_EINVAL;
        if (uint64_t(a.num_blocks) * a.block_size >= (1ull << 31)) return GRANITE_HIP_EINVAL;
        if (a.positions) {
            // sequences that shared a table would append to the same block at once
            if (a.seq_len > 1 && a.table_stride < int64_t(a.max_blocks_per_seq)) return GRANITE_HIP_EINVAL;
        } else if ((end + a.block_size - 1) / a.block_size > a.max_blocks_per_seq) {
            return GRANITE_HIP_EOVERFLOW;
        }
        if (!aligned(a.k_cache, 16) || !aligned(a.v_cache, 16) || !aligned(a.k, 16) || !aligned(a.v, 16)) return GRANITE_HIP_EINVAL;
    }
    if ((a.q && (!aligned(a.q, 16) || !aligned(a.q_out, 16))) ||
        (a.cos_table && (!aligned(a.cos_table, 8) || !aligned(a.sin_table, 8))))
        return GRANITE_HIP_EINVAL;
    if (!ctx().initialized) return GRANITE_HIP_ENOTINIT;
    if (a.seq_len == 0) return GRANITE_HIP_OK;

    RopeQ8Params p{};
    p.q = a.q;
    p.q_out = a.q_out;
    p.k = a.k;
    p.v = a.v;
    p.k_cache = static_cast<uint8_t*>(a.k_cache);
    p.v_cache = static_cast<uint8_t*>(a.v_cache);
    p.k_scale = a.k_scale;
    p.v_scale = a.v_scale;
    p.table = a.block_table;
    p.positions = a.positions;
    p.table_stride = a.table_stride;
    p.cos_t = a.cos_table;
    p.sin_t = a.sin_table;
    p.table_positions = a.table_positions;
    p.freq_base = a.freq_base;
    p.num_heads_q = a.num_heads_q;
    p.num_heads_k = a.num_heads_k;
    p.seq_len = a.seq_len;
    p.start_pos = a.positions ? 0 : a.start_pos;
    p.block_size = a.block_size;
    p.num_blocks = a.num_blocks;
    p.max_blocks = a.max_blocks_per_seq;
    p.q_out_f32 = a.q_out_dtype == GRANITE_HIP_F32;

    uint64_t kv_groups = 0, q_groups = 0;
    uint32_t n_waves = kWaves;
    if (a.k) {
        const uint64_t units = a.positions ? uint64_t(a.seq_len)
                                           : uint64_t((end - 1) / a.block_size) - a.start_pos / a.block_size + 1;
        if (units * a.num_heads_k > 0x7FFFFFFFull) return GRANITE_HIP_EINVAL;
        p.kv_units = uint32_t(units * a.num_heads_k);
        const uint32_t held = kHold * (512 / a.head_dim);  // rows a wave holds
        p.unit_waves = 1;
        // as many waves as hold the block's rows, more than four only at head size 128 and while a launch has no more than 4096 of
        // them: blocks of 128 tokens, 64 units 23.9 us with four waves, 18 with eight, 13.6 with sixteen; 784 units 40, 43 and
        // 50; at head size 64 16.2 us with four, 18.4 with eight (176 units)
        const uint32_t most = a.positions || a.head_dim == 64 ? kWaves : kMaxWaves;
        while (p.unit_waves < most && p.unit_waves * held < a.block_size && (p.unit_waves < kWaves || 2ull * p.unit_waves * p.kv_units <= 4096))
            p.unit_waves *= 2;
        if (!a.positions) n_waves = std::max(kWaves, p.unit_waves);
        const uint32_t per_group = a.positions ? kWaves : n_waves / p.unit_waves;
        kv_groups = (units * a.num_heads_k + per_group - 1) / per_group;
    }
    if (a.q) {
        const uint64_t octs = uint64_t(a.seq_len) * (a.head_dim / 8) * a.num_heads_q;
        // one head per thread until there are four times as many threads as the part holds at once
        // (256 CUs x 2048): the lookup of cos and sin is then shared by two heads (8187 tokens: 62.5 us; by four 65)
        p.q_heads = octs >= (2ull << 20) ? kQHeads : 1;
        const uint64_t threads = uint64_t(a.seq_len) * (a.head_dim / 8) * ((a.num_heads_q + p.q_heads - 1) / p.q_heads);
        q_groups = (threads + 64 * n_waves - 1) / (64 * n_waves);
    }
    if (kv_groups + q_groups > 0x7FFFFFFFull) return GRANITE_HIP_EINVAL;
    p.kv_groups = uint32_t(kv_groups);
    const dim3 grid(uint32_t(kv_groups + q_groups)), block(64 * n_waves);
    hipStream_t st = ctx().stream;
    {
        KernelTimerScope timer("rope_append_q8");
        if (a.src_dtype == GRANITE_HIP_F16 && a.head_dim == 128) rope_q8_kernel<true, 128><<<grid, block, 0, st>>>(p);
        else if (a.src_dtype == GRANITE_HIP_F16) rope_q8_kernel<true, 64><<<grid, block, 0, st>>>(p);
        else if (a.head_dim == 128) rope_q8_kernel<false, 128><<<grid, block, 0, st>>>(p);
        else rope_q8_kernel<false, 64><<<grid, block, 0, st>>>(p);
    }
    return launch_status();
}

}  // namespace ghip
