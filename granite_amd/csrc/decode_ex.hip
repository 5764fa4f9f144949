// Attention over 8-bit paged pools and through a sliding window with sinks: the row kernel, its merge, and
// the entry points' argument checks and choice of kernel.
//
// The row kernel takes 16 rows of a KV head a workgroup; its eight waves take the visible tiles (64 tokens of 8 bits, 32 of half) in
// turn, straight from memory as MFMA operands, and are joined through LDS, so a call is one launch unless its keys are
// cut.  One sequence of 512 tokens of float queries 8.2 us a call (a wave has one tile; eight workgroups behind the
// chain of length, table entry, scale and row), 64 sequences of 256 to 8192 over blocks of 20 tokens 170 us, 3.3 TB/s.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "kv_attend.h"

namespace ghip {
namespace {

constexpr uint32_t kRowWaves = 8;
constexpr uint32_t kStreamRows = 1280;  // most rows of a KV head that the persistent kernel takes

// One workgroup per (run of 16 query rows, KV head, sequence, key split).  A row is a (query, head of
// the KV head's group) pair, row r = query * group + head, so a decode step's group, a few draft tokens and a
// long chunk are the same thing here.  The waves take the visible tiles in turn and are merged through LDS.
// kMulti: several queries, whose rows differ in what they see.
template <bool kQF32, bool kF8, int kRows, int kD, bool kMulti>
__global__ void __launch_bounds__(kRowWaves* kWave, 2) kv_rows_kernel(KvParams p) {
    using T = Tile<kF8, kRows, kD>;
    const uint32_t lane = threadIdx.x & 63, wave = ex_uniform(threadIdx.x >> 6);
    const uint32_t n = lane & 15, g = lane >> 4;
    const uint32_t split = blockIdx.x % p.n_splits, rt = blockIdx.x / p.n_splits;
    const uint32_t kvh = blockIdx.y, b = blockIdx.z;
    const uint32_t len = p.decode ? ex_uniform(ex_seq_len(p, b)) : p.max_tokens;
    if (p.decode && len == 0) return;  // an empty sequence: its output rows stay as they are

    const uint32_t n_rows = p.seq_q * p.group;
    const uint32_t r = min(rt * 16 + n, n_rows - 1);
    const bool live = rt * 16 + n < n_rows;
    const uint32_t qt = r / p.group, head = kvh * p.group + r % p.group;
    const uint32_t start = p.decode ? len - 1 : p.start_pos;
    const uint32_t first_pos = start + rt * 16 / p.group;
    const uint32_t last_pos = start + (min(rt * 16 + 16, n_rows) - 1) / p.group;
    const VisibleTiles seen = visible_tiles<T::kTokens>(first_pos, p.causal ? min(len, last_pos + 1) : len, p.window, p.sinks);
    const uint32_t hi = p.causal ? min(len, start + qt + 1) : len;
    const uint32_t lo = window_begin(start + qt, p.window);
    // what every row sees: up to the first row's position, from the last row's window on
    const uint32_t hi_all = p.causal ? min(len, first_pos + 1) : len, lo_all = window_begin(last_pos, p.window);

    Rows16<kQF32, kF8, kD> st;
    st.clear();
    st.load_q(p, int64_t(b) * p.q_batch + int64_t(qt) * p.q_tok + int64_t(head) * p.q_head, live, g);
    const int32_t* table = kRows != kExContiguous ? p.tables + size_t(b) * p.max_blocks : nullptr;

    const uint32_t i_begin = uint32_t(uint64_t(seen.count) * split / p.n_splits);
    const uint32_t i_end = uint32_t(uint64_t(seen.count) * (split + 1) / p.n_splits);
    for (uint32_t i = i_begin + wave; i < i_end; i += kRowWaves) {
        const uint32_t tok0 = seen.tile(i) * T::kTokens;
        T tile;
        const auto rows = T::rows_from(p, T::entry_of(p, table, tok0, seen, lane), kvh, tok0, seen, lane);
        tile.load(p, rows, kvh, lane);
        const bool masked = T::needs_mask(p, rows, tok0, lo_all, hi_all);
        attend_tile<kQF32, kF8, kRows, kD, kMulti>(p, tile, rows, tok0, seen, lo, hi, masked, st, lane);
    }

    // ---- the waves' results, combined through LDS
    __shared__ float s_ml[kRowWaves][16][2];
    extern __shared__ float s_o_raw[];  // [kRowWaves][16][kD + 4]
    auto s_o = [&](uint32_t w, uint32_t row, uint32_t d) __attribute__((always_inline)) -> float& { return s_o_raw[(w * 16 + row) * (kD + 4) + d]; };
    {
        float l = st.l;
        l += wave_shfl_xor(l, 16);
        l += wave_shfl_xor(l, 32);
        if (g == 0) {
            s_ml[wave][n][0] = st.m;
            s_ml[wave][n][1] = l;
        }
        const float unit = ex_unit(st.bound);
        if (32 * g < uint32_t(kD)) {
#pragma unroll
            for (int e = 0; e < 32; e++) s_o(wave, n, 32 * g + e) = st.acc[e & 7][e >> 3] * unit;
        }
    }
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < 16 * kD; x += blockDim.x) {
        const uint32_t row = x / kD, d = x % kD;
        if (rt * 16 + row >= n_rows) continue;
        float m = kExNegBig;
#pragma unroll
        for (uint32_t w = 0; w < kRowWaves; w++) m = fmaxf(m, s_ml[w][row][0]);
        float l = 0.0f, o = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kRowWaves; w++) {
            const float f = fast_exp2(s_ml[w][row][0] - m);
            l += s_ml[w][row][1] * f;
            o += s_o(w, row, d) * f;
        }
        const uint32_t q = (rt * 16 + row) / p.group, h = kvh * p.group + (rt * 16 + row) % p.group;
        if (p.n_splits > 1) {
            const size_t at = ((size_t(split) * p.batch + b) * p.num_heads + h) * p.seq_q + q;
            p.part_o[at * kD + d] = o;
            if (d == 0) {
                p.part_ml[at * 2] = m;
                p.part_ml[at * 2 + 1] = l;
            }
            continue;
        }
        const float result = settle_nan(p, l == 0.0f ? 0.0f : o / l, l, b, kvh, start + q, len, d);
        const int64_t at = int64_t(b) * p.out_batch + int64_t(q) * p.out_tok + int64_t(h) * p.out_head + d;
        if (p.out_f32) static_cast<float*>(p.out)[at] = result;
        else static_cast<_Float16*>(p.out)[at] = static_cast<_Float16>(result);
        if (p.lse && d == 0)
            p.lse[int64_t(b) * p.lse_batch + int64_t(q) * p.lse_tok + int64_t(h) * p.lse_head] =
                l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kExLn2;
    }
}

// Combines the key splits of one query row of one head: a thread per head-dim element.
__global__ void kv_rows_merge_kernel(KvParams p, uint32_t D) {
    const uint32_t h = blockIdx.x, q = blockIdx.y, b = blockIdx.z, d = threadIdx.x;
    if (p.decode && ex_seq_len(p, b) == 0) return;
    const size_t row = (size_t(b) * p.num_heads + h) * p.seq_q + q, step = size_t(p.batch) * p.num_heads * p.seq_q;
    float m = kExNegBig;
    for (uint32_t s = 0; s < p.n_splits; s++) m = fmaxf(m, p.part_ml[(row + s * step) * 2]);
    float l = 0.0f, o = 0.0f;
    for (uint32_t s = 0; s < p.n_splits; s++) {
        const float f = fast_exp2(p.part_ml[(row + s * step) * 2] - m);
        l += p.part_ml[(row + s * step) * 2 + 1] * f;
        o += p.part_o[(row + s * step) * D + d] * f;
    }
    const uint32_t len = p.decode ? ex_seq_len(p, b) : p.max_tokens;
    const float result = settle_nan(p, l == 0.0f ? 0.0f : o / l, l, b, h / p.group, p.decode ? len - 1 : p.start_pos + q, len, d);
    const int64_t at = int64_t(b) * p.out_batch + int64_t(q) * p.out_tok + int64_t(h) * p.out_head + d;
    if (p.out_f32) static_cast<float*>(p.out)[at] = result;
    else static_cast<_Float16*>(p.out)[at] = static_cast<_Float16>(result);
    if (p.lse && d == 0)
        p.lse[int64_t(b) * p.lse_batch + int64_t(q) * p.lse_tok + int64_t(h) * p.lse_head] =
            l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kExLn2;
}

template <bool kQF32, bool kF8, int kRows, int kD, bool kMulti>
int launch_rows_one(const KvParams& p, dim3 grid) {
    auto kernel = kv_rows_kernel<kQF32, kF8, kRows, kD, kMulti>;
    constexpr size_t kLds = size_t(kRowWaves) * 16 * (kD + 4) * sizeof(float);
    static bool configured[kMaxDevices];
    if (int rc = raise_dynamic_lds_limit(reinterpret_cast<const void*>(kernel), kLds, configured)) return rc;
    kernel<<<grid, dim3(kRowWaves * kWave), kLds, ctx().stream>>>(p);
    return launch_status();
}
template <bool kQF32, bool kF8, int kRows>
int launch_rows_dim(const KvParams& p, dim3 grid, uint32_t D) {
    if (p.decode)
        return D == 128 ? launch_rows_one<kQF32, kF8, kRows, 128, false>(p, grid) : launch_rows_one<kQF32, kF8, kRows, 64, false>(p, grid);
    return D == 128 ? launch_rows_one<kQF32, kF8, kRows, 128, true>(p, grid) : launch_rows_one<kQF32, kF8, kRows, 64, true>(p, grid);
}

template <bool kQF32>
int launch_rows_cache(const KvParams& p, dim3 grid, uint32_t D, bool f8, int rows) {
    if (f8 && rows == kExPaged16) return launch_rows_dim<kQF32, true, kExPaged16>(p, grid, D);
    if (f8) return launch_rows_dim<kQF32, true, kExPagedAny>(p, grid, D);
    if (rows == kExContiguous) return launch_rows_dim<kQF32, false, kExContiguous>(p, grid, D);
    if (rows == kExPaged16) return launch_rows_dim<kQF32, false, kExPaged16>(p, grid, D);
    return launch_rows_dim<kQF32, false, kExPagedAny>(p, grid, D);
}

KvCall call_of(const KvParams& p, uint32_t D, bool q_f32, bool f8, int rows) {
    KvCall c{};
    c.rows = uint64_t(p.seq_q) * p.group;
    c.lists = p.num_kv_heads * p.batch;
    c.queries = p.seq_q;
    c.group = p.group;
    c.head_dim = D;
    c.start_pos = p.start_pos;
    c.length = p.causal && !p.decode ? uint32_t(std::min(uint64_t(p.max_tokens), uint64_t(p.start_pos) + p.seq_q)) : p.max_tokens;
    c.window_keys = p.window ? uint64_t(p.window) + p.sinks : 0;
    c.causal = p.causal && !p.decode;
    c.f8 = f8;
    c.paged_runs = rows != kExPagedAny;
    c.wide = q_f32 || p.out_f32;
    c.cus = ctx().compute_units > 0 ? uint32_t(ctx().compute_units) : 256u;
    return c;
}

// The row kernel for any launch.
int launch_rows(KvParams p, uint32_t D, bool q_f32, bool f8, int rows, const ScratchSource& scratch) {
    const uint32_t row_tiles = uint32_t((uint64_t(p.seq_q) * p.group + 15) / 16);
    if (p.num_kv_heads > 65535u || p.batch > 65535u) return GRANITE_HIP_EINVAL;
    p.n_splits = p.seq_q > 65535u ? 1u : kv_rows_cut(call_of(p, D, q_f32, f8, rows)).pieces;  // (the merge's grid has a row per query)
    if (uint64_t(row_tiles) * p.n_splits > 0x7FFFFFFFull) return GRANITE_HIP_EINVAL;
    const size_t slots = p.n_splits > 1 ? size_t(p.n_splits) * p.batch * p.num_heads * p.seq_q : 0;
    const size_t need = slots * (D + 2) * sizeof(float);
    if (scratch.query) {
        *scratch.query = need;
        return GRANITE_HIP_OK;
    }
    if (need > 0) {
        void* ws = nullptr;
        const int rc = take_scratch(scratch, need, &ws);
        if (rc != GRANITE_HIP_OK) return rc;
        p.part_o = static_cast<float*>(ws);
        p.part_ml = p.part_o + slots * D;
    }
    int rc;
    {
        KernelTimerScope timer(p.decode ? "decode_ex" : "attention_ex");
        const dim3 grid(row_tiles * p.n_splits, p.num_kv_heads, p.batch);
        rc = q_f32 ? launch_rows_cache<true>(p, grid, D, f8, rows) : launch_rows_cache<false>(p, grid, D, f8, rows);
    }
    if (rc != GRANITE_HIP_OK || p.n_splits == 1) return rc;
    {
        KernelTimerScope timer(p.decode ? "decode_ex_merge" : "attention_ex_merge");
        kv_rows_merge_kernel<<<dim3(p.num_heads, p.seq_q, p.batch), dim3(D), 0, ctx().stream>>>(p, D);
    }
    return launch_status();
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What both forms have in common: the cache.
int check_form(const granite_hip_kv_form& f, const void* k, const void* v, const void* table, uint32_t block_size,
               uint32_t num_kv_heads, uint32_t D, KvParams& p, int& rows) {
    if (f.kv_dtype != GRANITE_HIP_F16 && f.kv_dtype != GRANITE_HIP_F8E4M3) return GRANITE_HIP_EINVAL;
    const bool f8 = f.kv_dtype == GRANITE_HIP_F8E4M3;
    if (f8 && !table) return GRANITE_HIP_EUNSUPPORTED;
    if (f8 && (!f.k_scale || !f.v_scale)) return GRANITE_HIP_ENULL;
    if (!aligned16(k) || !aligned16(v)) return GRANITE_HIP_EINVAL;
    if (table) {
        if (block_size == 0 || f.num_blocks == 0) return GRANITE_HIP_EINVAL;
        if (uint64_t(f.num_blocks) * block_size >= (1ull << 31)) return GRANITE_HIP_EINVAL;
        p.row_bytes = int64_t(num_kv_heads) * D * (f8 ? 1 : 2);
        p.head_bytes = int64_t(D) * (f8 ? 1 : 2);
        // (a lane's offset inside a run of 16 rows is a 32-bit product)
        rows = block_size % 16 == 0 && p.row_bytes < (1 << 27) ? kExPaged16 : kExPagedAny;
    } else {
        rows = kExContiguous;
    }
    p.k = static_cast<const uint8_t*>(k);
    p.v = static_cast<const uint8_t*>(v);
    p.k_scale = f8 ? f.k_scale : nullptr;  // (what the pointers of a half cache hold means nothing)
    p.v_scale = f8 ? f.v_scale : nullptr;
    p.num_blocks = f.num_blocks;
    p.block_size = table ? block_size : 1;
    p.bs_shift = (p.block_size & (p.block_size - 1)) == 0 ? __builtin_ctz(p.block_size) : -1;
    p.window = f.window;
    p.sinks = f.window ? std::min(f.num_sinks, 0x7FFFFFFFu) : 0;  // (std: the unqualified min of host code is one of ints)
    return GRANITE_HIP_OK;
}

bool plain_form(const granite_hip_kv_form& f) { return f.kv_dtype == GRANITE_HIP_F16 && f.window == 0; }

}  // namespace

int launch_decode_ex(const granite_hip_decode_args& a, const granite_hip_kv_form& f, const ScratchSource& scratch) {
    if (!a.q || !a.k_cache || !a.v_cache || !a.out) return GRANITE_HIP_ENULL;
    if (a.head_dim != 128 && a.head_dim != 64) return GRANITE_HIP_EUNSUPPORTED;
    if (a.num_heads == 0 || a.num_kv_heads == 0 || a.num_heads % a.num_kv_heads != 0) return GRANITE_HIP_EINVAL;
    if (a.q_dtype != GRANITE_HIP_F32 && a.q_dtype != GRANITE_HIP_F16) return GRANITE_HIP_EINVAL;
    if (!aligned16(a.q) || !aligned16(a.out)) return GRANITE_HIP_EINVAL;
    const uint32_t D = a.head_dim;
    KvParams p{};
    int rows = 0;
    if (int rc = check_form(f, a.k_cache, a.v_cache, a.block_tables, a.block_size, a.num_kv_heads, D, p, rows)) return rc;
    if (a.block_tables) {
        if (a.max_blocks_per_seq == 0) return GRANITE_HIP_EINVAL;
        const uint64_t tokens = uint64_t(a.block_size) * a.max_blocks_per_seq;
        if (tokens >= (1ull << 31)) return GRANITE_HIP_EINVAL;
        p.max_tokens = uint32_t(tokens);
        p.max_blocks = a.max_blocks_per_seq;
    } else {
        if (a.batch_size > 1 || a.max_seq == 0 || a.max_seq >= (1u << 31)) return GRANITE_HIP_EINVAL;
        p.max_tokens = a.max_seq;
        p.row_bytes = int64_t(D) * 2;
        p.head_bytes = int64_t(a.max_seq) * D * 2;
    }
    if (!a.seq_lens) {
        if (a.fixed_seq_len == 0 || a.fixed_seq_len > p.max_tokens) return GRANITE_HIP_EINVAL;
        p.max_tokens = a.fixed_seq_len;
    }
    if (!ctx().initialized) return GRANITE_HIP_ENOTINIT;
    if (scratch.query) *scratch.query = 0;
    if (a.batch_size == 0) return GRANITE_HIP_OK;
    if (plain_form(f)) return launch_decode(a, scratch);

    p.q = a.q;
    p.q_batch = int64_t(a.num_heads) * D;
    p.q_head = D;
    p.tables = a.block_tables;
    p.seq_lens = a.seq_lens;
    p.out = a.out;
    p.out_batch = p.q_batch;
    p.out_head = D;
    p.out_f32 = 1;
    p.lse = a.lse;
    p.lse_batch = a.num_heads;
    p.lse_head = 1;
    p.batch = a.batch_size;
    p.seq_q = 1;
    p.num_heads = a.num_heads;
    p.num_kv_heads = a.num_kv_heads;
    p.group = a.num_heads / a.num_kv_heads;
    p.decode = 1;
    p.causal = 1;
    p.scale_log2 = a.scale * kExLog2e;
    p.q_groups = (p.group + 15) / 16;
    // Tiles of the longest sequence: its whole length, or its window and sinks and the tiles their ends lie in.
    const bool f8 = f.kv_dtype == GRANITE_HIP_F8E4M3;
    constexpr uint32_t tile = 32;
    const uint64_t seen = p.window ? std::min(uint64_t(p.max_tokens), uint64_t(p.window) + p.sinks + 2 * tile) : p.max_tokens;
    const uint32_t tiles = uint32_t((seen + tile - 1) / tile);
    const bool q_f32 = a.q_dtype == GRANITE_HIP_F32;
    const KvCall call = call_of(p, D, q_f32, f8, rows);
    if (kv_stream_supports(p, f8, rows, tiles) && kv_stream_us(call) < kv_rows_cut(call).us) return launch_kv_stream(p, D, q_f32, f8, rows, tiles, scratch);
    return launch_rows(p, D, q_f32, f8, rows, scratch);
}

int launch_attention_ex(const granite_hip_attention_args& a, const granite_hip_kv_form& f, const ScratchSource& scratch) {
    if (!a.q || !a.out) return GRANITE_HIP_ENULL;
    if (a.head_dim != 128 && a.head_dim != 64) return GRANITE_HIP_EUNSUPPORTED;
    const uint32_t D = a.head_dim;
    if (a.num_heads == 0 || a.num_kv_heads == 0 || a.num_heads % a.num_kv_heads != 0) return GRANITE_HIP_EINVAL;
    if ((a.q_dtype != GRANITE_HIP_F32 && a.q_dtype != GRANITE_HIP_F16) ||
        (a.out_dtype != GRANITE_HIP_F32 && a.out_dtype != GRANITE_HIP_F16))
        return GRANITE_HIP_EINVAL;
    if (a.mask_mode == GRANITE_HIP_MASK_TREE || a.extra_len != 0) return GRANITE_HIP_EUNSUPPORTED;
    if (a.mask_mode != GRANITE_HIP_MASK_CAUSAL && a.mask_mode != GRANITE_HIP_MASK_NONE) return GRANITE_HIP_EINVAL;
    if (a.mask_mode == GRANITE_HIP_MASK_NONE && f.window != 0) return GRANITE_HIP_EUNSUPPORTED;
    if (a.cache_len == 0 || a.cache_len >= (1u << 31)) return GRANITE_HIP_EINVAL;
    if (uint64_t(a.start_pos) + a.seq_q >= (1ull << 31)) return GRANITE_HIP_EINVAL;
    if (uint64_t(a.seq_q) * (a.num_heads / a.num_kv_heads) >= (1ull << 31)) return GRANITE_HIP_EINVAL;  // rows of a KV head
    if (!a.k_cache || !a.v_cache) return GRANITE_HIP_ENULL;
    if (!a.block_table && a.max_seq < a.cache_len) return GRANITE_HIP_EINVAL;
    const int64_t qes = a.q_dtype == GRANITE_HIP_F32 ? 4 : 2, oes = a.out_dtype == GRANITE_HIP_F32 ? 4 : 2;
    if ((a.q_tok_stride * qes) % 16 || (a.q_head_stride * qes) % 16 || !aligned16(a.q) || (a.out_tok_stride * oes) % 16 ||
        (a.out_head_stride * oes) % 16 || !aligned16(a.out))
        return GRANITE_HIP_EINVAL;
    KvParams p{};
    int rows = 0;
    if (int rc = check_form(f, a.k_cache, a.v_cache, a.block_table, a.block_size, a.num_kv_heads, D, p, rows)) return rc;
    if (!a.block_table) {
        p.row_bytes = int64_t(D) * 2;
        p.head_bytes = int64_t(a.max_seq) * D * 2;
    }
    if (!ctx().initialized) return GRANITE_HIP_ENOTINIT;
    if (scratch.query) *scratch.query = 0;
    if (a.seq_q == 0) return GRANITE_HIP_OK;
    if (plain_form(f)) return launch_attention(a, scratch);

    p.q = a.q;
    p.q_tok = a.q_tok_stride;
    p.q_head = a.q_head_stride;
    p.tables = a.block_table;
    p.out = a.out;
    p.out_tok = a.out_tok_stride;
    p.out_head = a.out_head_stride;
    p.out_f32 = a.out_dtype == GRANITE_HIP_F32;
    p.lse = a.lse;
    p.lse_tok = 1;
    p.lse_head = a.seq_q;
    p.batch = 1;
    p.seq_q = a.seq_q;
    p.num_heads = a.num_heads;
    p.num_kv_heads = a.num_kv_heads;
    p.group = a.num_heads / a.num_kv_heads;
    p.max_tokens = a.cache_len;
    p.causal = a.mask_mode == GRANITE_HIP_MASK_CAUSAL;
    p.start_pos = a.start_pos;
    p.scale_log2 = a.scale * kExLog2e;
    // The quickest of three (kv_choice.h): the row kernel, which takes anything; the tiles kernel; for 8-bit pools the persistent
    // kernel of the decode step, 16 rows in the place of a head's group.
    const bool f8 = f.kv_dtype == GRANITE_HIP_F8E4M3, q_f32 = a.q_dtype == GRANITE_HIP_F32;
    const KvCall call = call_of(p, D, q_f32, f8, rows);
    int tile_rows = rows;
    if (rows == kExPagedAny && a.block_size % 4 == 0 && p.row_bytes < (1 << 27)) tile_rows = kExPaged4;
    const bool tiled = tile_rows != kExPagedAny;
    const uint64_t seen = p.window ? std::min(uint64_t(p.max_tokens), uint64_t(p.window) + a.seq_q + p.sinks + 64) : p.max_tokens;
    const uint32_t tiles = uint32_t((seen + 31) / 32);
    p.q_groups = uint32_t((call.rows + 15) / 16);
    const bool streamed = f8 && call.rows <= kStreamRows && kv_stream_supports(p, f8, rows, tiles);
    const double rows_us = kv_rows_cut(call).us, tiles_us = tiled ? kv_tiles_cut(call).us : INFINITY, stream_us = streamed ? kv_stream_us(call) : INFINITY;
    if (stream_us < std::min(rows_us, tiles_us)) return launch_kv_stream(p, D, q_f32, f8, rows, tiles, scratch);
    if (tiles_us < rows_us) return launch_kv_tiles(p, call, q_f32, tile_rows, scratch);
    return launch_rows(p, D, q_f32, f8, rows, scratch);
}

}  // namespace ghip
