// Decode through a window over half caches, persistent form: one workgroup per CU walks an equal share of the visible
// key tiles of the whole batch; the joining of its pieces, and of those of decode_ex_dma.hip, which does the same over
// 8-bit pools.  Contiguous caches, and pools whose blocks are multiples of 16 tokens: where every token has a table entry of
// its own the row kernel is as quick (64 sequences of 8192 over 8-bit blocks of 20: 227 us against 306).
//
// The flat list is ordered (sequence, list head, tile): the tiles are those of kv_visible.h, so under a window a long
// sequence contributes its window and its sinks and nothing else.  Workers take equal contiguous ranges of the list; one that
// crosses from a (sequence, list head) into the next writes a partial (m, l, O) for what it covered, and the merge
// kernel joins them.  A piece's slot is worker + segment, segment = sequence * lists + list head (from one piece
// to the next the worker or the segment grows), so there are workers + batch * lists slots however long
// the sequences are.  There is no planning launch: every workgroup scans the lengths into tile counts and
// their prefix sums itself, in LDS.
//
// A workgroup has eight waves, two per SIMD.  Where the KV heads (a head here: 16 query heads of a KV head's group, or
// fewer) come in multiples of kPer = 8, 4 or 2, a list head is kPer of them and a worker is kPer waves that walk the same tiles,
// one head each, so that together they read whole (halves, quarters of) token rows at about the same time; otherwise a
// worker is a wave.
//
// Inside a wave the K and V of the next tile are in flight while one is computed (16 KiB; 128 KiB per CU); its
// block-table entries are a tile further ahead.  Measured (32 heads over 8 KV heads of 128): 64 sequences of 256 to 8192 tokens
// through a window of 1024 58 us a call for 260 MB, 4.5 TB/s; through one of 4096 170 us, 4.8 TB/s.  All loads are unconditional: a load inside a branch would make the
// compiler wait for every outstanding one at the join.
#include <algorithm>

#include "common.h"
#include "kv_attend.h"

namespace ghip {
namespace {

constexpr uint32_t kWaves = 8;
constexpr uint32_t kPlanHeader = 4;

template <bool kQF32, int kRows, int kD, uint32_t kPer>
__global__ void __launch_bounds__(kWaves* kWave, 2) kv_stream_kernel(KvParams p) {
    using T = Tile<false, kRows, kD>;
    using R = Rows16<kQF32, false, kD>;
    const uint32_t lane = threadIdx.x & 63, wave = ex_uniform(threadIdx.x >> 6);
    const uint32_t n = lane & 15, g = lane >> 4;
    const uint32_t worker = blockIdx.x * (kWaves / kPer) + wave / kPer;

    // ---- tile counts and their prefix sums
    extern __shared__ uint32_t s_dyn[];
    uint32_t* s_prefix = s_dyn;             // [batch + 1]
    uint32_t* s_len = s_dyn + p.batch + 1;  // [batch]
    __shared__ uint32_t s_wave_sum[kWaves];
    const uint32_t vheads = p.num_kv_heads * p.q_groups;
    auto seen_of = [&](uint32_t len) __attribute__((always_inline)) { return visible_tiles<T::kTokens>(len - 1, len, p.window, p.sinks); };
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
    if (blockIdx.x == 0) {  // for the merge kernel
        for (uint32_t i = threadIdx.x; i <= p.batch; i += blockDim.x) p.plan[kPlanHeader + i] = s_prefix[i];
        if (threadIdx.x == 0) {
            p.plan[0] = per;
            p.plan[1] = kPer;
        }
    }

    const uint32_t u0 = worker * per;
    if (u0 >= total) return;
    const uint32_t n_units = min(per, total - u0);

    // ---- what the units are.  Lane u of a wave works out unit i0 + u of its worker's range, 64 at a time and in
    // parallel; the loop reads them back lane by lane, so that it carries no position in the list and no branches of
    // one.  Units behind the last are the last again (no load runs off the end).
    uint32_t d_tok = 0, d_len = 0, d_b = 0, d_lh = 0;  // first token, the sequence's length, sequence, list head | end of segment << 31
    uint32_t search_steps = 0;
    while ((1u << search_steps) < p.batch) search_steps++;
    auto plan_units = [&](uint32_t i0) __attribute__((always_inline)) {
        const uint32_t u = u0 + min(i0 + lane, n_units - 1);
        uint32_t lo = 0, hi = p.batch;  // prefix[lo] * lists <= u < prefix[hi] * lists
        for (uint32_t i = 0; i < search_steps; i++) {
            const uint32_t mid = (lo + hi) >> 1;
            const bool below = s_prefix[mid] * lists <= u;  // (mid = lo once they are neighbours: true)
            lo = below ? mid : lo;
            hi = below ? hi : mid;
        }
        const uint32_t len = s_len[lo], in_seq = u - s_prefix[lo] * lists;
        const VisibleTiles seen = seen_of(max(len, 1u));
        const uint32_t lh = in_seq / seen.count, t = in_seq - lh * seen.count;
        d_b = lo;
        d_len = len;
        d_lh = lh | (t + 1 == seen.count ? 0x80000000u : 0u);
        d_tok = seen.tile(t) * T::kTokens;
    };
    uint32_t i0 = 0;
    auto of_unit = [&](uint32_t d, uint32_t i) __attribute__((always_inline)) { return uint32_t(__builtin_amdgcn_readlane(int(d), int(i - i0))); };
    auto head_at = [&](uint32_t i) __attribute__((always_inline)) { return (of_unit(d_lh, i) & 0x7FFFFFFFu) * kPer + wave % kPer; };
    auto kv_head_at = [&](uint32_t i) __attribute__((always_inline)) { return p.q_groups == 1 ? head_at(i) : head_at(i) / p.q_groups; };
    auto entry_of = [&](uint32_t i) __attribute__((always_inline)) {
        return T::entry_of(p, kRows != kExContiguous ? p.tables + size_t(of_unit(d_b, i)) * p.max_blocks : nullptr, of_unit(d_tok, i),
                           seen_of(of_unit(d_len, i)), lane);
    };
    auto load_q = [&](uint32_t i, R& st) __attribute__((always_inline)) {
        const uint32_t vh = head_at(i), kvh = vh / p.q_groups, in_group = (vh % p.q_groups) * 16 + n;
        const bool live = in_group < p.group;
        st.load_q(p, int64_t(of_unit(d_b, i)) * p.q_batch + int64_t(kvh * p.group + (live ? in_group : 0)) * p.q_head, live, g);
    };
    auto compute = [&](uint32_t i, T& tile, const typename T::Rows& rows, R& st) __attribute__((always_inline)) {
        const uint32_t len = of_unit(d_len, i), tok0 = of_unit(d_tok, i);
        const VisibleTiles seen = seen_of(len);
        const bool masked = T::needs_mask(p, rows, tok0, seen.lo, len);
        attend_tile<kQF32, false, kRows, kD, false>(p, tile, rows, tok0, seen, seen.lo, len, masked, st, lane);
    };
    auto flush = [&](uint32_t i, R& st) __attribute__((always_inline)) {
        const uint32_t vh = head_at(i), lh = of_unit(d_lh, i) & 0x7FFFFFFFu;
        float l = st.l;
        l += wave_shfl_xor(l, 16);
        l += wave_shfl_xor(l, 32);
        const uint32_t in_group = (vh % p.q_groups) * 16 + n;
        if (in_group < p.group && 32 * g < uint32_t(kD)) {
            const uint32_t piece = worker + of_unit(d_b, i) * lists + lh;
            const size_t at = size_t(piece) * p.part_cap + (wave % kPer) * (p.part_cap / kPer) + n;
            float* po = p.part_o + at * kD + 32 * g;
            const float unit = ex_unit(st.bound);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float4v w;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int e = 4 * i + k;
                    w[k] = st.acc[e & 7][e >> 3] * unit;
                }
                *reinterpret_cast<float4v*>(po + 4 * i) = w;
            }
            if (g == 0) {
                p.part_ml[at * 2] = st.m;
                p.part_ml[at * 2 + 1] = l;
            }
        }
        st.clear();
    };

    T ta, tb;
    typename T::Rows ra, rb;
    R h;
    h.clear();
    auto rows_for = [&](uint32_t i, const typename T::Entry& e) __attribute__((always_inline)) {
        return T::rows_from(p, e, kv_head_at(i), of_unit(d_tok, i), seen_of(of_unit(d_len, i)), lane);
    };
    plan_units(0);
    typename T::Entry entry = entry_of(0);
    ra = rows_for(0, entry);
    entry = entry_of(1);
    ta.load(p, ra, kv_head_at(0), lane);
    load_q(0, h);
    // one unit: the next tile into (tn, rn) while (t, r) is computed; false behind the last
    auto unit = [&](uint32_t i, T& t, typename T::Rows& r, T& tn, typename T::Rows& rn) __attribute__((always_inline)) {
        if (i + 2 - i0 >= kWave) {
            i0 = i;
            plan_units(i0);
        }
        rn = rows_for(i + 1, entry);
        entry = entry_of(i + 2);
        tn.load(p, rn, kv_head_at(i + 1), lane);
        compute(i, t, r, h);
        const bool last = i + 1 >= n_units;
        if (last || (of_unit(d_lh, i) >> 31)) {
            flush(i, h);
            if (!last) load_q(i + 1, h);
        }
        return !last;
    };
    for (uint32_t i = 0;; i += 2) {
        if (!unit(i, ta, ra, tb, rb)) break;
        if (!unit(i + 1, tb, rb, ta, ra)) break;
    }
}

// Joins the pieces of one (sequence, row): the workers that touched its list head are consecutive.  kJoin
// groups of threads take four pieces at a time in turn and are joined through LDS: 4 where sequences are few (a long
// one alone has a piece of every worker: 2 sequences of 131072 tokens 17.5 -> 7.3 us), 1 where they are many and short
// of pieces (64 sequences: 5.3 us against 6.8).
template <int kD, uint32_t kJoin>
__global__ void __launch_bounds__(kD* kJoin) kv_stream_merge_kernel(KvParams p) {
    const uint32_t n_rows = p.seq_q * p.group;  // of a KV head: (query, head of the group) pairs
    const uint32_t kvh = blockIdx.x / n_rows, row = blockIdx.x - kvh * n_rows;
    const uint32_t b = blockIdx.y, d = threadIdx.x % kD, part = threadIdx.x / kD;
    const uint32_t* prefix = p.plan + kPlanHeader;
    const uint32_t nt = prefix[b + 1] - prefix[b];
    if (nt == 0 && p.decode) return;  // empty sequence: its output stays
    // (several queries whose windows lie behind the cache have no tile either: they see nothing, which is a result)
    const uint32_t per = p.plan[0], per_list = p.plan[1];
    const uint32_t lists = p.num_kv_heads * p.q_groups / per_list;
    const uint32_t vh = kvh * p.q_groups + row / 16, lh = vh / per_list;
    const uint32_t u_start = prefix[b] * lists + lh * nt;
    const uint32_t first_worker = u_start / per, n_parts = nt == 0 ? 0 : (u_start + nt - 1) / per - first_worker + 1;
    const size_t at0 = size_t(first_worker + b * lists + lh) * p.part_cap + (vh % per_list) * (p.part_cap / per_list) + row % 16;
    float mx = kExNegBig, o = 0.0f, l = 0.0f;
    for (uint32_t c0 = 4 * part; c0 < n_parts; c0 += 4 * kJoin) {  // four at a time: their loads are in flight together
        float m[4], ls[4], os[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const size_t at = at0 + size_t(min(c0 + i, n_parts - 1)) * p.part_cap;
            m[i] = p.part_ml[2 * at];
            ls[i] = p.part_ml[2 * at + 1];
            os[i] = p.part_o[at * kD + d];
        }
        float m_new = mx;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) m_new = fmaxf(m_new, c0 + i < n_parts ? m[i] : kExNegBig);
        const float keep = fast_exp2(mx - m_new);
        o *= keep;
        l *= keep;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            if (c0 + i >= n_parts) continue;
            const float f = fast_exp2(m[i] - m_new);
            l += ls[i] * f;
            o += os[i] * f;
        }
        mx = m_new;
    }
    if (kJoin > 1 && n_parts > 4) {  // uniform
        __shared__ float s_o[kJoin][kD], s_m[kJoin], s_l[kJoin];
        s_o[part][d] = o;
        if (d == 0) {
            s_m[part] = mx;
            s_l[part] = l;
        }
        __syncthreads();
        if (part != 0) return;
        for (uint32_t i = 0; i < kJoin; i++) mx = fmaxf(mx, s_m[i]);
        o = l = 0.0f;
        for (uint32_t i = 0; i < kJoin; i++) {
            const float f = fast_exp2(s_m[i] - mx);
            o += s_o[i][d] * f;
            l += s_l[i] * f;
        }
    } else if (part != 0) {
        return;
    }
    const uint32_t query = row / p.group, head = kvh * p.group + (row - query * p.group);
    const int64_t at = int64_t(b) * p.out_batch + int64_t(query) * p.out_tok + int64_t(head) * p.out_head + d;
    const uint32_t len = ex_seq_len(p, b);
    const float result = settle_nan(p, l == 0.0f ? 0.0f : o / l, l, b, kvh, p.decode ? len - 1 : p.start_pos + query, len, d);
    if (p.out_f32) static_cast<float*>(p.out)[at] = result;
    else static_cast<_Float16*>(p.out)[at] = static_cast<_Float16>(result);
    if (p.lse && d == 0)
        p.lse[int64_t(b) * p.lse_batch + int64_t(query) * p.lse_tok + int64_t(head) * p.lse_head] =
            l == 0.0f ? -INFINITY : (mx + __builtin_amdgcn_logf(l)) * kExLn2;
}

template <bool kQF32, int kRows, int kD>
void launch_shape(const KvParams& p, uint32_t per_list, dim3 grid, size_t lds) {
    const dim3 block(kWaves * kWave);
    hipStream_t st = ctx().stream;
    if (per_list == 8) kv_stream_kernel<kQF32, kRows, kD, 8><<<grid, block, lds, st>>>(p);
    else if (per_list == 4) kv_stream_kernel<kQF32, kRows, kD, 4><<<grid, block, lds, st>>>(p);
    else if (per_list == 2) kv_stream_kernel<kQF32, kRows, kD, 2><<<grid, block, lds, st>>>(p);
    else kv_stream_kernel<kQF32, kRows, kD, 1><<<grid, block, lds, st>>>(p);
}
template <int kD>
void launch_types(const KvParams& p, uint32_t per_list, dim3 grid, size_t lds, bool q_f32, int rows) {
    if (q_f32 && rows == kExContiguous) launch_shape<true, kExContiguous, kD>(p, per_list, grid, lds);
    else if (q_f32) launch_shape<true, kExPaged16, kD>(p, per_list, grid, lds);
    else if (rows == kExContiguous) launch_shape<false, kExContiguous, kD>(p, per_list, grid, lds);
    else launch_shape<false, kExPaged16, kD>(p, per_list, grid, lds);
}

// At most kStreamMaxBatch sequences, whose lengths and prefix sums lie in LDS.
int launch_part(KvParams p, uint32_t D, bool q_f32, bool f8, int rows, uint32_t tiles_per_seq, const ScratchSource& scratch) {
    const uint32_t cus = ctx().compute_units > 0 ? uint32_t(ctx().compute_units) : 256u;
    const uint32_t vheads = p.num_kv_heads * p.q_groups;
    const uint32_t per_list = vheads % 8 == 0 ? 8 : vheads % 4 == 0 ? 4 : vheads % 2 == 0 ? 2 : 1;
    const uint32_t lists = vheads / per_list;
    p.workers = cus * (kWaves / per_list);
    // smallest range of a worker: a short batch is not cut into ranges of a tile or two, each with a partial to join
    p.min_per = std::clamp((tiles_per_seq + 31) / 32, 1u, 4u);
    p.part_cap = per_list * std::min(p.seq_q * p.group, 16u);
    const size_t slots = (size_t(p.workers) + size_t(p.batch) * lists) * p.part_cap;
    const size_t plan_bytes = ((kPlanHeader + size_t(p.batch) + 1) * sizeof(uint32_t) + 255) & ~size_t(255);
    const size_t need = plan_bytes + slots * (D + 2) * sizeof(float);
    if (scratch.query) {
        *scratch.query = need;
        return GRANITE_HIP_OK;
    }
    void* ws = nullptr;
    if (int rc = take_scratch(scratch, need, &ws)) return rc;
    p.plan = static_cast<uint32_t*>(ws);
    p.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + plan_bytes);
    p.part_ml = p.part_o + slots * D;
    const size_t lds = (2 * size_t(p.batch) + 1) * sizeof(uint32_t);
    {
        KernelTimerScope timer(p.decode ? "decode_ex" : "attention_ex");
        const dim3 grid(cus);
        if (f8) {
            if (int rc = launch_kv_dma(p, D, q_f32, per_list, grid)) return rc;
        } else if (D == 128) {
            launch_types<128>(p, per_list, grid, lds, q_f32, rows);
        } else {
            launch_types<64>(p, per_list, grid, lds, q_f32, rows);
        }
    }
    if (int rc = launch_status()) return rc;
    {
        KernelTimerScope timer(p.decode ? "decode_ex_merge" : "attention_ex_merge");
        const dim3 grid(p.seq_q * p.num_heads, p.batch);
        const bool few = size_t(p.batch) * lists * 16 <= p.workers;  // 16 pieces a segment or more if all are as long
        hipStream_t st = ctx().stream;
        if (D == 128 && few) kv_stream_merge_kernel<128, 4><<<grid, dim3(512), 0, st>>>(p);
        else if (D == 128) kv_stream_merge_kernel<128, 1><<<grid, dim3(128), 0, st>>>(p);
        else if (few) kv_stream_merge_kernel<64, 4><<<grid, dim3(256), 0, st>>>(p);
        else kv_stream_merge_kernel<64, 1><<<grid, dim3(64), 0, st>>>(p);
    }
    return launch_status();
}

}  // namespace

bool kv_stream_supports(const KvParams& p, bool f8, int rows, uint32_t tiles_per_seq) {
    if (rows == kExPagedAny || (f8 && rows == kExContiguous)) return false;
    const uint64_t units = uint64_t(std::min(p.batch, kStreamMaxBatch)) * tiles_per_seq * p.num_kv_heads * p.q_groups;
    return units < (1ull << 31) && uint64_t(p.seq_q) * p.num_heads <= 0x7FFFFFFFu;
}

int launch_kv_stream(KvParams p, uint32_t D, bool q_f32, bool f8, int rows, uint32_t tiles_per_seq, const ScratchSource& scratch) {
    const uint32_t batch = p.batch;
    for (uint32_t b = 0; b < batch; b += kStreamMaxBatch) {  // (the parts follow each other on the stream and may share the workspace)
        p.batch = std::min(batch - b, kStreamMaxBatch);
        if (int rc = launch_part(p, D, q_f32, f8, rows, tiles_per_seq, scratch)) return rc;
        if (scratch.query) break;  // the first part is the largest
        p.q = static_cast<const char*>(p.q) + size_t(p.batch) * p.q_batch * (q_f32 ? 4 : 2);
        p.out = static_cast<char*>(p.out) + size_t(p.batch) * p.out_batch * (p.out_f32 ? 4 : 2);
        if (p.tables) p.tables += size_t(p.batch) * p.max_blocks;
        if (p.seq_lens) p.seq_lens += p.batch;
        if (p.lse) p.lse += size_t(p.batch) * p.lse_batch;
    }
    return GRANITE_HIP_OK;
}

}  // namespace ghip
