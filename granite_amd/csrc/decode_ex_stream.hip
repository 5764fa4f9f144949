// Decode over 8-bit pools and windowed caches, persistent form: one workgroup per CU walks an equal share of the
// visible key tiles of the whole batch.
//
// The flat list is ordered (sequence, list head, tile): the tiles are those of kv_visible.h, so under a window a long
// sequence contributes its window and its sinks and nothing else.  Workers take equal contiguous ranges of the list; one that
// crosses from a (sequence, list head) into the next writes a partial (m, l, O) for what it covered, and the merge
// kernel joins them.  A piece's slot is worker + segment, segment = sequence * lists + list head (from one piece
// to the next the worker or the segment grows), so there are workers + batch * lists slots however long
// the sequences are.  There is no planning launch: every workgroup scans the lengths into tile counts and
// their prefix sums itself, in LDS.
//
// Three shapes of the list, by how many heads there are (a head here: 16 query heads of a KV head's group, or fewer):
//   kPair   a multiple of 8: a list head is 8 of them, a worker is a workgroup, its four waves walk the
//           same tiles for two heads each, in alternation, so that a workgroup reads whole token rows at a time,
//   kQuad   a multiple of 4: the same with one head per wave,
//   kFlat   otherwise: a worker is a wave, a list head is one head.
//
// Inside a wave the K and V of the next tile (or the other head) are in flight while one is computed; its
// block-table entries are a tile further ahead, and the scales, which need the entries, are requested just before
// the K and V they belong to.  All loads are unconditional: a load inside a branch would make the
// compiler wait for every outstanding one at the join.
#include "common.h"
#include "kv_attend.h"

namespace ghip {
namespace {

constexpr uint32_t kWaves = 4;
constexpr uint32_t kPlanHeader = 4;
constexpr uint32_t kMaxPrefix = 7680;  // lengths and prefix sums in LDS: 60 KiB
enum : int { kFlat = 0, kQuad = 1, kPair = 2 };

__device__ __forceinline__ uint32_t list_heads(int shape) { return shape == kPair ? 8u : shape == kQuad ? 4u : 1u; }

// First query head of list head `lh`.
__device__ __forceinline__ uint32_t first_query_head(const KvParams& p, uint32_t lh, uint32_t per_list) {
    const uint32_t v0 = lh * per_list;
    return (v0 / p.q_groups) * p.group + (v0 % p.q_groups) * 16;
}

template <bool kQF32, bool kF8, int kRows, int kD, int kShape>
__global__ void __launch_bounds__(kWaves* kWave, 1) kv_stream_kernel(KvParams p) {
    using T = Tile<kF8, kRows, kD>;
    using R = Rows16<kQF32, kF8, kD>;
    const uint32_t lane = threadIdx.x & 63, wave = ex_uniform(threadIdx.x >> 6);
    const uint32_t n = lane & 15, g = lane >> 4;
    const uint32_t worker = kShape == kFlat ? blockIdx.x * kWaves + wave : blockIdx.x;
    const uint32_t per_list = list_heads(kShape);

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
    const uint32_t lists = vheads / per_list;
    const uint32_t total = tiles_total * lists;
    const uint32_t per = max((total + p.workers - 1) / p.workers, p.min_per);
    if (blockIdx.x == 0) {  // for the merge kernel
        for (uint32_t i = threadIdx.x; i <= p.batch; i += blockDim.x) p.plan[kPlanHeader + i] = s_prefix[i];
        if (threadIdx.x == 0) {
            p.plan[0] = per;
            p.plan[1] = per_list;
        }
    }
    auto prefix_u = [&](uint32_t i) __attribute__((always_inline)) { return ex_uniform(s_prefix[i]); };

    const uint32_t u0 = worker * per;
    if (u0 >= total) return;
    const uint32_t n_units = min(per, total - u0);

    struct Cursor {
        uint32_t b, lh, t;  // sequence, list head, tile among those it visits
        uint32_t len;
        VisibleTiles seen;
    };
    Cursor first;
    {
        uint32_t lo = 0, hi = p.batch;  // prefix[lo] * lists <= u0 < prefix[hi] * lists
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (prefix_u(mid) * lists <= u0) lo = mid;
            else hi = mid;
        }
        first.b = lo;
        first.len = ex_uniform(s_len[lo]);
        first.seen = seen_of(first.len);
        const uint32_t in_seq = u0 - prefix_u(lo) * lists;
        first.lh = in_seq / first.seen.count;
        first.t = in_seq - first.lh * first.seen.count;
    }
    // next tile in list order, skipping empty sequences; `more` false: stays (the last tile is read again
    // instead of running off the end)
    auto advance = [&](Cursor& c, bool more) __attribute__((always_inline)) {
        if (!more) return;
        if (++c.t < c.seen.count) return;
        c.t = 0;
        if (++c.lh < lists) return;
        c.lh = 0;
        uint32_t len = 0;
        while (len == 0 && ++c.b < p.batch) len = ex_uniform(s_len[c.b]);
        if (len == 0) {  // (not reached with `more`)
            c.b = p.batch - 1;
            len = 1;
        }
        c.len = len;
        c.seen = seen_of(len);
    };
    auto head_of = [&](const Cursor& c, uint32_t side) __attribute__((always_inline)) {
        return kShape == kPair ? c.lh * 8 + 2 * wave + side : kShape == kQuad ? c.lh * 4 + wave : c.lh;
    };
    auto tok_of = [&](const Cursor& c) __attribute__((always_inline)) { return c.seen.tile(c.t) * T::kTokens; };
    auto entry_of = [&](const Cursor& c) __attribute__((always_inline)) {
        return T::entry_of(p, kRows != kExContiguous ? p.tables + size_t(c.b) * p.max_blocks : nullptr, tok_of(c), c.seen, lane);
    };
    auto load_q = [&](const Cursor& c, uint32_t vh, R& st) __attribute__((always_inline)) {
        const uint32_t kvh = vh / p.q_groups, in_group = (vh % p.q_groups) * 16 + n;
        const bool live = in_group < p.group;
        st.load_q(p, int64_t(c.b) * p.q_batch + int64_t(kvh * p.group + (live ? in_group : 0)) * p.q_head, live, g);
    };
    auto compute = [&](T& tile, const typename T::Rows& rows, const Cursor& c, R& st) __attribute__((always_inline)) {
        const uint32_t tok0 = tok_of(c);
        const bool masked = T::needs_mask(p, rows, tok0, c.seen.lo, c.len);
        attend_tile<kQF32, kF8, kRows, kD, false>(p, tile, rows, tok0, c.seen, c.seen.lo, c.len, masked, st, lane);
    };
    auto flush = [&](const Cursor& c, uint32_t vh, R& st) __attribute__((always_inline)) {
        float l = st.l;
        l += wave_shfl_xor(l, 16);
        l += wave_shfl_xor(l, 32);
        const uint32_t kvh = vh / p.q_groups, in_group = (vh % p.q_groups) * 16 + n;
        if (in_group < p.group && 32 * g < uint32_t(kD)) {
            const uint32_t piece = worker + c.b * lists + c.lh;
            const uint32_t local = kvh * p.group + in_group - first_query_head(p, c.lh, per_list);
            const size_t at = size_t(piece) * p.part_cap + local;
            float* po = p.part_o + at * kD + 32 * g;
            const float unit = st.vref * (1.0f / kExBoost);
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

    Cursor cc = first, cl = first, cr = first;  // tile computed, tile whose K and V are requested, tile looked up
    T ta, tb;
    typename T::Rows ra, rb;
    if constexpr (kShape == kPair) {
        // buffer a: the wave's first head of a tile, b: its second
        R ha, hb;
        ha.clear();
        hb.clear();
        typename T::Entry entry = entry_of(cr);
        advance(cr, 1 < n_units);
        auto rows_for = [&](const Cursor& c, uint32_t side) __attribute__((always_inline)) {
            return T::rows_from(p, entry, head_of(c, side) / p.q_groups, tok_of(c), c.seen, lane);
        };
        ra = rows_for(cl, 0);
        rb = rows_for(cl, 1);
        entry = entry_of(cr);
        advance(cr, 2 < n_units);
        ta.load(p, ra, head_of(cl, 0) / p.q_groups, lane);
        load_q(cc, head_of(cc, 0), ha);
        load_q(cc, head_of(cc, 1), hb);
        for (uint32_t i = 0; i < n_units; i++) {
            tb.load(p, rb, head_of(cl, 1) / p.q_groups, lane);
            advance(cl, i + 1 < n_units);
            compute(ta, ra, cc, ha);
            ra = rows_for(cl, 0);
            const typename T::Rows rb_next = rows_for(cl, 1);
            entry = entry_of(cr);
            advance(cr, i + 3 < n_units);
            ta.load(p, ra, head_of(cl, 0) / p.q_groups, lane);  // the next tile (at the very end this one again)
            compute(tb, rb, cc, hb);
            rb = rb_next;
            const bool last = i + 1 >= n_units, seg_end = last || cc.t + 1 == cc.seen.count;
            const Cursor done = cc;
            advance(cc, !last);
            if (seg_end) {
                flush(done, head_of(done, 0), ha);
                flush(done, head_of(done, 1), hb);
                if (!last) {
                    load_q(cc, head_of(cc, 0), ha);
                    load_q(cc, head_of(cc, 1), hb);
                }
            }
        }
    } else {
        R h;
        h.clear();
        auto rows_for = [&](const Cursor& c, const typename T::Entry& e) __attribute__((always_inline)) {
            return T::rows_from(p, e, head_of(c, 0) / p.q_groups, tok_of(c), c.seen, lane);
        };
        typename T::Entry entry = entry_of(cr);
        advance(cr, 1 < n_units);
        ra = rows_for(cl, entry);
        entry = entry_of(cr);
        advance(cr, 2 < n_units);
        ta.load(p, ra, head_of(cl, 0) / p.q_groups, lane);
        advance(cl, 1 < n_units);
        load_q(cc, head_of(cc, 0), h);
        // one unit: the next tile into (tn, rn) while (t, r) is computed; false behind the last
        auto unit = [&](uint32_t i, T& t, typename T::Rows& r, T& tn, typename T::Rows& rn) __attribute__((always_inline)) {
            rn = rows_for(cl, entry);
            entry = entry_of(cr);
            advance(cr, i + 3 < n_units);
            tn.load(p, rn, head_of(cl, 0) / p.q_groups, lane);
            advance(cl, i + 2 < n_units);
            compute(t, r, cc, h);
            const bool last = i + 1 >= n_units, seg_end = last || cc.t + 1 == cc.seen.count;
            const Cursor done = cc;
            advance(cc, !last);
            if (seg_end) {
                flush(done, head_of(done, 0), h);
                if (!last) load_q(cc, head_of(cc, 0), h);
            }
            return !last;
        };
        for (uint32_t i = 0;; i += 2) {
            if (!unit(i, ta, ra, tb, rb)) break;
            if (!unit(i + 1, tb, rb, ta, ra)) break;
        }
    }
}

// Joins the pieces of one (sequence, query head): the workers that touched its list head are consecutive.
__global__ void __launch_bounds__(kHeadDim) kv_stream_merge_kernel(KvParams p, uint32_t D) {
    const uint32_t qh = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
    const uint32_t* prefix = p.plan + kPlanHeader;
    const uint32_t nt = prefix[b + 1] - prefix[b];
    if (nt == 0) return;  // empty sequence: its output stays
    const uint32_t per = p.plan[0], per_list = p.plan[1];
    const uint32_t lists = p.num_kv_heads * p.q_groups / per_list;
    const uint32_t lh = ((qh / p.group) * p.q_groups + (qh % p.group) / 16) / per_list;
    const uint32_t u_start = prefix[b] * lists + lh * nt;
    const uint32_t first_worker = u_start / per, n_parts = (u_start + nt - 1) / per - first_worker + 1;
    const size_t at0 = size_t(first_worker + b * lists + lh) * p.part_cap + (qh - first_query_head(p, lh, per_list));
    float mx = kExNegBig, o = 0.0f, l = 0.0f;
    for (uint32_t c0 = 0; c0 < n_parts; c0 += 4) {  // four at a time: their loads are in flight together
        float m[4], ls[4], os[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const size_t at = at0 + size_t(min(c0 + i, n_parts - 1)) * p.part_cap;
            m[i] = p.part_ml[2 * at];
            ls[i] = p.part_ml[2 * at + 1];
            os[i] = p.part_o[at * D + d];
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
    static_cast<float*>(p.out)[int64_t(b) * p.out_batch + int64_t(qh) * p.out_head + d] = l == 0.0f ? 0.0f : o / l;
    if (p.lse && d == 0)
        p.lse[int64_t(b) * p.lse_batch + int64_t(qh) * p.lse_head] = l == 0.0f ? -INFINITY : (mx + __builtin_amdgcn_logf(l)) * kExLn2;
}

template <bool kQF32, bool kF8, int kRows, int kD>
void launch_shape(const KvParams& p, int shape, dim3 grid, size_t lds) {
    const dim3 block(kWaves * kWave);
    hipStream_t st = ctx().stream;
    if (shape == kPair) kv_stream_kernel<kQF32, kF8, kRows, kD, kPair><<<grid, block, lds, st>>>(p);
    else if (shape == kQuad) kv_stream_kernel<kQF32, kF8, kRows, kD, kQuad><<<grid, block, lds, st>>>(p);
    else kv_stream_kernel<kQF32, kF8, kRows, kD, kFlat><<<grid, block, lds, st>>>(p);
}
template <bool kQF32, int kD>
void launch_cache(const KvParams& p, int shape, dim3 grid, size_t lds, bool f8, int rows) {
    if (f8 && rows == kExPaged16) launch_shape<kQF32, true, kExPaged16, kD>(p, shape, grid, lds);
    else if (f8) launch_shape<kQF32, true, kExPagedAny, kD>(p, shape, grid, lds);
    else if (rows == kExContiguous) launch_shape<kQF32, false, kExContiguous, kD>(p, shape, grid, lds);
    else if (rows == kExPaged16) launch_shape<kQF32, false, kExPaged16, kD>(p, shape, grid, lds);
    else launch_shape<kQF32, false, kExPagedAny, kD>(p, shape, grid, lds);
}

}  // namespace

bool kv_stream_supports(const KvParams& p, uint32_t tiles_per_seq) {
    const uint64_t units = uint64_t(p.batch) * tiles_per_seq * p.num_kv_heads * p.q_groups;
    return p.batch + 1 <= kMaxPrefix && units < (1ull << 31) && p.num_heads <= 0x7FFFFFFFu && p.batch <= 65535u;
}

int launch_kv_stream(KvParams p, uint32_t D, bool q_f32, bool f8, int rows, uint32_t tiles_per_seq, const ScratchSource& scratch) {
    const uint32_t cus = ctx().compute_units > 0 ? uint32_t(ctx().compute_units) : 256u;
    const uint32_t vheads = p.num_kv_heads * p.q_groups;
    const int shape = vheads % 8 == 0 ? kPair : vheads % 4 == 0 ? kQuad : kFlat;
    const uint32_t per_list = shape == kPair ? 8 : shape == kQuad ? 4 : 1;
    const uint32_t lists = vheads / per_list;
    p.workers = shape == kFlat ? cus * kWaves : cus;
    // smallest range of a worker: a short batch is not cut into ranges of a tile or two, each with a partial to join
    p.min_per = max(1u, min(4u, (tiles_per_seq + 31) / 32));
    p.part_cap = per_list * min(p.group, 16u);
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
        KernelTimerScope timer("decode_ex");
        const dim3 grid(cus);
        if (D == 128) {
            if (q_f32) launch_cache<true, 128>(p, shape, grid, lds, f8, rows);
            else launch_cache<false, 128>(p, shape, grid, lds, f8, rows);
        } else {
            if (q_f32) launch_cache<true, 64>(p, shape, grid, lds, f8, rows);
            else launch_cache<false, 64>(p, shape, grid, lds, f8, rows);
        }
    }
    if (int rc = launch_status()) return rc;
    {
        KernelTimerScope timer("decode_ex_merge");
        kv_stream_merge_kernel<<<dim3(p.num_heads, p.batch), dim3(D), 0, ctx().stream>>>(p, D);
    }
    return launch_status();
}

}  // namespace ghip
