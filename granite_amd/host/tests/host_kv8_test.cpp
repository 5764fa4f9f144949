// HipCompute's methods over 8-bit pools: append, decode and a chunk of queries of one sequence, against
// double-precision attention on the codes and scales the append left.
#include <cmath>
#include <cstdint>
#include <vector>

#include "check.h"
#include "granite/hip_compute.h"
#include "granite_hip.h"

using namespace granite;

static double e4m3(uint8_t c) {
    const int e = (c >> 3) & 15, m = c & 7;
    if ((c & 0x7F) == 0x7F) return NAN;
    const double v = e == 0 ? m * std::ldexp(1.0, -9) : std::ldexp(1.0 + m / 8.0, e - 7);
    return c & 0x80 ? -v : v;
}

TEST_CASE(append_decode_and_chunk_over_8bit_pools) {
    HipCompute* hc = get_hip_compute();
    REQUIRE(hc != nullptr);
    const uint32_t n = 45, hq = 4, hkv = 2, D = 64, bs = 16, blocks = 5, window = 20, sinks = 2;
    std::vector<float> k(n * hkv * D), v(k.size()), q(n * hq * D);
    uint32_t state = 12345;
    auto draw = [&] {
        state = state * 1664525u + 1013904223u;
        return float(int32_t(state)) / 1.0e9f;
    };
    for (auto* x : {&k, &v, &q})
        for (float& e : *x) e = draw();
    const std::vector<int32_t> table = {3, 0, 4};
    const int32_t len = int32_t(n);
    auto device = [&](const void* src, size_t bytes) {
        HipBuffer* b = hc->create_buffer(bytes, false);
        if (src) CHECK_OK(hc->upload(b, src, bytes));
        return b;
    };
    const size_t pool = size_t(blocks) * bs * hkv * D, scales = size_t(blocks) * hkv * sizeof(float);
    const std::vector<uint8_t> nan(pool, 0x7F);
    HipBuffer *dk = device(k.data(), k.size() * 4), *dv = device(v.data(), v.size() * 4), *dq = device(q.data(), q.size() * 4);
    HipBuffer *kc = device(nan.data(), pool), *vc = device(nan.data(), pool), *ks = device(nullptr, scales), *vs = device(nullptr, scales);
    HipBuffer *dt = device(table.data(), table.size() * 4), *dl = device(&len, 4), *rq = device(nullptr, q.size() * 4);
    HipBuffer *out = device(nullptr, q.size() * 4), *lse = device(nullptr, size_t(n) * hq * 4);

    granite_hip_rope_q8_args r{};
    r.q = dq; r.q_out = rq; r.k = dk; r.v = dv;
    r.src_dtype = GRANITE_HIP_F32; r.q_out_dtype = GRANITE_HIP_F32;
    r.k_cache = kc; r.v_cache = vc;
    r.k_scale = static_cast<float*>(ks); r.v_scale = static_cast<float*>(vs);
    r.block_table = static_cast<const int32_t*>(dt);
    r.freq_base = 10000.0f;
    r.num_heads_q = hq; r.num_heads_k = hkv; r.seq_len = n; r.head_dim = D;
    r.block_size = bs; r.num_blocks = blocks; r.max_blocks_per_seq = 3;
    CHECK_OK(hc->rope_append_q8(r));
    r.seq_len = 49;
    CHECK_CODE(hc->rope_append_q8(r), ErrorCode::InvalidArgument);  // beyond the block table
    hc->sync();

    std::vector<uint8_t> kcode(pool), vcode(pool);
    std::vector<float> kscale(scales / 4), vscale(scales / 4), rot(q.size());
    CHECK_OK(hc->download(kcode.data(), kc, pool));
    CHECK_OK(hc->download(vcode.data(), vc, pool));
    CHECK_OK(hc->download(kscale.data(), ks, scales));
    CHECK_OK(hc->download(vscale.data(), vs, scales));
    CHECK_OK(hc->download(rot.data(), rq, q.size() * 4));
    auto want = [&](uint32_t pos, uint32_t h, std::vector<double>& o) {
        std::vector<double> s(n, -INFINITY);
        double top = -INFINITY, sum = 0;
        for (uint32_t t = 0; t <= pos; t++) {
            if (t + window <= pos && t >= sinks) continue;
            const uint32_t b = uint32_t(table[t / bs]);
            double x = 0;
            for (uint32_t d = 0; d < D; d++)
                x += double(rot[(size_t(pos) * hq + h) * D + d]) * e4m3(kcode[((b * bs + t % bs) * hkv + h / 2) * D + d]);
            s[t] = x * kscale[b * hkv + h / 2] * 0.125;
            top = std::fmax(top, s[t]);
        }
        o.assign(D, 0.0);
        for (uint32_t t = 0; t <= pos; t++) {
            const double e = std::exp(s[t] - top);
            sum += e;
            const uint32_t b = uint32_t(table[t / bs]);
            for (uint32_t d = 0; d < D && e > 0; d++)
                o[d] += e * e4m3(vcode[((b * bs + t % bs) * hkv + h / 2) * D + d]) * vscale[b * hkv + h / 2];
        }
        for (double& x : o) x /= sum;
        return top + std::log(sum);
    };
    // a score is a float sum of D products of at most 2.15 * 2.15 * 1.5 (the rotation), times 0.125: its D + 4
    // roundings move it by at most (64 + 4) * 2^-24 * 64 * 7 * 0.125 = 2.3e-4; output and log-sum-exp are off by at
    // most twice that on values below 2.3, with the sums of 22 terms beside it
    const double tol = 2 * 2.4e-4 * 2.3;

    granite_hip_kv_form f{};
    f.kv_dtype = GRANITE_HIP_F8E4M3;
    f.k_scale = r.k_scale; f.v_scale = r.v_scale;
    f.num_blocks = blocks; f.window = window; f.num_sinks = sinks;
    granite_hip_attention_args a{};
    a.q = rq; a.q_dtype = GRANITE_HIP_F32; a.q_tok_stride = hq * D; a.q_head_stride = D;
    a.out = out; a.out_dtype = GRANITE_HIP_F32; a.out_tok_stride = hq * D; a.out_head_stride = D;
    a.lse = static_cast<float*>(lse);
    a.k_cache = kc; a.v_cache = vc; a.block_table = r.block_table; a.block_size = bs;
    a.cache_len = n; a.mask_mode = GRANITE_HIP_MASK_CAUSAL; a.seq_q = n;
    a.num_heads = hq; a.num_kv_heads = hkv; a.head_dim = D; a.scale = 0.125f;
    auto need = hc->attention_ex_workspace_required(a, f);
    CHECK(need.ok());
    CHECK_OK(hc->attention_ex(a, f));
    hc->sync();
    std::vector<float> got(q.size()), got_lse(size_t(n) * hq);
    std::vector<double> o;
    CHECK_OK(hc->download(got.data(), out, got.size() * 4));
    CHECK_OK(hc->download(got_lse.data(), lse, got_lse.size() * 4));
    int bad = 0;
    for (uint32_t p = 0; p < n; p++)
        for (uint32_t h = 0; h < hq; h++) {
            bad += !(std::fabs(got_lse[size_t(h) * n + p] - want(p, h, o)) <= tol);
            for (uint32_t d = 0; d < D; d++) bad += !(std::fabs(got[(size_t(p) * hq + h) * D + d] - o[d]) <= tol);
        }
    CHECK(bad == 0);

    granite_hip_decode_args d{};
    d.q = static_cast<float*>(rq) + size_t(n - 1) * hq * D;  // the last token's queries
    d.q_dtype = GRANITE_HIP_F32;
    d.k_cache = kc; d.v_cache = vc; d.block_tables = r.block_table;
    d.seq_lens = static_cast<const int32_t*>(dl);
    d.out = out; d.lse = static_cast<float*>(lse);
    d.batch_size = 1; d.num_heads = hq; d.num_kv_heads = hkv; d.head_dim = D;
    d.block_size = bs; d.max_blocks_per_seq = 3; d.scale = 0.125f;
    auto dneed = hc->decode_ex_workspace_required(d, f);
    CHECK(dneed.ok());
    HipBuffer* ws = device(nullptr, dneed.value() + 256);
    CHECK_OK(hc->decode_attention_ex(d, f, ws, dneed.value() + 256));
    hc->sync();
    CHECK_OK(hc->download(got.data(), out, size_t(hq) * D * 4));
    CHECK_OK(hc->download(got_lse.data(), lse, hq * 4));
    for (uint32_t h = 0; h < hq; h++) {
        CHECK(std::fabs(got_lse[h] - want(n - 1, h, o)) <= tol);
        for (uint32_t e = 0; e < D; e++) bad += !(std::fabs(got[h * D + e] - o[e]) <= tol);
    }
    CHECK(bad == 0);
    f.kv_dtype = 7;
    CHECK_CODE(hc->decode_attention_ex(d, f), ErrorCode::InvalidArgument);
    CHECK_CODE(hc->attention_ex(a, f), ErrorCode::InvalidArgument);
    for (HipBuffer* b : {dk, dv, dq, kc, vc, ks, vs, dt, dl, rq, out, lse, ws}) hc->release_buffer(b);
}

int main(int argc, char** argv) {
    if (!get_hip_compute()) {
        std::printf("no usable gfx950 GPU\n");
        return 77;
    }
    return hosttest::run_all(argc, argv);
}
