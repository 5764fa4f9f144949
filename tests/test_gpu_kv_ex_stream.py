"""granite_hip_decode_attention_ex on steps big enough that a fixed number of waves shares them (dozens of sequences of
thousands of tokens), against kv8.attend (float64) for some of the sequences: windows, pages, scales, garbage."""
import numpy as np
import pytest

import kv8
from granite_amd import F16, F32, F8E4M3, MASK_CAUSAL
from gpu_util import dev, say
from test_gpu_kv_ex import NAN8, Cache, Captured, check, v_top

pytestmark = pytest.mark.gpu


def run(gpu, cache, hq, q_dtype, window=0, sinks=0, some=None, what="", scale=None):
    b, d, lens = len(cache.lens), cache.d, np.asarray(cache.lens, np.int32)
    scale = d ** -0.5 if scale is None else scale
    q = np.random.default_rng(b).standard_normal((b, hq, d), dtype=np.float32).astype(np.float16 if q_dtype == F16 else np.float32)
    out, lse = dev(np.full((b, hq, d), 7.0, np.float32)), dev(np.full((b, hq), 7.0, np.float32))
    dq, dl = dev(q), dev(lens)
    gpu.decode_attention_ex(q=dq, q_dtype=q_dtype, out=out, lse=lse, batch_size=b, num_heads=hq, scale=scale,
                            block_tables=cache.dev[4], seq_lens=dl, max_blocks_per_seq=cache.max_blocks, window=window,
                            num_sinks=sinks, **cache.kwargs())
    gpu.sync()
    got, got_lse = out.read(np.float32, (b, hq, d)), lse.read(np.float32, (b, hq))
    for i in (range(b) if some is None else some):
        n = int(lens[i])
        if n <= 0:
            assert (got[i] == 7.0).all() and (got_lse[i] == 7.0).all(), f"{what}: an empty sequence was written"
            continue
        (k, v), valid = cache.rows(i, n)
        vis = kv8.visible([n - 1], n, window, sinks, valid)
        o, l, ds = kv8.attend(q[i:i + 1], k, v, vis, scale)
        check(got[i:i + 1], got_lse[i:i + 1], o, l, ds, v_top(v, vis), int(vis.sum()), False, f"{what} seq {i} len {n}")
    return got, got_lse


def lens_of(rng, batch, top):
    lens = rng.integers(1, top + 1, batch)
    lens[:8] = [0, 1, 31, 32, 33, top, 0, top - 1]
    return [int(x) for x in lens]


@pytest.mark.parametrize("hq,hkv,d,batch,top", [(32, 8, 128, 24, 2900), (16, 16, 64, 24, 2900), (28, 4, 128, 40, 2900), (48, 1, 64, 60, 4000),
                                                (40, 5, 128, 30, 2900), (34, 2, 128, 40, 4000)])
@pytest.mark.parametrize("q_dtype", [F16, F32])
def test_8bit(gpu, hq, hkv, d, batch, top, q_dtype):
    say(f"stream 8-bit hq={hq} hkv={hkv} d={d}")
    cache = Cache(np.random.default_rng(d + hq), lens_of(np.random.default_rng(hq), batch, top), 32 if d == 64 else 64, hkv, d, F8E4M3).upload()
    run(gpu, cache, hq, q_dtype, some=(0, 1, 2, 3, 4, 5, 6, 7, 11, batch - 1))
    run(gpu, cache, hq, q_dtype, 2500, 37, some=(0, 1, 4, 5, 6, 7, 13, batch - 1))


@pytest.mark.parametrize("bs", [0, 16, 48])
@pytest.mark.parametrize("window,sinks", [(4000, 0), (2600, 37), (3001, 100), (2000, 2000)])
def test_half_windows(gpu, bs, window, sinks):
    say(f"stream half window={window} sinks={sinks} bs={bs}")
    for hq, hkv, d, q in ((16, 8, 128, F16), (24, 24, 64, F32)):
        if bs:
            lens = lens_of(np.random.default_rng(window), 16, 4000)
        else:
            lens, hq, hkv, window = [16000], hq * 2, hkv * 2, window * 4 - 1001
        cache = Cache(np.random.default_rng(d), lens, bs, hkv, d, F16).upload()
        run(gpu, cache, hq, q, window, sinks, some=None if not bs else (0, 1, 2, 3, 4, 5, 6, 7, 15))


def test_released_and_invalid_pages(gpu):
    rng = np.random.default_rng(4)
    lens = lens_of(rng, 24, 3000)
    for kv in (F8E4M3, F16):
        cache = Cache(np.random.default_rng(5), lens, 16, 16, 64 if kv == F16 else 128, kv)
        for i, n in enumerate(lens):
            for j in range(-(-n // 16)):
                if j > 0 and 16 * (j + 1) <= n - 2000:
                    cache.table[i, j] = rng.choice([-1, cache.num_blocks, 2147483647, -2147483648])
                elif rng.random() < 0.05 and n > 100:
                    cache.table[i, j] = -1
        cache.table[9] = -1
        cache.upload()
        got, lse = run(gpu, cache, 16, F16, 2000, 4, some=(5, 6, 7, 9, 10, 11), what="released")
        assert (got[9] == 0).all() and np.isneginf(lse[9]).all()
        if kv == F8E4M3:
            run(gpu, cache, 16, F32, some=(5, 7, 10, 12), what="invalid pages")


def test_scales_and_factors(gpu):
    lens = lens_of(np.random.default_rng(6), 24, 2500)
    for scales, spread in (("any", 1.0), ("pow2", 1000.0), ("any", 1000.0)):
        cache = Cache(np.random.default_rng(9), lens, 16, 16, 64, F8E4M3, spread=spread, scales=scales).upload()
        run(gpu, cache, 16, F16, some=(1, 4, 5, 9), what=f"scales {scales} {spread}")
    for scale in (100.0, -100.0, 0.0):
        run(gpu, cache, 16, F32, some=(5, 7), scale=scale, what=f"factor {scale}")


def test_nan_and_infinities(gpu):
    """They reach what sees them, and nothing else."""
    lens = [3000] * 24
    cache = Cache(np.random.default_rng(11), lens, 16, 16, 64, F8E4M3)
    at = lambda c, i, t: c.table[i, t // 16] * 16 + t % 16  # noqa: E731
    cache.v[at(cache, 3, 2990), 1, 7] = NAN8
    cache.v[at(cache, 4, 100), 1, 7] = NAN8       # behind the window
    got, _ = run(gpu, cache.upload(), 16, F16, 2500, 4, some=(2, 3, 4, 5))
    assert np.isnan(got[3, 1, 7]) and np.isnan(got).sum() == 1
    half = Cache(np.random.default_rng(12), lens, 16, 16, 64, F16)
    half.v[at(half, 3, 2990), 1, 7] = np.inf
    half.v[at(half, 3, 2991), 2, 7], half.v[at(half, 3, 1500), 2, 7] = np.inf, -np.inf
    half.v[at(half, 4, 100), 1, 7] = np.nan
    half.k[at(half, 4, 101), 1, 7] = np.inf
    got, _ = run(gpu, half.upload(), 16, F16, 2500, 4, some=(2, 3, 4, 5))
    assert np.isposinf(got[3, 1, 7]) and np.isnan(got[3, 2, 7]) and (~np.isfinite(got)).sum() == 2


def test_captured_launches_of_every_kernel(gpu):
    """The persistent kernels with their merges, and the tiles kernel with keys cut, each in a graph with a workspace of its
    own: replays with other queries and lengths, in turn and with eager calls between them, equal the eager calls."""
    rng = np.random.default_rng(30)
    graphs, jobs = [], []
    for kv, hq, hkv, d, window in ((F8E4M3, 16, 16, 64, 0), (F16, 24, 24, 64, 2600)):
        cache = Cache(rng, [2900] * 24, 48, hkv, d, kv).upload()
        q, out, lse, n = (dev(np.zeros((24, hq, d), np.float16)), dev(np.zeros((24, hq, d), np.float32)), dev(np.zeros((24, hq), np.float32)),
                          dev(np.full(24, 2900, np.int32)))
        kw = dict(q=q, q_dtype=F16, out=out, lse=lse, batch_size=24, num_heads=hq, scale=0.1, block_tables=cache.dev[4], seq_lens=n,
                  max_blocks_per_seq=cache.max_blocks, window=window, num_sinks=3, **cache.kwargs())
        jobs.append((gpu.decode_attention_ex, kw, q, out, lse, n, cache))
    cache = Cache(rng, [4000], 20, 2, 64, F8E4M3).upload()
    q, out, lse = dev(np.zeros((300, 96, 64), np.float16)), dev(np.zeros((300, 96, 64), np.float16)), dev(np.zeros((96, 300), np.float32))
    kw = dict(q=q, q_dtype=F16, q_tok_stride=96 * 64, q_head_stride=64, out=out, out_dtype=F16, out_tok_stride=96 * 64, out_head_stride=64,
              seq_q=300, num_heads=96, scale=0.1, cache_len=4000, block_table=cache.dev[4], mask_mode=MASK_CAUSAL, start_pos=3700, lse=lse,
              **cache.kwargs())
    jobs.append((gpu.attention_ex, kw, q, out, lse, None, cache))
    for call, kw, q, out, lse, n, _ in jobs:
        need = call(**kw, query_workspace=True)
        assert need > 0
        kw["workspace"] = dev(np.zeros(need, np.uint8))
        graphs.append(Captured(gpu, lambda call=call, kw=kw: call(**kw)))
    for i in range(4):
        for _, _, q, out, lse, n, _ in jobs:
            q.write(rng.standard_normal(q.nbytes // 2).astype(np.float16))
            out.fill(0)
            lse.fill(0)
            if n is not None:
                n.write(rng.integers(1, 2901, 24).astype(np.int32))
        for g in graphs:
            g.replay()
        replayed = [(out.read(np.uint8, out.nbytes), lse.read(np.uint8, lse.nbytes)) for _, _, _, out, lse, _, _ in jobs]
        for (call, kw, _, out, lse, _, _), got in zip(jobs, replayed):
            out.fill(0)
            lse.fill(0)
            call(**kw)
            gpu.sync()
            assert np.array_equal(got[0], out.read(np.uint8, out.nbytes)) and np.array_equal(got[1], lse.read(np.uint8, lse.nbytes)), f"replay {i}"
            assert got[0].any()
    for g in graphs:
        g.close()
