"""granite_hip_attention_ex with so many rows that they share tiles of keys (hundreds of queries of dozens of heads per KV
head), against kv8.attend (float64) for some of the queries and heads: windows and sinks, block sizes, garbage, scales."""
import numpy as np
import pytest

import kv8
from granite_amd import F16, F32, F8E4M3, MASK_CAUSAL, MASK_NONE
from gpu_util import dev, say
from test_gpu_kv_ex import NAN8, Cache, check, v_top

pytestmark = pytest.mark.gpu
TYPES = [(F16, F16), (F32, F32), (F16, F32), (F32, F16)]


def run(gpu, cache, n, start, hq, q_dtype, out_dtype, window=0, sinks=0, cache_len=None, mask=MASK_CAUSAL, what="", scale=None, must=()):
    """`must`: queries that are looked at in any case."""
    d = cache.d
    scale = d ** -0.5 if scale is None else scale
    length = cache.lens[0] if cache_len is None else cache_len
    rng = np.random.default_rng(n)
    q = rng.standard_normal((n, hq, d), dtype=np.float32).astype(np.float16 if q_dtype == F16 else np.float32)
    odt = np.float16 if out_dtype == F16 else np.float32
    out, lse, dq = dev(np.full(q.shape, 7.0, odt)), dev(np.full((hq, n), 7.0, np.float32)), dev(q)
    gpu.attention_ex(q=dq, q_dtype=q_dtype, q_tok_stride=hq * d, q_head_stride=d, out=out, out_dtype=out_dtype,
                     out_tok_stride=hq * d, out_head_stride=d, seq_q=n, num_heads=hq, scale=scale, cache_len=length,
                     block_table=cache.dev[4], mask_mode=mask, start_pos=start, lse=lse, window=window, num_sinks=sinks,
                     **cache.kwargs())
    gpu.sync()
    got, got_lse = out.read(odt, q.shape), lse.read(np.float32, (hq, n)).T
    (k, v), valid = cache.rows(0, length)
    group = hq // cache.hkv
    some = np.unique([0, 1, n // 2, n - 2, n - 1, *must, *rng.integers(0, n, 70)])
    vis = kv8.visible(start + some, length, window, sinks, valid, mask == MASK_CAUSAL)
    for kvh in range(cache.hkv):
        heads = [kvh * group, kvh * group + group // 3, kvh * group + group - 1]
        o, l, ds = kv8.attend(q[np.ix_(some, heads)], k[:, kvh:kvh + 1], v[:, kvh:kvh + 1], vis, scale)
        check(got[np.ix_(some, heads)], got_lse[np.ix_(some, heads)], o, l, ds, v_top(v[:, kvh], vis), int(vis.sum(1).max()),
              out_dtype == F16, f"{what} KV head {kvh}")
    return got, got_lse


@pytest.mark.parametrize("kv,bs", [(F8E4M3, 16), (F8E4M3, 20), (F8E4M3, 8), (F16, 16), (F16, 0), (F16, 12)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 2), (64, 0), (100, 4), (130, 70), (256, 300), (4000, 4)])
def test_windows(gpu, kv, bs, window, sinks):
    say(f"tiles window={window} sinks={sinks} kv={kv} bs={bs}")
    for i, (n, start, hq, hkv) in enumerate(((400, 700, 96, 1), (611, 0, 96, 2))):
        types = TYPES[(window + i) % 4]
        cache = Cache(np.random.default_rng(n), [start + n], bs, hkv, 64 if (window + bs // 4) % 2 == i else 128, kv).upload()
        run(gpu, cache, n, start, hq, *types, window, sinks, what=f"n={n} d={cache.d} types={types}")


@pytest.mark.parametrize("bs", [4, 8, 16, 20, 48])
@pytest.mark.parametrize("types", TYPES)
def test_every_key(gpu, bs, types):
    say(f"tiles bs={bs} types={types}")
    for n, start, hq, hkv, d in ((400, 700, 96, 1, 128), (700, 0, 96, 2, 64), (513, 1130, 56, 1, 64)):
        run(gpu, Cache(np.random.default_rng(n), [start + n], bs, hkv, d, F8E4M3).upload(), n, start, hq, *types, what=f"n={n}")
    cache = Cache(np.random.default_rng(1), [1033], bs, 1, 64, F8E4M3).upload()
    run(gpu, cache, 450, 0, 96, *types, mask=MASK_NONE, what="no mask")


@pytest.mark.parametrize("types", TYPES[:2])
@pytest.mark.parametrize("bs", [16, 20])
def test_garbage_no_query_sees(gpu, types, bs):
    """NaN and infinities in keys that some queries see and others do not: they reach the former only."""
    n = 420
    cache = Cache(np.random.default_rng(2), [n + 300], bs, 2, 64, F16)
    at = lambda t: cache.table[0, t // bs] * bs + t % bs  # noqa: E731
    cache.v[at(300 + n // 2), 0, 3] = np.inf
    cache.v[at(300 + n // 2), 1, 4] = np.nan
    cache.v[at(300 + n // 3), 1, 5] = -np.inf
    cache.k[at(340), 1, :] = np.nan
    must = [n // 2 - 1, n // 2, n // 2 + 39, n // 2 + 40, n // 3, n // 3 + 39, n // 3 + 40, 39, 40, 79, 80]
    run(gpu, cache.upload(), n, 300, 96, *types, 40, 4, must=must)
    f8 = Cache(np.random.default_rng(2), [n + 300], bs, 2, 128, F8E4M3)
    f8.v[f8.table[0, (300 + n // 2) // bs] * bs + (300 + n // 2) % bs, 1, 9] = NAN8
    f8.vs[f8.table[0, 5]] = np.nan  # a block between the sinks and the first window
    f8.ks[f8.table[0, 6]] = np.inf
    run(gpu, f8.upload(), n, 300, 96, *types, 40, 4, must=must)
    f8.table[0, 2:8] = (-1, f8.num_blocks, 2147483647, -2147483648, -1, -1)
    f8.table[0, 30] = -1
    run(gpu, f8.upload(), n, 300, 96, *types, must=must)
    run(gpu, f8, n, 200, 96, *types, 300, 50, cache_len=200 + n, must=must)


@pytest.mark.parametrize("types", TYPES[:2])
def test_rows_that_see_nothing(gpu, types):
    """Queries beyond the cache whose window lies behind its end, pages that are all invalid."""
    for bs in (16, 20):
        cache = Cache(np.random.default_rng(1), [500], bs, 1, 128, F8E4M3).upload()
        got, lse = run(gpu, cache, 420, 400, 96, *types, 20, must=range(95, 125))
        assert (got[120:] == 0).all() and np.isneginf(lse[120:]).all()
        run(gpu, cache, 420, 400, 96, *types, 20, 3, must=range(95, 125))
        cache.table[:] = -1
        cache.upload()
        assert (run(gpu, cache, 500, 0, 96, *types)[0] == 0).all()


@pytest.mark.parametrize("bs", [16, 20])
@pytest.mark.parametrize("types", TYPES[:2])
def test_scales_and_factors(gpu, bs, types):
    for scales, spread in (("any", 1.0), ("pow2", 1000.0), ("any", 1000.0)):
        cache = Cache(np.random.default_rng(9), [900], bs, 1, 64, F8E4M3, spread=spread, scales=scales).upload()
        run(gpu, cache, 420, 480, 96, *types, what=f"scales {scales} {spread}")
    for scale in (20.0, -0.3, 0.0, 1e-30):
        for kv in (F8E4M3, F16):
            cache = Cache(np.random.default_rng(20), [900], bs, 1, 64, kv).upload()
            run(gpu, cache, 420, 480, 96, *types, 320, 3, scale=scale, what=f"scale {scale}")


@pytest.mark.parametrize("types", TYPES[:2])
@pytest.mark.parametrize("bs", [16, 12, 0])
def test_infinities_that_are_seen(gpu, types, bs):
    cache = Cache(np.random.default_rng(21), [1000], bs, 2, 64, F16)
    at = (lambda t: cache.table[0, t // bs] * bs + t % bs) if bs else (lambda t: t)
    n = 1000
    put = (lambda t, h, d, x: cache.v.__setitem__((at(t), h, d), x)) if bs else (lambda t, h, d, x: cache.v.__setitem__((h, t, d), x))
    put(n - 1, 0, 3, np.inf), put(n - 60, 0, 4, np.inf), put(n - 40, 1, 5, -np.inf), put(n - 41, 1, 6, np.inf), put(n - 42, 1, 6, -np.inf)
    run(gpu, cache.upload(), 420, n - 420, 96, *types, n - 7, 2, scale=0.02, must=range(350, 420))
