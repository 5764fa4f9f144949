"""V and K scales of 8-bit pools: blocks whose scales are up to 2^100 apart, each of them counting for what it is, against
float64 with bounds that go with what each result is made of, sum(p |v|)."""
import numpy as np
import pytest

import kv8
from granite_amd import F16, F32, F8E4M3
from kv_ex_calls import RUNS, STEPS, check_run, check_step, run_cache, step_cache
from test_gpu_kv_ex import Cache

pytestmark = pytest.mark.gpu


def far_block(cache, table, block, power, score):
    """Block `block` of a sequence gets V scales 2^power times larger and keys whose first element, with queries whose first
    element is 16, makes its scores `score` (natural log) for all heads, others keeping theirs small."""
    b = int(table[block])
    d = cache.d
    codes = np.zeros((cache.bs, cache.hkv, d), np.uint8)
    x = score / (16.0 * d ** -0.5)
    s = kv8.scale_for(abs(x))
    codes[:, :, 0] = kv8.encode8(x / s)
    cache.k[b * cache.bs:(b + 1) * cache.bs] = codes
    cache.ks[b] = s
    cache.vs[b] *= np.float32(2.0 ** power)
    # (whole blocks only: what lies behind a sequence's end is NaN)
    assert not np.isnan(kv8.decode8(cache.v[b * cache.bs:(b + 1) * cache.bs])).any()


def queries(rng, shape, dtype):
    q = rng.standard_normal(shape)
    q[..., 0] = 16.0
    return q.astype(dtype)


def first_element(cache, x):
    """K's first element everywhere `x`, where a block is used."""
    for b in range(cache.num_blocks):
        for h in range(cache.hkv):
            if np.isfinite(cache.ks[b, h]):
                rows = cache.k[b * cache.bs:(b + 1) * cache.bs, h]
                rows[~np.isnan(kv8.decode8(rows[:, 0])), 0] = kv8.encode8(x / cache.ks[b, h])


@pytest.mark.parametrize("power,score", [(24, -60), (40, -80), (100, -140), (-40, 0), (-80, 0)])
@pytest.mark.parametrize("name", [n for n in STEPS if STEPS[n][0] == F8E4M3])
def test_one_block_of_another_scale_in_a_step(gpu, name, power, score):
    """A visible block whose V scale is 2^power times the others' and whose probability is next to nothing."""
    for q_dtype in (np.float16, np.float32):
        cache, shape, window, some = step_cache(name)
        first_element(cache, 0.0)
        for seq in range(len(cache.lens)):
            if cache.lens[seq] > 1000:
                far_block(cache, cache.table[seq], 3, power, score)
                far_block(cache, cache.table[seq], cache.lens[seq] // cache.bs - 2, power, score)
            elif cache.lens[seq] > 500:
                far_block(cache, cache.table[seq], 7, power, score)
        check_step(gpu, cache.upload(), queries(np.random.default_rng(2), shape, q_dtype), window, some, what=f"{name} 2^{power}")


@pytest.mark.parametrize("power,score", [(24, -60), (40, -80), (100, -140), (-40, 0), (-80, 0)])
@pytest.mark.parametrize("name", [n for n in RUNS if RUNS[n][0] == F8E4M3])
def test_one_block_of_another_scale_in_a_run(gpu, name, power, score):
    for q_dtype, out_dtype in ((np.float16, F32), (np.float32, F32), (np.float16, F16)):
        cache, shape, start, window, some, tiles = run_cache(name)
        first_element(cache, 0.0)
        far_block(cache, cache.table[0], (start + 8) // cache.bs - (2 if window[0] else 10), power, score)
        check_run(gpu, cache.upload(), queries(np.random.default_rng(2), shape, q_dtype), start, window, some, tiles, out_dtype, what=f"{name} 2^{power}")


@pytest.mark.parametrize("name", ["rows", "rows any block", "persistent"])
def test_a_later_tokens_scale_does_not_count(gpu, name):
    """The V scale of the last token's block, 2^60 above the others', is nothing to the queries in front of it."""
    kv, bs, hq, hkv, d, n, start, window, some, tiles = RUNS[name]
    total = -(-(start + n) // bs) * bs + 1  # the last token starts a block
    cache = Cache(np.random.default_rng(5), [total], bs, hkv, d, kv)
    cache.vs[cache.table[0, total // bs]] *= np.float32(2.0 ** 60)
    q = np.random.default_rng(6).standard_normal((n, hq, d)).astype(np.float32)
    check_run(gpu, cache.upload(), q, total - n, window, range(n - 1), tiles, F32, what=name)


@pytest.mark.parametrize("other", [20, 60, 110])
@pytest.mark.parametrize("name", [n for n in RUNS if RUNS[n][0] == F8E4M3])
def test_blocks_of_zeros_keep_their_weight(gpu, name, other):
    """Every other block's V is zero (its scale 2^-96, as the append leaves it), the rest have scales of 2^other: the zeros
    count in the sums as any value does."""
    cache, shape, start, window, some, tiles = run_cache(name)
    cache.vs[:] = 2.0 ** other / 64
    for block in range(0, -(-cache.lens[0] // cache.bs), 2):
        b = cache.table[0, block]
        cache.v[b * cache.bs:(b + 1) * cache.bs] = 0
        cache.vs[b] = 2.0 ** -96
    cache.upload()
    for q_dtype in (np.float16, np.float32):
        q = np.random.default_rng(2).standard_normal(shape).astype(q_dtype)
        check_run(gpu, cache, q, start, window, some, tiles, F32, what=f"{name} 2^{other}")


@pytest.mark.parametrize("name", [n for n in STEPS if STEPS[n][0] == F8E4M3])
def test_both_ends_of_the_scales(gpu, name):
    for ks, vs, scale in ((2.0 ** -96, 2.0 ** -96, 2.0 ** 90), (2.0 ** 112, 2.0 ** 112, 2.0 ** -118)):
        cache, shape, window, some = step_cache(name)
        cache.ks[:], cache.vs[:] = ks, vs
        q = np.random.default_rng(2).standard_normal(shape).astype(np.float16)
        check_step(gpu, cache.upload(), q, window, some, scale, f"{name} {ks}")


@pytest.mark.parametrize("name", [n for n in RUNS if RUNS[n][0] == F8E4M3])
def test_both_ends_of_the_scales_in_a_run(gpu, name):
    for ks, vs, scale in ((2.0 ** -96, 2.0 ** -96, 2.0 ** 90), (2.0 ** 112, 2.0 ** 112, 2.0 ** -118)):
        for q_dtype in (np.float16, np.float32):
            cache, shape, start, window, some, tiles = run_cache(name)
            cache.ks[:], cache.vs[:] = ks, vs
            q = np.random.default_rng(2).standard_normal(shape).astype(q_dtype)
            check_run(gpu, cache.upload(), q, start, window, some, tiles, F32, scale, f"{name} {ks}")


@pytest.mark.parametrize("bs,hq,hkv,d", [(16, 48, 3, 64), (20, 48, 1, 128), (8, 64, 4, 64), (1, 40, 8, 64), (48, 64, 2, 128)])
def test_scales_of_any_value_in_a_step(gpu, bs, hq, hkv, d):
    """Few keys a row, so that a single probability that is off shows."""
    for q_dtype in (np.float16, np.float32):
        cache = Cache(np.random.default_rng(hq), [*range(1, 25), 40, 80], bs, hkv, d, F8E4M3, scales="any", spread=3.0).upload()
        q = np.random.default_rng(2).standard_normal((26, hq, d)).astype(q_dtype)
        check_step(gpu, cache, q, (0, 0), range(26), what=f"bs={bs} {q_dtype.__name__}")


@pytest.mark.parametrize("name", [n for n in STEPS if STEPS[n][0] == F8E4M3])
def test_scales_of_any_value_behind_long_contexts(gpu, name):
    cache, shape, window, some = step_cache(name)
    cache.vs *= np.random.default_rng(3).uniform(1, 1.9, cache.vs.shape).astype(np.float32)
    cache.ks *= np.random.default_rng(4).uniform(1, 1.9, cache.ks.shape).astype(np.float32)
    q = (np.random.default_rng(2).standard_normal(shape) * 12).astype(np.float16)  # a few keys carry each row
    check_step(gpu, cache.upload(), q, window, some, what=name)


@pytest.mark.parametrize("n,start,bs,hq,hkv,d,tiles", [(30, 5, 32, 64, 2, 64, False), (60, 11, 5, 34, 2, 64, False), (12, 19, 16, 64, 2, 128, False),
                                                       (420, 0, 16, 96, 1, 64, True), (420, 3, 20, 96, 1, 128, True)])
def test_scales_of_any_value_in_a_run(gpu, n, start, bs, hq, hkv, d, tiles):
    for q_dtype in (np.float16, np.float32):
        cache = Cache(np.random.default_rng(hq), [start + n], bs, hkv, d, F8E4M3, scales="any", spread=3.0).upload()
        q = np.random.default_rng(2).standard_normal((n, hq, d)).astype(q_dtype)
        check_run(gpu, cache, q, start, (0, 0), range(0, min(n, 60), 2), tiles, F32, what=f"n={n} {q_dtype.__name__}")


@pytest.mark.parametrize("name", [n for n in RUNS if RUNS[n][0] == F8E4M3])
def test_scales_all_over_the_range_in_a_run(gpu, name):
    """Every block's V scale anywhere from 2^-88 to 2^95, so that the largest come late for some rows and early for others."""
    for seed, q_dtype in ((1, np.float16), (2, np.float32), (3, np.float16)):
        cache, shape, start, window, some, tiles = run_cache(name)
        rng = np.random.default_rng(seed)
        cache.vs = (cache.vs * 2.0 ** rng.integers(-80, 100, cache.vs.shape)).astype(np.float32)
        q = (rng.standard_normal(shape) * rng.choice([0.3, 3.0])).astype(q_dtype)
        check_run(gpu, cache.upload(), q, start, window, some, tiles, F32, what=f"{name} {seed}")


@pytest.mark.parametrize("name", [n for n in STEPS if STEPS[n][0] == F8E4M3])
def test_scales_all_over_the_range_in_a_step(gpu, name):
    for seed, q_dtype in ((1, np.float16), (2, np.float32)):
        cache, shape, window, some = step_cache(name)
        rng = np.random.default_rng(seed)
        cache.vs = (cache.vs * 2.0 ** rng.integers(-80, 100, cache.vs.shape)).astype(np.float32)
        q = (rng.standard_normal(shape) * rng.choice([0.3, 3.0])).astype(q_dtype)
        check_step(gpu, cache.upload(), q, window, some, what=f"{name} {seed}")
