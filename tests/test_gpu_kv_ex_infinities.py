"""Infinities in V of a half cache seen through a window: whatever kernel a call goes to and however its keys are cut,
the rows that see one get it, and the other elements stay finite."""
import numpy as np
import pytest

import kv_ex_calls
from granite_amd import F16, F32
from gpu_util import dev
from test_gpu_kv_ex import Cache

pytestmark = pytest.mark.gpu


def with_infinities(rng, length, bs, hkv, d, at):
    """A half cache with +inf in V at (token, element) of KV head 0."""
    cache = Cache(rng, [length], bs, hkv, d, F16)
    for token, e in at:
        if bs:
            cache.v[cache.table[0, token // bs] * bs + token % bs, 0, e] = np.inf
        else:
            cache.v[0, token, e] = np.inf
    return cache.upload()


def check(got, positions, window, at, group, what):
    want = np.zeros(got.shape, bool)
    for token, e in at:
        sees = (token <= positions) & (token > positions - window)
        want[sees, :group, e] = True
    assert np.array_equal(np.isposinf(got), want), f"{what}: infinities at {np.argwhere(np.isposinf(got) != want)[0]}"
    assert np.isfinite(got[~want]).all(), f"{what}: not finite at {np.argwhere(~np.isfinite(got) & ~want)[0]}"


@pytest.mark.parametrize("types", [(F16, F16), (F32, F32)])
@pytest.mark.parametrize("bs,n,hq,hkv,d", [(16, 300, 4, 1, 128), (0, 300, 4, 1, 64), (12, 300, 4, 1, 128), (16, 3, 4, 2, 64), (20, 17, 4, 1, 128)])
def test_scores_far_apart(gpu, types, bs, n, hq, hkv, d):
    """Scores hundreds apart: where keys are cut, the piece that holds the infinity has a weight of zero."""
    length, window = 6000, 5000
    at = [(1100, 3), (2900, 4), (4444, 5), (length - n, 6)]
    cache = with_infinities(np.random.default_rng(n), length, bs, hkv, d, at)
    q = np.random.default_rng(n + 1).standard_normal((n, hq, d)).astype(np.float16 if types[0] == F16 else np.float32)
    got, lse = kv_ex_calls.prefill(gpu, cache, q, length - n, types[1], window, scale=100.0)
    check(got, length - n + np.arange(n), window, at, hq // hkv, f"bs={bs} n={n}")
    assert np.isfinite(lse).all()


@pytest.mark.parametrize("bs,batch,hq,hkv,d", [(16, 1, 4, 2, 128), (20, 1, 4, 2, 64), (16, 24, 16, 16, 64)])
def test_scale_pointers_of_a_half_cache_mean_nothing(gpu, bs, batch, hq, hkv, d):
    """The same form structure for both kinds of cache: k_scale and v_scale left set with kv_dtype F16."""
    lens = [3000] * batch
    cache = Cache(np.random.default_rng(3), lens, bs, hkv, d, F16)
    for token, e in ((2999, 3), (2940, 4), (1200, 5)):
        cache.v[cache.table[0, token // bs] * bs + token % bs, 0, e] = np.inf
    cache.upload()
    q = np.random.default_rng(4).standard_normal((batch, hq, d)).astype(np.float16)
    scales = dev(np.full((cache.num_blocks, hkv), np.nan, np.float32))
    plain, plain_lse = kv_ex_calls.decode(gpu, cache, q, 2500, 4)
    got, lse = kv_ex_calls.decode(gpu, cache, q, 2500, 4, k_scale=scales, v_scale=scales)
    assert np.isposinf(plain[0, :hq // hkv, 3:6]).all() and np.isfinite(np.delete(plain[0], (3, 4, 5), -1)).all()
    assert np.array_equal(got, plain) and np.array_equal(lse, plain_lse)
    rows = kv_ex_calls.prefill(gpu, cache, np.repeat(q[:1], 5, 0), 2995, F32, 2500, 4)[0]
    same = kv_ex_calls.prefill(gpu, cache, np.repeat(q[:1], 5, 0), 2995, F32, 2500, 4, k_scale=scales, v_scale=scales)[0]
    assert np.array_equal(rows, same)


@pytest.mark.parametrize("bs,n,hq,hkv,d", [(16, 1, 4, 2, 128), (20, 5, 4, 2, 64), (16, 420, 96, 1, 64), (0, 300, 32, 1, 128)])
def test_infinite_keys_under_half_queries(gpu, bs, n, hq, hkv, d):
    """A key whose score is minus infinity has no weight; with a score of plus infinity a row is NaN."""
    length, window, token = 700 + n, 600, 690
    cache = Cache(np.random.default_rng(n), [length], bs, hkv, d, F16)
    row = cache.table[0, token // bs] * bs + token % bs if bs else token
    cache.k[(row, 0, 7) if bs else (0, row, 7)] = -np.inf
    q = np.random.default_rng(n + 1).standard_normal((n, hq, d)).astype(np.float16)
    got, lse = kv_ex_calls.prefill(gpu, cache.upload(), q, length - n, F32, window)
    group = hq // hkv
    position = length - n + np.arange(n)[:, None]
    sees = (token <= position) & (token > position - window) & (np.arange(hq)[None] < group)
    assert sees.any()
    above = sees & (q[..., 7] < 0)
    assert np.array_equal(np.isnan(got).all(-1), above) and np.array_equal(np.isnan(got).any(-1), above) and np.array_equal(np.isnan(lse), above)
    # the others: as with a finite key of no weight there
    cache.k[(row, 0, 7) if bs else (0, row, 7)] = -60000.0
    inf, inf_lse = got[sees & ~above], lse[sees & ~above]
    got, lse = kv_ex_calls.prefill(gpu, cache.upload(), q, length - n, F32, window)
    with_weight = sees & ~above & (q[..., 7] > 0.02)  # -60000 * 0.02 / sqrt(d): more than 100 below the other scores
    pick = with_weight[sees & ~above]
    np.testing.assert_allclose(inf[pick], got[with_weight], rtol=0, atol=1e-6)
    np.testing.assert_allclose(inf_lse[pick], lse[with_weight], rtol=0, atol=1e-6)
