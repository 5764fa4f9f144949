"""Scores of any finite size: rows all of whose scores are below -1e31, which is where a running maximum might start."""
import numpy as np
import pytest

import kv8
from granite_amd import F16, F32, F8E4M3
from kv_ex_calls import RUNS, STEPS, decode, prefill, run_cache, step_cache

pytestmark = pytest.mark.gpu


def negative_scores(cache):
    """K's first elements become -2 and less, so that with queries (1, 0, 0 ...) they are the scores."""
    if cache.kv == F8E4M3:
        k = kv8.decode8(cache.k)
        k[..., 0] = np.where(np.isnan(k[..., 0]), np.nan, -2.0 - np.abs(k[..., 0]))
        cache.k, cache.ks[:] = kv8.encode8(k), 1.0
    else:
        cache.k[..., 0] = -2.0 - np.abs(cache.k[..., 0])
    return cache.upload()


def check(cache, seq, got, lse, position, window, scale, half, what):
    """The values of the keys with the least negative score, averaged."""
    length, group = cache.lens[seq], got.shape[0] // cache.hkv
    (k, v), valid = cache.rows(seq, length)
    vis = kv8.visible([position], length, *window, valid)[0]
    for h in range(got.shape[0]):
        x = np.where(vis, k[:, h // group, 0], -np.inf)
        top = v[x == x.max(), h // group]
        np.testing.assert_allclose(lse[h], x.max() * scale, rtol=2.0 ** -20)
        # one rounding of a probability (2^-22; 2^-11 in half results of the tiles kernel) and one of the result
        tol = (2.0 ** -10 if half else 2.0 ** -18) * np.abs(top).max() + (2.0 ** -25 if half else 0)
        np.testing.assert_allclose(got[h], top.mean(0), rtol=0, atol=tol, err_msg=f"{what} position {position} head {h}")


@pytest.mark.parametrize("scale", [1e7, 1e9, 1e31, -1e31])
@pytest.mark.parametrize("name", STEPS)
def test_scores_far_below_zero_in_a_step(gpu, name, scale):
    cache, shape, window, some = step_cache(name)
    q = np.zeros(shape, np.float32)
    q[..., 0] = np.sign(scale)
    got, lse = decode(gpu, negative_scores(cache), q, *window, scale=scale)
    for i in some:
        check(cache, i, got[i], lse[i], cache.lens[i] - 1, window, abs(scale), False, name)


@pytest.mark.parametrize("scale", [1e7, 1e9, 1e31, -1e31])
@pytest.mark.parametrize("name", RUNS)
def test_scores_far_below_zero_in_a_run(gpu, name, scale):
    for q_dtype, out_dtype in ((np.float32, F32), (np.float16, F16), (np.float16, F32)):
        cache, shape, start, window, some, tiles = run_cache(name)
        q = np.zeros(shape, q_dtype)
        q[..., 0] = np.sign(scale)
        got, lse = prefill(gpu, negative_scores(cache), q, start, out_dtype, *window, scale=scale)
        for i in some:
            check(cache, 0, np.asarray(got[i], np.float64), lse[i], start + i, window, abs(scale), out_dtype == F16, name)


@pytest.mark.parametrize("name", RUNS)
def test_scores_far_above_zero_in_a_run(gpu, name):
    cache, shape, start, window, some, tiles = run_cache(name)
    q = np.zeros(shape, np.float16)
    q[..., 0] = -1.0  # the largest |element| has the largest score
    negative_scores(cache)
    got, lse = prefill(gpu, cache, q, start, F32, *window, scale=1e30)
    (k, v), valid = cache.rows(0, cache.lens[0])
    for i in some:
        vis = kv8.visible([start + i], cache.lens[0], *window, valid)[0]
        for h in range(shape[1]):
            kvh = h // (shape[1] // cache.hkv)
            x = np.where(vis, -k[:, kvh, 0], -np.inf)
            top = v[x == x.max(), kvh]
            np.testing.assert_allclose(lse[i, h], x.max() * 1e30, rtol=2.0 ** -20)
            np.testing.assert_allclose(got[i, h], top.mean(0), rtol=0, atol=2.0 ** -18 * np.abs(top).max(), err_msg=f"{name} query {i} head {h}")
