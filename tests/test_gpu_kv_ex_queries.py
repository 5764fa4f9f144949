"""Float queries of magnitudes from 1e-31 to 1e31, with K scales and the call's factor the other way, on every kernel, against
float64 with bounds that go with what each result is made of."""
import numpy as np
import pytest

from granite_amd import F16, F32, F8E4M3
from gpu_util import say
from kv_ex_calls import RUNS, STEPS, check_run, check_step, decode, run_cache, step_cache

pytestmark = pytest.mark.gpu


def spread_queries(rng, shape, factor):
    """Rows of one magnitude each, a thousand times apart from row to row, and elements of a row up to 2^12 apart."""
    q = rng.standard_normal(shape) * 2.0 ** rng.integers(-12, 1, shape[-1])
    return q * factor * 10.0 ** rng.uniform(-1.5, 1.5, shape[:-1] + (1,))


def rescaled(cache, shift):
    """The cache's K scales moved the other way, as far as the scales' range goes; what is left for the call's scale."""
    if cache.kv != F8E4M3:
        return 1.0
    e = int(np.clip(shift, -80, 80))
    cache.ks *= np.float32(2.0 ** -e)
    return 2.0 ** e


@pytest.mark.parametrize("power", [-100, -30, -14, 17, 40, 100])
@pytest.mark.parametrize("name", STEPS)
def test_float_queries_of_a_step(gpu, name, power):
    say(f"{name} 2^{power}")
    cache, shape, window, some = step_cache(name)
    q = spread_queries(np.random.default_rng(2), shape, 2.0 ** power).astype(np.float32)
    left = rescaled(cache, power)
    scale = shape[-1] ** -0.5 * 0.05 * left * 2.0 ** -power
    check_step(gpu, cache.upload(), q, window, some, float(scale), f"{name} 2^{power}")


@pytest.mark.parametrize("power", [-100, -30, -14, 17, 40, 100])
@pytest.mark.parametrize("name", RUNS)
def test_float_queries_of_a_run(gpu, name, power):
    say(f"{name} 2^{power}")
    for out_dtype in (F32, F16):
        cache, shape, start, window, some, tiles = run_cache(name)
        q = spread_queries(np.random.default_rng(2), shape, 2.0 ** power).astype(np.float32)
        left = rescaled(cache, power)
        scale = shape[-1] ** -0.5 * 0.05 * left * 2.0 ** -power
        check_run(gpu, cache.upload(), q, start, window, some, tiles, out_dtype, float(scale), f"{name} 2^{power}")


@pytest.mark.parametrize("name", ["rows", "persistent 8-bit", "persistent half"])
def test_rows_of_zeros_infinities_and_nan(gpu, name):
    """A row of zeros sees every key alike; infinities and NaN stay in their row."""
    cache, shape, window, some = step_cache(name)
    q = np.random.default_rng(2).standard_normal(shape).astype(np.float32)
    q[0, 0] = 0.0
    q[0, 1, 5], q[0, 2, 6] = np.inf, np.nan
    got, lse = decode(gpu, cache.upload(), q, *window)
    clean = q.copy()
    clean[0, 1:3] = 0.0
    want, want_lse = check_step(gpu, cache, clean, window, some, what=name)
    rest = np.ones(shape[:2], bool)
    rest[0, 1:3] = False
    assert np.array_equal(got[rest], want[rest]) and np.array_equal(lse[rest], want_lse[rest])
    assert np.isnan(got[0, 2]).all()


@pytest.mark.parametrize("name", ["rows", "persistent", "tiles", "tiles half"])
def test_products_of_zero_under_any_factor(gpu, name):
    """Keys of zeros have scores of zero, also where the K scale times the query's power is beyond a float."""
    cache, shape, start, window, some, tiles = run_cache(name)
    cache.k[:] = 0
    if cache.kv == F8E4M3:
        cache.ks[:] = 2.0 ** 119
    q = (np.random.default_rng(2).standard_normal(shape) * 1e37).astype(np.float32)
    check_run(gpu, cache.upload(), q, start, window, some, tiles, F32, 1.0, name)
