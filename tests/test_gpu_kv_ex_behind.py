"""Queries all of whose windows lie behind the cache: zeros and a log-sum-exp of minus infinity, from every kernel.  The
lengths are multiples of the kernels' tiles, so that there is no key tile to visit at all; granite_amd/host/tests/kv_behind_test.cpp
checks which kernel the calls go to."""
import numpy as np
import pytest

import kv_ex_calls
from granite_amd import F16, F32, F8E4M3
from test_gpu_kv_ex import Cache

pytestmark = pytest.mark.gpu


# queries, first position, cached tokens, window, heads, KV heads, head size
CALLS = [(2, 2048, 1024, 1024, 32, 8, 128), (2, 2048, 1024, 1024, 32, 8, 64), (4, 5000, 2048, 2048, 16, 8, 128), (1, 3140, 2080, 1000, 16, 16, 64),
         (1, 128, 64, 20, 4, 2, 128), (400, 2000, 1024, 700, 32, 1, 64)]


@pytest.mark.parametrize("types", [(F16, F16), (F32, F32), (F16, F32)])
@pytest.mark.parametrize("n,start,length,window,hq,hkv,d", CALLS)
def test_windows_behind_the_cache(gpu, n, start, length, window, hq, hkv, d, types):
    q_dtype, out_dtype = types
    cache = Cache(np.random.default_rng(n), [length], 16, hkv, d, F8E4M3).upload()
    q = np.random.default_rng(1).standard_normal((n, hq, d)).astype(np.float16 if q_dtype == F16 else np.float32)
    for _ in range(2):
        got, lse = kv_ex_calls.prefill(gpu, cache, q, start, out_dtype, window)
        assert (got == 0).all() and np.isneginf(lse).all()
    # sinks are seen from anywhere
    got, lse = kv_ex_calls.prefill(gpu, cache, q[:2], start, out_dtype, window, sinks=3)
    kv_ex_calls.compare(got, lse, kv_ex_calls.reference(cache, 0, q[:2], start + np.arange(len(q[:2])), window, 3, None, half=out_dtype == F16), "sinks")
