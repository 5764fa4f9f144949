"""Infinities in V of a half cache seen through a window: whatever kernel a call goes to and however its keys are cut,
the rows that see one get it, and the other elements stay finite."""
import numpy as np
import pytest

import kv_ex_calls
from granite_amd import F16, F32
from gpu_util import dev
from test_gpu_kv_ex import Cache

pytestmark = pytest.mark.gpu


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
