"""Windows and sinks up to what 32 bits hold, and calls whose kernels are estimated less than a microsecond apart."""
import numpy as np
import pytest

import kv_ex_calls
from granite_amd import F16, F32, F8E4M3
from gpu_util import dev
from test_gpu_kv_ex import Cache

pytestmark = pytest.mark.gpu
TOP = 0xFFFFFFFF


@pytest.mark.parametrize("window,sinks", [(100, TOP), (100, 1 << 31), (100, (1 << 31) - 1), (1, TOP - 15), (TOP, TOP), (1 << 31, 0), (TOP, 0), ((1 << 31) - 1, 1 << 31)])
@pytest.mark.parametrize("kv,bs,n,start,hq,hkv,d", [(F8E4M3, 16, 420, 480, 96, 1, 64), (F16, 0, 420, 480, 96, 1, 64), (F8E4M3, 20, 420, 480, 96, 1, 64),
                                                    (F8E4M3, 16, 5, 595, 8, 2, 128), (F16, 12, 5, 595, 8, 2, 128), (F8E4M3, 48, 3, 8100, 16, 2, 128)])
def test_windows_and_sinks_that_hide_nothing(gpu, kv, bs, n, start, hq, hkv, d, window, sinks):
    cache = Cache(np.random.default_rng(n), [start + n], bs, hkv, d, kv).upload()
    q = np.random.default_rng(1).standard_normal((n, hq, d)).astype(np.float16)
    some = np.unique([0, n // 2, n - 1])
    got, lse = kv_ex_calls.prefill(gpu, cache, q, start, F32, window, sinks)
    want = kv_ex_calls.reference(cache, 0, q[some], start + some, window, sinks, None, tiles=n > 100)
    kv_ex_calls.compare(got[some], lse[some], want, f"window {window} sinks {sinks}")
    if n == 5:
        got, lse = kv_ex_calls.decode(gpu, cache, q[-1:], window, sinks)
        want = kv_ex_calls.reference(cache, 0, q[-1:], [start + n - 1], window, sinks, None)
        kv_ex_calls.compare(got, lse, want, f"step, window {window} sinks {sinks}")


def test_estimates_less_than_a_microsecond_apart(gpu):
    """2 queries of 32 heads of 64 over 1024 keys of 8 KV heads: 11.1 us on the persistent kernel, whose pieces and plan need
    scratch memory, 11.5 on the row kernel, which needs none uncut."""
    cache = Cache(np.random.default_rng(1), [1024], 16, 8, 64, F8E4M3).upload()
    q = dev(np.zeros((2, 32, 64), np.float16))
    need = gpu.attention_ex(q=q, q_dtype=F16, q_tok_stride=2048, q_head_stride=64, out=q, out_dtype=F16, out_tok_stride=2048,
                            out_head_stride=64, seq_q=2, num_heads=32, scale=0.1, cache_len=1024, block_table=cache.dev[4], start_pos=1022,
                            window=1024, query_workspace=True, **cache.kwargs())
    assert need > 0
