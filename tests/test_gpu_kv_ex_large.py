"""granite_hip_decode_attention_ex and granite_hip_attention_ex on many sequences, many tiles a worker and many heads,
against kv8.attend (float64).  Pages are shared between sequences and the reference is computed for some of the
sequences and heads, so that the pools and the reference stay small."""
import numpy as np
import pytest

import kv8
from granite_amd import F16, F32, F8E4M3, MASK_CAUSAL
from gpu_util import dev, say
from test_gpu_kv_ex import NAN8, Cache, check, run_prefill, v_top

pytestmark = pytest.mark.gpu


class Shared:
    """A pool of `blocks` blocks; every table entry is one of them, whichever sequence it belongs to."""

    def __init__(self, rng, batch, max_blocks, blocks, bs, hkv, d, kv):
        self.bs, self.hkv, self.d, self.kv, self.blocks = bs, hkv, d, kv, blocks
        shape = (blocks * bs, hkv, d)
        if kv == F8E4M3:
            self.k, self.v = (np.where((c & 0x7F) < 0x70, c, c & 0x8F) for c in rng.integers(0, 256, (2, *shape), dtype=np.uint8))
            self.ks, self.vs = (2.0 ** rng.integers(-7, -4, (2, blocks, hkv))).astype(np.float32)
        else:
            self.k, self.v = rng.standard_normal((2, *shape), dtype=np.float32).astype(np.float16)
            self.ks = self.vs = None
        self.table = rng.integers(0, blocks, (batch, max_blocks)).astype(np.int32)
        self.dev = [None if x is None else dev(x) for x in (self.k, self.v, self.ks, self.vs, self.table)]

    def kwargs(self):
        k, v, ks, vs, _ = self.dev
        return dict(k_cache=k, v_cache=v, kv_dtype=self.kv, k_scale=ks, v_scale=vs, num_blocks=self.blocks, block_size=self.bs,
                    num_kv_heads=self.hkv, head_dim=self.d, max_seq=0)

    def rows(self, i, length, heads=slice(None)):
        scale = [None if s is None else s[:, heads] for s in (self.ks, self.vs)]
        return [kv8.rows_of(x[:, heads], s, self.table[i], self.bs, self.blocks, length)[0] for x, s in zip((self.k, self.v), scale)]


def decode(gpu, cache, lens, hq, q_dtype, window, sinks, some, what):
    b, d = len(lens), cache.d
    q = np.random.default_rng(5).standard_normal((b, hq, d)).astype(np.float16 if q_dtype == F16 else np.float32)
    out, lse = dev(np.full((b, hq, d), 7.0, np.float32)), dev(np.full((b, hq), 7.0, np.float32))
    dq, dl = dev(q), dev(lens)
    gpu.decode_attention_ex(q=dq, q_dtype=q_dtype, out=out, lse=lse, batch_size=b, num_heads=hq, scale=d ** -0.5,
                            block_tables=cache.dev[4], seq_lens=dl, max_blocks_per_seq=cache.table.shape[1], window=window,
                            num_sinks=sinks, **cache.kwargs())
    gpu.sync()
    got, got_lse = out.read(np.float32, (b, hq, d)), lse.read(np.float32, (b, hq))
    assert (got[lens <= 0] == 7.0).all() and np.isfinite(got).all()
    for i in some:
        n = int(lens[i])
        if n <= 0:
            continue
        k, v = cache.rows(i, n)
        vis = kv8.visible([n - 1], n, window, sinks)
        o, l, ds = kv8.attend(q[i:i + 1], k, v, vis, d ** -0.5)
        check(got[i:i + 1], got_lse[i:i + 1], o, l, ds, v_top(v, vis), int(vis.sum()), False, f"{what} seq {i} len {n}")


@pytest.mark.parametrize("kv,bs", [(F8E4M3, 32), (F8E4M3, 24), (F16, 32)])
@pytest.mark.parametrize("batch,top", [(40, 9000), (85, 9000)])
def test_decode_many_tiles_a_worker(gpu, kv, bs, batch, top):
    """Workers walk 40 to 90 tiles of 32 tokens each, over several sequences."""
    say(f"decode many tiles batch={batch} kv={kv} bs={bs}")
    rng = np.random.default_rng(batch)
    cache = Shared(rng, batch, -(-top // bs), 200, bs, 8, 64, kv)
    lens = rng.integers(top - 2000, top + 1, batch).astype(np.int32)
    lens[3], lens[batch // 2], lens[-1] = 0, 1, top
    some = (0, 1, 4, batch // 2, batch - 2, batch - 1)
    if kv == F8E4M3:
        decode(gpu, cache, lens, 8, F16, 0, 0, some, "every key")
    decode(gpu, cache, lens, 16, F32, 6000, 70, some, "window")


@pytest.mark.parametrize("kv,bs", [(F8E4M3, 16), (F8E4M3, 20), (F16, 16)])
@pytest.mark.parametrize("batch", [2560, 2600, 9001])
def test_decode_many_sequences(gpu, kv, bs, batch):
    say(f"decode many sequences batch={batch} kv={kv} bs={bs}")
    rng = np.random.default_rng(batch)
    cache = Shared(rng, batch, -(-1000 // bs), 100, bs, 2, 64, kv)
    lens = rng.choice([0, 1, 15, 16, 33, 64, 200, 1000], batch, p=[.2, .2, .1, .1, .1, .1, .15, .05]).astype(np.int32)
    lens[0], lens[-1] = 777, 1000
    some = [0, 1, 2, 255, 256, 2047, 2048, batch - 2, batch - 1, *rng.integers(0, batch, 60)]
    if kv == F8E4M3:
        decode(gpu, cache, lens, 4, F16, 0, 0, some, "every key")
    decode(gpu, cache, lens, 2, F16, 100, 3, some, "window")


@pytest.mark.parametrize("kv,window,sinks", [(F8E4M3, 0, 0), (F8E4M3, 8800, 300), (F16, 8800, 300)])
@pytest.mark.parametrize("q_dtype,out_dtype", [(F16, F16), (F32, F32)])
def test_prefill_many_tiles_in_one_go(gpu, kv, window, sinks, q_dtype, out_dtype):
    """Enough KV heads for the keys not to be split: a workgroup walks about 150 tiles of 64 keys."""
    say(f"prefill many tiles kv={kv} window={window}")
    n, hq, d, start = 165, 512, 64, 9400
    rng = np.random.default_rng(window)
    cache = Shared(rng, 1, -(-(start + n) // 32), 40, 32, 256, d, kv)
    q = rng.standard_normal((n, hq, d)).astype(np.float16 if q_dtype == F16 else np.float32)
    odt = np.float16 if out_dtype == F16 else np.float32
    out, lse, dq = dev(np.full(q.shape, 7.0, odt)), dev(np.full((hq, n), 7.0, np.float32)), dev(q)
    gpu.attention_ex(q=dq, q_dtype=q_dtype, q_tok_stride=hq * d, q_head_stride=d, out=out, out_dtype=out_dtype,
                     out_tok_stride=hq * d, out_head_stride=d, seq_q=n, num_heads=hq, scale=d ** -0.5, cache_len=start + n,
                     block_table=cache.dev[4], mask_mode=MASK_CAUSAL, start_pos=start, lse=lse, window=window, num_sinks=sinks,
                     **cache.kwargs())
    gpu.sync()
    got, got_lse = out.read(odt, q.shape), lse.read(np.float32, (hq, n)).T
    assert np.isfinite(got).all()
    for kvh in (0, 101, 255):
        k, v = cache.rows(0, start + n, slice(kvh, kvh + 1))
        heads, some = slice(2 * kvh, 2 * kvh + 2), [0, 1, 31, 32, 63, 64, 100, 127, 128, n - 1]
        vis = kv8.visible(start + np.asarray(some), start + n, window, sinks)
        o, l, ds = kv8.attend(q[some, heads], k, v, vis, d ** -0.5)
        check(got[some, heads], got_lse[some, heads], o, l, ds, v_top(v, vis), int(vis.sum(1).max()), out_dtype == F16, f"head {kvh}")


@pytest.mark.parametrize("n,start,bs,hq,hkv,d", [(1, 7000, 16, 8, 2, 128), (2, 6600, 32, 4, 4, 64), (3, 8100, 48, 16, 2, 128), (4, 6143, 16, 7, 1, 64)])
@pytest.mark.parametrize("q_dtype,out_dtype", [(F16, F16), (F32, F32)])
def test_prefill_few_rows_many_keys(gpu, n, start, bs, hq, hkv, d, q_dtype, out_dtype):
    """A draft's worth of queries behind a long context, with released pages and NaNs that not every query sees."""
    say(f"prefill few rows n={n} start={start} bs={bs}")
    cache = Cache(np.random.default_rng(n), [start + n], bs, hkv, d, F8E4M3)
    for j in range(20, 30):
        cache.table[0, j] = (-1, cache.num_blocks, 2147483647)[j % 3]
    at = lambda t: cache.table[0, t // bs] * bs + t % bs  # noqa: E731
    cache.v[at(start + n // 2), 0, 3] = NAN8          # the later queries'
    cache.v[at(start - 6200), 0, 4] = NAN8            # behind the window, of those without one
    cache.upload()
    run_prefill(gpu, cache, n, start, hq, q_dtype, out_dtype)
    run_prefill(gpu, cache, n, start, hq, q_dtype, out_dtype, 6190, 5)
    run_prefill(gpu, cache, n, start, hq, q_dtype, out_dtype, 6200 + n // 2, 0)   # the first queries'


@pytest.mark.parametrize("kv,bs", [(F8E4M3, 5), (F8E4M3, 16), (F16, 7), (F16, 12)])
def test_prefill_seventy_thousand_queries(gpu, kv, bs):
    say(f"prefill 70000 queries kv={kv} bs={bs}")
    n, d, start = 70000, 64, 11
    rng = np.random.default_rng(bs)
    cache = Shared(rng, 1, -(-(start + n) // bs), 50, bs, 1, d, kv)
    q = rng.standard_normal((n, 1, d), dtype=np.float32).astype(np.float16)
    out, dq = dev(np.full(q.shape, 7.0, np.float16)), dev(q)
    lse = dev(np.full((1, n), 7.0, np.float32))
    gpu.attention_ex(q=dq, q_dtype=F16, q_tok_stride=d, q_head_stride=d, out=out, out_dtype=F16, out_tok_stride=d, out_head_stride=d,
                     seq_q=n, num_heads=1, scale=d ** -0.5, cache_len=start + n, block_table=cache.dev[4], mask_mode=MASK_CAUSAL,
                     start_pos=start, lse=lse, window=33, num_sinks=2, **cache.kwargs())
    gpu.sync()
    got, got_lse = out.read(np.float16, q.shape), lse.read(np.float32, (1, n)).T
    assert np.isfinite(got).all()
    k, v = cache.rows(0, start + n)
    for some in ([0, 1, 30], [32760, 32767, 32768], [65534, 65535, 65536, n - 1]):
        vis = kv8.visible(start + np.asarray(some), start + n, 33, 2)
        o, l, ds = kv8.attend(q[some], k, v, vis, d ** -0.5)
        check(got[some], got_lse[some], o, l, ds, v_top(v, vis), int(vis.sum(1).max()), True, f"queries {some}")
