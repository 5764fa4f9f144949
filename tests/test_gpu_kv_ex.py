"""GPU parity of granite_hip_decode_attention_ex and granite_hip_attention_ex against kv8.attend (float64):
8-bit pools, sliding windows with sinks, ragged and odd sizes, garbage in every place no query sees."""
import ctypes as C

import numpy as np
import pytest

import kv8
from granite_amd import F16, F32, F8E4M3, MASK_CAUSAL, MASK_NONE, GraniteHipError, _capi
from gpu_util import dev, say

pytestmark = pytest.mark.gpu
NAN8, NAN16 = 0x7F, np.float16(np.nan)


class Cache:
    """Paged (bs > 0) or contiguous cache of sequences of the given lengths.  Everything no token occupies is NaN: rows
    behind a sequence's end, blocks of nobody, their scales; table entries behind a sequence's last block are -1."""

    def __init__(self, rng, lens, bs, hkv, d, kv, spare=3, spread=1.0, scales="pow2"):
        self.bs, self.hkv, self.d, self.kv, self.lens = bs, hkv, d, kv, list(lens)
        f8 = kv == F8E4M3
        if not bs:
            n = max(self.lens)
            self.max_seq = n + spare
            self.k = np.full((hkv, self.max_seq, d), NAN16)
            self.v = self.k.copy()
            self.k[:, :n], self.v[:, :n] = rng.standard_normal((2, hkv, n, d)).astype(np.float16)
            self.ks = self.vs = self.table = None
            self.num_blocks = self.max_blocks = 0
        else:
            used = [-(-n // bs) for n in self.lens]
            self.num_blocks, self.max_blocks, self.max_seq = sum(used) + spare, max(max(used), 1) + 1, 0
            order = rng.permutation(self.num_blocks).astype(np.int32)
            self.table = np.full((len(self.lens), self.max_blocks), -1, np.int32)
            shape = (self.num_blocks * bs, hkv, d)
            self.k = np.full(shape, NAN8, np.uint8) if f8 else np.full(shape, NAN16)
            self.v = self.k.copy()
            self.ks = np.full((self.num_blocks, hkv), np.nan, np.float32)
            self.vs = self.ks.copy()
            at = 0
            for i, (n, u) in enumerate(zip(self.lens, used)):
                self.table[i, :u] = order[at:at + u]
                at += u
                for j in range(u):
                    b, rows = self.table[i, j], min(bs, n - j * bs)
                    for pool, scale, spr in ((self.k, self.ks, 1.0), (self.v, self.vs, spread)):
                        x = rng.standard_normal((rows, hkv, d))
                        if not f8:
                            pool[b * bs:b * bs + rows] = x.astype(np.float16)
                            continue
                        x *= spr ** rng.uniform(-1, 1, (1, hkv, 1))
                        s = np.array([kv8.scale_for(np.abs(x[:, h]).max()) for h in range(hkv)], np.float32)
                        if scales == "any":
                            s = (s * rng.uniform(1, 1.9, hkv)).astype(np.float32)
                        pool[b * bs:b * bs + rows] = kv8.encode8(x / s[None, :, None])
                        scale[b] = s

    def upload(self):
        self.dev = [None if x is None else dev(x) for x in (self.k, self.v, self.ks, self.vs, self.table)]
        return self

    def kwargs(self):
        k, v, ks, vs, _ = self.dev
        return dict(k_cache=k, v_cache=v, kv_dtype=self.kv, k_scale=ks if self.kv == F8E4M3 else None,
                    v_scale=vs if self.kv == F8E4M3 else None, num_blocks=self.num_blocks, block_size=self.bs,
                    num_kv_heads=self.hkv, head_dim=self.d, max_seq=self.max_seq)

    def rows(self, i, length):
        if not self.bs:
            return (np.swapaxes(x[:, :length], 0, 1).astype(np.float64) for x in (self.k, self.v)), np.ones(length, bool)
        k, valid = kv8.rows_of(self.k, self.ks, self.table[i], self.bs, self.num_blocks, length)
        v, _ = kv8.rows_of(self.v, self.vs, self.table[i], self.bs, self.num_blocks, length)
        return (k, v), valid


def check(got, got_lse, out, lse, ds, v_top, tokens, half, what):
    tol, tol_lse = kv8.bounds(out, lse, ds, v_top, tokens, half)
    got, got_lse = np.asarray(got, np.float64), np.asarray(got_lse, np.float64)
    assert np.array_equal(np.isnan(out), np.isnan(got)), f"{what}: NaN"
    with np.errstate(invalid="ignore"):
        off = np.where(out == got, 0, np.abs(got - out))
        off_lse = np.where(lse == got_lse, 0, np.abs(got_lse - lse))
    bad = np.argwhere(off > tol)
    assert len(bad) == 0, f"{what}: {len(bad)} of {out.size} off, first {bad[0]}: {got[tuple(bad[0])]} for {out[tuple(bad[0])]}, allowed {tol[tuple(bad[0])]}"
    bad = np.argwhere(off_lse > tol_lse)
    assert len(bad) == 0, f"{what}: lse {bad[0]}: {got_lse[tuple(bad[0])]} for {lse[tuple(bad[0])]}"


def v_top(v, vis):
    seen = v[vis.any(0)]
    return float(np.abs(seen[np.isfinite(seen)]).max(initial=0.0))


def run_decode(gpu, cache, hq, q_dtype, window=0, sinks=0, lens=None, seed=0, what="decode", scale=None, **more):
    lens = np.asarray(cache.lens if lens is None else lens, np.int32)
    b, d = len(lens), cache.d
    scale = d ** -0.5 if scale is None else scale
    q = np.random.default_rng(seed + 99).standard_normal((b, hq, d)).astype(np.float16 if q_dtype == F16 else np.float32)
    out, lse = dev(np.full((b, hq, d), 7.0, np.float32)), dev(np.full((b, hq), 7.0, np.float32))
    dq, dl = dev(q), dev(lens)
    gpu.decode_attention_ex(q=dq, q_dtype=q_dtype, out=out, lse=lse, batch_size=b, num_heads=hq, scale=scale,
                            block_tables=cache.dev[4], seq_lens=dl, max_blocks_per_seq=cache.max_blocks, window=window,
                            num_sinks=sinks, **cache.kwargs(), **more)
    gpu.sync()
    got, got_lse = out.read(np.float32, (b, hq, d)), lse.read(np.float32, (b, hq))
    for i, n in enumerate(lens):
        if n <= 0:
            assert (got[i] == 7.0).all() and (got_lse[i] == 7.0).all(), f"{what}: an empty sequence was written"
            continue
        (k, v), valid = cache.rows(i, int(n))
        vis = kv8.visible([n - 1], int(n), window, sinks, valid)
        o, l, ds = kv8.attend(q[i:i + 1], k, v, vis, scale)
        check(got[i:i + 1], got_lse[i:i + 1], o, l, ds, v_top(v, vis), int(vis.sum()), False, f"{what} seq {i} len {n}")
    return got, got_lse


def run_prefill(gpu, cache, n, start, hq, q_dtype, out_dtype, window=0, sinks=0, cache_len=None, seed=0, heads_first=False,
                mask=MASK_CAUSAL, what="prefill", scale=None, **more):
    d = cache.d
    scale = d ** -0.5 if scale is None else scale
    length = cache.lens[0] if cache_len is None else cache_len
    rng = np.random.default_rng(seed + 7)
    q = rng.standard_normal((n, hq, d)).astype(np.float16 if q_dtype == F16 else np.float32)
    odt = np.float16 if out_dtype == F16 else np.float32
    stored = np.ascontiguousarray(q.transpose(1, 0, 2)) if heads_first else q
    strides = (d, n * d) if heads_first else (hq * d, d)
    out, lse, dq = dev(np.full(stored.shape, 7.0, odt)), dev(np.full((hq, n), 7.0, np.float32)), dev(stored)
    gpu.attention_ex(q=dq, q_dtype=q_dtype, q_tok_stride=strides[0], q_head_stride=strides[1], out=out, out_dtype=out_dtype,
                     out_tok_stride=strides[0], out_head_stride=strides[1], seq_q=n, num_heads=hq, scale=scale,
                     cache_len=length, block_table=cache.dev[4], mask_mode=mask, start_pos=start, lse=lse, window=window,
                     num_sinks=sinks, **cache.kwargs(), **more)
    gpu.sync()
    got = out.read(odt, stored.shape)
    got = got.transpose(1, 0, 2) if heads_first else got
    (k, v), valid = cache.rows(0, length)
    vis = kv8.visible(start + np.arange(n), length, window, sinks, valid, mask == MASK_CAUSAL)
    o, l, ds = kv8.attend(q, k, v, vis, scale)
    check(got, lse.read(np.float32, (hq, n)).T, o, l, ds, v_top(v, vis), int(vis.sum(1).max()), out_dtype == F16, what)
    return got


# ------------------------------------------------------------------ decode

@pytest.mark.parametrize("q_dtype", [F16, F32])
@pytest.mark.parametrize("bs,hq,hkv,d", [(16, 32, 8, 128), (32, 8, 8, 64), (1, 4, 2, 128), (20, 28, 4, 128), (8, 12, 2, 64),
                                         (48, 16, 1, 128), (64, 48, 1, 64), (128, 40, 5, 128)])
def test_decode_8bit(gpu, bs, hq, hkv, d, q_dtype):
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 200, 0, 511, 777]
    say(f"decode 8-bit bs={bs} hq={hq} hkv={hkv} d={d} q={q_dtype}")
    run_decode(gpu, Cache(np.random.default_rng(bs + hq), lens, bs, hkv, d, F8E4M3).upload(), hq, q_dtype)


@pytest.mark.parametrize("kv,bs", [(F8E4M3, 16), (F8E4M3, 20), (F16, 16), (F16, 24), (F16, 48)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (7, 1), (16, 4), (64, 0), (100, 33), (128, 16), (500, 4), (5000, 4), (40, 5000)])
def test_decode_window(gpu, kv, bs, window, sinks):
    say(f"decode window={window} sinks={sinks} kv={kv} bs={bs}")
    lens = [1, 2, 16, 40, 41, 129, 0, 333, 640, 1001]
    for hq, hkv, d, q in ((8, 2, 128, F16), (6, 3, 64, F32)):
        run_decode(gpu, Cache(np.random.default_rng(window), lens, bs, hkv, d, kv).upload(), hq, q, window, sinks)


@pytest.mark.parametrize("n,window,sinks", [(1, 3, 0), (77, 10, 2), (1000, 256, 4), (3001, 1024, 16)])
def test_decode_window_contiguous(gpu, n, window, sinks):
    for hq, hkv, d, q in ((8, 8, 128, F32), (14, 2, 64, F16)):
        run_decode(gpu, Cache(np.random.default_rng(n), [n], 0, hkv, d, F16).upload(), hq, q, window, sinks)


@pytest.mark.parametrize("lens,bs,hq,hkv,d", [([5000], 16, 32, 8, 128), ([20011, 3], 32, 8, 1, 128), ([9000, 1, 8191, 64], 16, 16, 16, 64),
                                              ([4099] * 3 + [12000], 24, 12, 4, 128), (list(range(1, 2000, 40)), 16, 16, 2, 64)])
def test_decode_long_and_mixed(gpu, lens, bs, hq, hkv, d):
    """Contexts that are cut into several parts and joined, with and without a window."""
    say(f"decode long {len(lens)} x {max(lens)} bs={bs}")
    cache = Cache(np.random.default_rng(len(lens)), lens, bs, hkv, d, F8E4M3).upload()
    run_decode(gpu, cache, hq, F16)
    run_decode(gpu, cache, hq, F32, 3000, 5)


def test_decode_fixed_length_and_bounds(gpu):
    """seq_lens NULL: the host's length for all; lengths beyond the table are cut at its end, negative ones are empty."""
    cache = Cache(np.random.default_rng(3), [100, 100], 16, 2, 128, F8E4M3).upload()
    q = np.random.default_rng(4).standard_normal((2, 4, 128)).astype(np.float16)
    dq, outs = dev(q), []
    for lens, fixed in ((None, 100), (dev(np.array([100, 100], np.int32)), 0)):
        out = dev(np.zeros((2, 4, 128), np.float32))
        gpu.decode_attention_ex(q=dq, q_dtype=F16, out=out, batch_size=2, num_heads=4, scale=0.1, block_tables=cache.dev[4],
                                seq_lens=lens, fixed_seq_len=fixed, max_blocks_per_seq=cache.max_blocks, **cache.kwargs())
        gpu.sync()
        outs.append(out.read(np.float32, (2, 4, 128)))
    assert np.array_equal(outs[0], outs[1])
    run_decode(gpu, cache, 4, F16, lens=[-5, 100])
    full = Cache(np.random.default_rng(3), [cache_len := 96, 96], 16, 2, 128, F8E4M3)
    full.table, full.max_blocks = np.ascontiguousarray(full.table[:, :6]), 6
    full.upload()
    out = dev(np.zeros((2, 4, 128), np.float32))
    far, near = dev(np.array([2147483647, 97], np.int32)), dev(np.array([96, 96], np.int32))
    res = []
    for lens in (far, near):
        gpu.decode_attention_ex(q=dq, q_dtype=F16, out=out, batch_size=2, num_heads=4, scale=0.1, block_tables=full.dev[4],
                                seq_lens=lens, max_blocks_per_seq=6, **full.kwargs())
        gpu.sync()
        res.append(out.read(np.float32, (2, 4, 128)))
    assert cache_len == 96 and np.array_equal(res[0], res[1])


@pytest.mark.parametrize("bs", [16, 20, 8])
def test_decode_released_pages(gpu, bs):
    """Under a window the blocks between the sinks and the window are released: their entries are stale (-1, or
    anything).  Without one, tokens of invalid pages do not count; a sequence of only such pages gets zeros."""
    rng = np.random.default_rng(bs)
    lens = [1000, 500, 130, 64]
    cache = Cache(rng, lens, bs, 2, 128, F8E4M3)
    for i, n in enumerate(lens):
        keep = {t // bs for t in range(4)} | {t // bs for t in range(max(0, n - 100), n)}
        for j in range(-(-n // bs)):
            if j not in keep:
                cache.table[i, j] = rng.choice([-1, cache.num_blocks, 2147483647, -2147483648])
    cache.upload()
    run_decode(gpu, cache, 8, F16, 100, 4, what="released")
    run_decode(gpu, cache, 8, F32, what="invalid pages")
    cache.table[1:3] = -1
    cache.upload()
    got, lse = run_decode(gpu, cache, 8, F16, what="no page at all")
    assert (got[1:3] == 0).all() and np.isneginf(lse[1:3]).all()


def test_decode_scales(gpu):
    """Scales that are no powers of two, and V scales that differ by a factor of a million between blocks."""
    lens = [700, 33, 1500]
    for scales, spread in (("any", 1.0), ("pow2", 1000.0), ("any", 1000.0)):
        for bs in (16, 20):
            run_decode(gpu, Cache(np.random.default_rng(9), lens, bs, 2, 128, F8E4M3, spread=spread, scales=scales).upload(), 8, F16,
                       what=f"scales {scales} {spread}")


def test_decode_large_scores(gpu):
    """Scores of a few thousand: the softmax is one key or two."""
    cache = Cache(np.random.default_rng(10), [900, 70], 16, 2, 64, F8E4M3).upload()
    run_decode(gpu, cache, 4, F32, scale=100.0)
    run_decode(gpu, cache, 4, F32, scale=-100.0)
    run_decode(gpu, cache, 4, F32, scale=0.0)


def test_nan_where_it_is_seen(gpu):
    """A NaN or an infinity in a visible row does reach the result, and only that sequence's and head's."""
    cache = Cache(np.random.default_rng(11), [200, 200], 16, 2, 128, F8E4M3)
    row = cache.table[0, 5] * 16 + 3
    cache.v[row, 1, 7] = NAN8
    got, _ = run_decode(gpu, cache.upload(), 4, F16)
    assert np.isnan(got[0, 2:, 7]).all() and np.isnan(got).sum() == 2
    half = Cache(np.random.default_rng(12), [300], 16, 1, 64, F16)
    half.v[half.table[0, 18] * 16 + 2, 0, 5] = np.inf    # token 290: in the window
    half.v[half.table[0, 3] * 16 + 2, 0, 6] = np.nan     # token 50: not
    half.k[half.table[0, 3] * 16 + 3, 0, :] = np.inf
    got, _ = run_decode(gpu, half.upload(), 2, F16, 64, 4)
    assert np.isposinf(got[0, :, 5]).all() and np.isfinite(np.delete(got, 5, -1)).all()


def test_infinities_that_are_seen(gpu):
    """An infinity anywhere in what a row sees makes its sum infinite, whatever the probability's rounding."""
    for bs, lens in ((16, [2000, 90]), (20, [2000, 90]), (16, [300])):
        cache = Cache(np.random.default_rng(21), lens, bs, 2, 64, F16)
        at = lambda t: cache.table[0, t // bs] * bs + t % bs  # noqa: E731
        n = lens[0]
        cache.v[at(n - 1), 0, 3] = cache.v[at(n - 60), 0, 4] = np.inf
        cache.v[at(n - 40), 1, 5] = -np.inf
        cache.v[at(n - 41), 1, 6], cache.v[at(n - 42), 1, 6] = np.inf, -np.inf
        cache.upload()
        got, _ = run_decode(gpu, cache, 4, F16, n - 7, 2)
        assert np.isposinf(got[0, :2, 3:5]).all() and np.isneginf(got[0, 2:, 5]).all() and np.isnan(got[0, 2:, 6]).all()
        for q, o in ((F16, F16), (F32, F32)):
            for rows in (5, 130):
                run_prefill(gpu, cache, rows, n - rows, 4, q, o, n - 7, 2, cache_len=n, scale=0.02)


# ------------------------------------------------------------------ several queries

@pytest.mark.parametrize("n,start,bs,hq,hkv,d", [
    (1, 0, 16, 8, 2, 128), (2, 63, 16, 8, 8, 64), (5, 1000, 16, 32, 8, 128), (16, 0, 20, 4, 1, 128), (37, 500, 32, 12, 4, 64),
    (64, 0, 16, 6, 2, 128), (100, 29, 8, 4, 4, 64), (129, 200, 64, 8, 2, 128), (257, 0, 16, 4, 2, 128), (300, 77, 48, 14, 2, 64),
    (513, 130, 128, 2, 1, 128), (70, 3, 1, 2, 2, 64), (31, 2500, 16, 48, 1, 128)])
@pytest.mark.parametrize("q_dtype,out_dtype", [(F16, F16), (F32, F32), (F16, F32), (F32, F16)])
def test_prefill_8bit(gpu, n, start, bs, hq, hkv, d, q_dtype, out_dtype):
    say(f"prefill 8-bit n={n} start={start} bs={bs} hq={hq} hkv={hkv} d={d} q={q_dtype} out={out_dtype}")
    cache = Cache(np.random.default_rng(n), [start + n], bs, hkv, d, F8E4M3).upload()
    run_prefill(gpu, cache, n, start, hq, q_dtype, out_dtype, heads_first=n % 2 == 1)


@pytest.mark.parametrize("kv,bs", [(F8E4M3, 16), (F8E4M3, 20), (F16, 16), (F16, 0), (F16, 12)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 2), (64, 0), (100, 4), (130, 70), (256, 300), (4000, 4)])
def test_prefill_window(gpu, kv, bs, window, sinks):
    say(f"prefill window={window} sinks={sinks} kv={kv} bs={bs}")
    for n, start, hq, hkv, d, q, o in ((300, 0, 4, 2, 128, F16, F16), (65, 700, 6, 2, 64, F32, F32), (3, 901, 8, 8, 128, F16, F32),
                                       (200, 400, 2, 1, 128, F32, F16)):
        run_prefill(gpu, Cache(np.random.default_rng(n), [start + n], bs, hkv, d, kv).upload(), n, start, hq, q, o, window, sinks,
                    what=f"n={n} start={start}")


@pytest.mark.parametrize("out_dtype", [F16, F32])
def test_prefill_every_key(gpu, out_dtype):
    for n, length, bs in ((50, 333, 16), (200, 31, 20), (3, 1, 16)):
        run_prefill(gpu, Cache(np.random.default_rng(n), [length], bs, 2, 128, F8E4M3).upload(), n, 0, 4, F16, out_dtype, mask=MASK_NONE)


@pytest.mark.parametrize("out_dtype", [F16, F32])
def test_prefill_rows_that_see_nothing(gpu, out_dtype):
    """Queries beyond the cache whose window lies behind its end, pages that are all invalid."""
    cache = Cache(np.random.default_rng(1), [100], 16, 2, 128, F8E4M3).upload()
    got = run_prefill(gpu, cache, 60, 90, 4, F16, out_dtype, window=20)
    assert (got[30:] == 0).all() and (got[:29] != 0).any()
    run_prefill(gpu, cache, 300, 90, 4, F16, out_dtype, window=20)
    run_prefill(gpu, cache, 300, 90, 4, F16, out_dtype, window=20, sinks=3)
    run_prefill(gpu, cache, 10, 5000, 4, F32, out_dtype, window=20)
    cache.table[:] = -1
    cache.upload()
    assert (run_prefill(gpu, cache, 100, 0, 4, F16, out_dtype) == 0).all()


@pytest.mark.parametrize("out_dtype", [F16, F32])
@pytest.mark.parametrize("n", [6, 200])
def test_prefill_garbage_no_query_sees(gpu, out_dtype, n):
    """NaN and infinities in keys that some queries see and others do not: they reach the former only."""
    for bs in (16, 20):
        cache = Cache(np.random.default_rng(2), [n + 300], bs, 2, 64, F16)
        at = lambda t: cache.table[0, t // bs] * bs + t % bs  # noqa: E731
        cache.v[at(300 + n // 2), 0, 3] = np.inf
        cache.v[at(300 + n // 2), 1, 4] = np.nan
        cache.v[at(300 + n // 3), 1, 5] = -np.inf
        cache.k[at(310 if n > 100 else 303), 1, :] = np.nan
        run_prefill(gpu, cache.upload(), n, 300, 4, F16, out_dtype, window=40, sinks=4)
    f8 = Cache(np.random.default_rng(2), [n + 300], 16, 2, 128, F8E4M3)
    f8.v[f8.table[0, (300 + n // 2) // 16] * 16 + (300 + n // 2) % 16, 1, 9] = NAN8
    f8.vs[f8.table[0, 5]] = np.nan  # a block between the sinks and the first window
    f8.ks[f8.table[0, 6]] = np.inf
    run_prefill(gpu, f8.upload(), n, 300, 4, F16, out_dtype, window=40, sinks=4)
    run_prefill(gpu, f8, n, 150, 4, F16, out_dtype, window=20, sinks=4, cache_len=150 + n)


def test_prefill_released_pages(gpu):
    cache = Cache(np.random.default_rng(3), [900], 16, 2, 128, F8E4M3)
    cache.table[0, 1:40] = [-1, cache.num_blocks, 2147483647] * 13
    run_prefill(gpu, cache.upload(), 200, 700, 4, F16, F16, window=60, sinks=16)


def test_prefill_scales(gpu):
    for scales, spread in (("any", 1.0), ("pow2", 1000.0)):
        for out in (F16, F32):
            for bs in (16, 20):
                run_prefill(gpu, Cache(np.random.default_rng(9), [700], bs, 2, 128, F8E4M3, spread=spread, scales=scales).upload(), 180, 520,
                            4, F16, out, what=f"scales {scales} {spread}")


@pytest.mark.parametrize("out_dtype", [F16, F32])
@pytest.mark.parametrize("scale", [20.0, -0.3, 0.0, 1e-30])
def test_prefill_other_factors(gpu, out_dtype, scale):
    for kv, bs in ((F8E4M3, 16), (F16, 16), (F16, 0)):
        cache = Cache(np.random.default_rng(20), [400], bs, 2, 64, kv).upload()
        run_prefill(gpu, cache, 150, 250, 4, F32, out_dtype, window=120, sinks=3, scale=scale, what=f"scale {scale}")


@pytest.mark.parametrize("n,start,hq,hkv", [(9, 20000, 8, 1), (40, 9000, 4, 2), (300, 5000, 2, 1), (64, 3333, 8, 2)])
def test_prefill_keys_split(gpu, n, start, hq, hkv):
    """Few rows over many keys: the keys are cut into several parts, with odd numbers of tiles in them."""
    for q, o in ((F16, F16), (F32, F32)):
        cache = Cache(np.random.default_rng(n), [start + n], 16, hkv, 128, F8E4M3).upload()
        run_prefill(gpu, cache, n, start, hq, q, o)
        run_prefill(gpu, cache, n, start, hq, q, o, window=2345, sinks=70)


# ------------------------------------------------------------------ both

def test_half_caches_without_a_window_are_the_other_entry_points(gpu):
    cache = Cache(np.random.default_rng(4), [300, 40], 16, 2, 128, F16).upload()
    q = np.random.default_rng(5).standard_normal((2, 4, 128)).astype(np.float16)
    dq, dl, a, b = dev(q), dev(np.array([300, 40], np.int32)), dev(np.zeros((2, 4, 128), np.float32)), dev(np.zeros((2, 4, 128), np.float32))
    kw = dict(q=dq, q_dtype=F16, batch_size=2, num_heads=4, scale=0.1, block_tables=cache.dev[4], seq_lens=dl, max_blocks_per_seq=cache.max_blocks)
    gpu.decode_attention_ex(out=a, **kw, **cache.kwargs())
    gpu.decode_attention(out=b, k_cache=cache.dev[0], v_cache=cache.dev[1], num_kv_heads=2, head_dim=128, block_size=16, **kw)
    gpu.sync()
    assert np.array_equal(a.read(np.float32, (2, 4, 128)), b.read(np.float32, (2, 4, 128)))


def test_pools_beyond_four_gibibytes(gpu):
    """The sequence's blocks lie at the far end of pools of 4.5 GiB: offsets beyond 32 bits."""
    hkv, d, bs, n = 8, 128, 16, 300
    num_blocks = int(4.5 * 2 ** 30) // (bs * hkv * d)
    small = Cache(np.random.default_rng(6), [n], bs, hkv, d, F8E4M3, spare=0)
    used = small.num_blocks
    pools = [gpu.create_buffer(num_blocks * bs * hkv * d) for _ in range(2)]
    scales = [gpu.create_buffer(num_blocks * hkv * 4) for _ in range(2)]
    first = num_blocks - used
    for buf, x in zip(pools + scales, (small.k, small.v, small.ks, small.vs)):
        buf.write(x, first * x.nbytes // used)
    table = dev(np.where(small.table >= 0, small.table + first, -1).astype(np.int32))
    q = np.random.default_rng(7).standard_normal((1, 16, d)).astype(np.float16)
    dq, dl, out, lse = dev(q), dev(np.array([n], np.int32)), dev(np.zeros((1, 16, d), np.float32)), dev(np.zeros((1, 16), np.float32))
    kw = dict(q=dq, q_dtype=F16, out=out, lse=lse, num_heads=16, num_kv_heads=hkv, head_dim=d, scale=d ** -0.5, kv_dtype=F8E4M3,
              k_cache=pools[0], v_cache=pools[1], k_scale=scales[0], v_scale=scales[1], num_blocks=num_blocks, block_size=bs)
    (k, v), valid = small.rows(0, n)
    vis = kv8.visible([n - 1], n, 0, 0, valid)
    o, l, ds = kv8.attend(q, k, v, vis, d ** -0.5)
    gpu.decode_attention_ex(batch_size=1, block_tables=table, seq_lens=dl, max_blocks_per_seq=small.max_blocks, **kw)
    gpu.sync()
    check(out.read(np.float32, (1, 16, d)), lse.read(np.float32, (1, 16)), o, l, ds, v_top(v, vis), n, False, "decode far")
    gpu.attention_ex(q_tok_stride=16 * d, q_head_stride=d, out_dtype=F32, out_tok_stride=16 * d, out_head_stride=d, seq_q=1,
                     cache_len=n, block_table=table, start_pos=n - 1, **kw)
    gpu.sync()
    check(out.read(np.float32, (1, 16, d)), lse.read(np.float32, (16, 1)).T, o, l, ds, v_top(v, vis), n, False, "prefill far")
    # and the append there
    x = np.random.default_rng(8).standard_normal((1, hkv, d)).astype(np.float32)
    dx = dev(x)
    gpu.rope_append_q8(seq_len=1, head_dim=d, src_dtype=F32, k=dx, v=dx, num_heads_k=hkv, k_cache=pools[0], v_cache=pools[1],
                       k_scale=scales[0], v_scale=scales[1], block_table=table, block_size=bs, num_blocks=num_blocks,
                       max_blocks_per_seq=small.max_blocks, start_pos=n)
    gpu.sync()
    want, want_s = small.v.copy(), small.vs.copy()
    kv8.append8(x, want, want_s, small.table[0], n, bs, used)
    assert np.array_equal(pools[1].read(np.uint8, want.shape, first * want.nbytes // used), want)
    for b in pools + scales:
        b.free()


def test_workspace(gpu):
    """The scratch a launch asks for is enough and is all it uses; less is refused before anything runs."""
    cache = Cache(np.random.default_rng(13), [9000, 17], 16, 2, 128, F8E4M3).upload()
    q = np.random.default_rng(14).standard_normal((2, 4, 128)).astype(np.float16)
    dq, dl = dev(q), dev(np.array([9000, 17], np.int32))
    out = dev(np.zeros((2, 4, 128), np.float32))
    kw = dict(q=dq, q_dtype=F16, out=out, batch_size=2, num_heads=4, scale=0.1, block_tables=cache.dev[4], seq_lens=dl,
              max_blocks_per_seq=cache.max_blocks, **cache.kwargs())
    pkw = dict(q=dq, q_dtype=F16, q_tok_stride=512, q_head_stride=128, out=out, out_dtype=F32, out_tok_stride=512, out_head_stride=128,
               seq_q=2, num_heads=4, scale=0.1, cache_len=9000, block_table=cache.dev[4], start_pos=8998, **cache.kwargs())
    for call, args in ((gpu.decode_attention_ex, kw), (gpu.attention_ex, pkw)):
        need = call(**args, query_workspace=True)
        assert need > 0
        guard = 4096
        ws = dev(np.full(need + guard, 0xAB, np.uint8))
        call(**args)
        gpu.sync()
        want = out.read(np.float32, (2, 4, 128))
        out.fill(0)
        call(**args, workspace=ws, workspace_bytes=need)
        gpu.sync()
        assert np.array_equal(out.read(np.float32, (2, 4, 128)), want)
        assert (ws.read(np.uint8, guard, need) == 0xAB).all()
        with pytest.raises(GraniteHipError) as e:
            call(**args, workspace=ws, workspace_bytes=need - 1)
        assert e.value.code == _capi.ESCRATCH
        with pytest.raises(GraniteHipError) as e:
            call(**args, workspace=ws.ptr + 16, workspace_bytes=need)
        assert e.value.code == _capi.EINVAL


def test_prompt_in_chunks_then_decode_steps(gpu, oracle):
    """The operators together, as a serving loop uses them: a prompt appended and attended in chunks, then steps of
    a batch in which it is joined by a second sequence, all of it under a window with sinks and with the blocks
    behind the window released; results against float64 on the cache the appends should have left."""
    hq, hkv, d, bs, window, sinks = 8, 2, 128, 16, 96, 4
    rng = np.random.default_rng(15)
    total, chunks, second = 330, (100, 1, 150), 40
    blocks = 40
    table = np.full((2, 24), -1, np.int32)
    table[0, :21], table[1, :4] = rng.permutation(blocks)[:21], 0
    rest = [b for b in range(blocks) if b not in table[0, :21]]
    table[1, :4] = rest[:4]
    k_pool, v_pool = np.full((blocks * bs, hkv, d), NAN8, np.uint8), np.full((blocks * bs, hkv, d), NAN8, np.uint8)
    ks, vs = np.full((blocks, hkv), np.nan, np.float32), np.full((blocks, hkv), np.nan, np.float32)
    buf = [dev(x) for x in (k_pool, v_pool, ks, vs)]
    cos, sin = oracle.rope_table(400, d, 10000.0)
    dcos, dsin = dev(cos), dev(sin)
    dtable = dev(table)
    form = dict(k_cache=buf[0], v_cache=buf[1], k_scale=buf[2], v_scale=buf[3], num_blocks=blocks, block_size=bs)
    att = dict(kv_dtype=F8E4M3, window=window, num_sinks=sinks, num_heads=hq, num_kv_heads=hkv, head_dim=d, scale=d ** -0.5)

    def tokens(n, h):
        return rng.standard_normal((n, h, d)).astype(np.float32)

    def remember(seq, pos, k, v):
        kv8.append8(oracle.rope_apply(k, pos, cos, sin), k_pool, ks, table[seq], pos, bs, blocks)
        kv8.append8(v, v_pool, vs, table[seq], pos, bs, blocks)

    def want(seq, pos, q):
        n = len(q)
        k, valid = kv8.rows_of(k_pool, ks, table[seq], bs, blocks, pos + n)
        v, _ = kv8.rows_of(v_pool, vs, table[seq], bs, blocks, pos + n)
        vis = kv8.visible(pos + np.arange(n), pos + n, window, sinks, valid)
        # the half copy of the rotated queries is what the attention reads
        rq = oracle.rope_apply(q, pos, cos, sin).astype(np.float16)
        return (*kv8.attend(rq, k, v, vis, d ** -0.5), v_top(v, vis), int(vis.sum(1).max()))

    def chunk(seq, pos, n):
        q, k, v = tokens(n, hq), tokens(n, hkv), tokens(n, hkv)
        keep = [dev(x) for x in (q, k, v, table[seq])]
        q16, out, lse = dev(np.zeros((n, hq, d), np.float16)), dev(np.zeros((n, hq, d), np.float16)), dev(np.zeros((hq, n), np.float32))
        gpu.rope_append_q8(seq_len=n, head_dim=d, src_dtype=F32, q=keep[0], q_out=q16, num_heads_q=hq, k=keep[1], v=keep[2],
                           num_heads_k=hkv, start_pos=pos, cos_table=dcos, sin_table=dsin, table_positions=400,
                           block_table=keep[3], max_blocks_per_seq=24, **form)
        gpu.attention_ex(q=q16, q_dtype=F16, q_tok_stride=hq * d, q_head_stride=d, out=out, out_dtype=F16, out_tok_stride=hq * d,
                         out_head_stride=d, lse=lse, seq_q=n, cache_len=pos + n, start_pos=pos, block_table=keep[3], **form, **att)
        gpu.sync()
        remember(seq, pos, k, v)
        o, l, ds, top, seen = want(seq, pos, q)
        check(out.read(np.float16, o.shape), lse.read(np.float32, (hq, n)).T, o, l, ds, top, seen, True, f"chunk at {pos}")

    pos = 0
    for n in chunks:
        chunk(0, pos, n)
        pos += n
    chunk(1, 0, second)
    lens = [pos, second]
    for step in range(24):
        dead = max(0, (lens[0] + 1 - window) // bs)  # blocks before the window's first
        table[0, -(-sinks // bs):dead] = -1
        dtable.write(table)
        q, k, v = tokens(2, hq), tokens(2, hkv), tokens(2, hkv)
        p = np.array(lens, np.int32)
        keep = [dev(x) for x in (q, k, v, p, p + 1)]
        q16, out, lse = dev(np.zeros((2, hq, d), np.float16)), dev(np.zeros((2, hq, d), np.float32)), dev(np.zeros((2, hq), np.float32))
        gpu.rope_append_q8(seq_len=2, head_dim=d, src_dtype=F32, q=keep[0], q_out=q16, num_heads_q=hq, k=keep[1], v=keep[2],
                           num_heads_k=hkv, positions=keep[3], table_stride=24, cos_table=dcos, sin_table=dsin, table_positions=400,
                           block_table=dtable, max_blocks_per_seq=24, **form)
        gpu.decode_attention_ex(q=q16, q_dtype=F16, out=out, lse=lse, batch_size=2, block_tables=dtable, seq_lens=keep[4],
                                max_blocks_per_seq=24, **form, **att)
        gpu.sync()
        got, got_lse = out.read(np.float32, (2, hq, d)), lse.read(np.float32, (2, hq))
        for i in range(2):
            remember(i, lens[i], k[i:i + 1], v[i:i + 1])
            o, l, ds, top, seen = want(i, lens[i], q[i:i + 1])
            check(got[i:i + 1], got_lse[i:i + 1], o, l, ds, top, seen, False, f"step {step} seq {i}")
            lens[i] += 1
    assert lens[0] <= total


class Captured:
    """Launches recorded on a stream of their own; replay() runs them again there."""

    def __init__(self, gpu, launches):
        self.hip, self.gpu = C.CDLL("libamdhip64.so"), gpu
        self.stream, graph, self.exec = C.c_void_p(), C.c_void_p(), C.c_void_p()
        self._ok(self.hip.hipStreamCreateWithFlags(C.byref(self.stream), 1))
        _capi.check(gpu.lib.granite_hip_set_stream(self.stream), "set_stream")
        try:
            self._ok(self.hip.hipStreamBeginCapture(self.stream, 0))
            launches()
            self._ok(self.hip.hipStreamEndCapture(self.stream, C.byref(graph)))
        finally:
            _capi.check(gpu.lib.granite_hip_set_stream(None), "set_stream")
        self._ok(self.hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, 0))
        self.graph = graph

    @staticmethod
    def _ok(rc):
        assert rc == 0, f"HIP call failed: {rc}"

    def replay(self):
        self._ok(self.hip.hipGraphLaunch(self.exec, self.stream))
        self._ok(self.hip.hipStreamSynchronize(self.stream))

    def close(self):
        self._ok(self.hip.hipGraphExecDestroy(self.exec))
        self._ok(self.hip.hipGraphDestroy(self.graph))
        self._ok(self.hip.hipStreamDestroy(self.stream))


def test_captured_step_replays(gpu, oracle):
    """A decode step (append, then attention on a workspace of its own) and a second one with another workspace,
    each captured once and replayed while positions, lengths and inputs change in place, with eager work and
    the other graph between the replays: every replay equals the eager call."""
    hq, hkv, d, bs, b = 8, 2, 128, 16, 3
    rng = np.random.default_rng(16)
    lens = np.array([2000, 5, 700], np.int32)
    cos, sin = oracle.rope_table(2100, d, 10000.0)
    dcos, dsin = dev(cos), dev(sin)

    class Step:
        def __init__(self, window):
            cache = self.cache = Cache(rng, [2020, 25, 720], bs, hkv, d, F8E4M3).upload()
            self.pools = list(zip(cache.dev[:4], (cache.k, cache.v, cache.ks, cache.vs)))
            self.inputs = [dev(np.zeros((b, h, d), np.float32)) for h in (hq, hkv, hkv)]
            self.pos, self.n = dev(lens), dev(lens)
            self.out = [dev(np.zeros((b, hq, d), np.float16)), dev(np.zeros((b, hq, d), np.float32)), dev(np.zeros((b, hq), np.float32))]
            form = cache.kwargs()
            form.pop("max_seq")
            self.att = dict(q=self.out[0], q_dtype=F16, out=self.out[1], lse=self.out[2], batch_size=b, num_heads=hq, scale=d ** -0.5,
                            block_tables=cache.dev[4], seq_lens=self.n, window=window, num_sinks=4, max_blocks_per_seq=cache.max_blocks, **form)
            for name in ("kv_dtype", "num_kv_heads", "head_dim"):
                form.pop(name)
            self.app = dict(seq_len=b, head_dim=d, src_dtype=F32, q=self.inputs[0], q_out=self.out[0], num_heads_q=hq, k=self.inputs[1],
                            v=self.inputs[2], num_heads_k=hkv, positions=self.pos, table_stride=cache.max_blocks, cos_table=dcos,
                            sin_table=dsin, table_positions=2100, block_table=cache.dev[4], max_blocks_per_seq=cache.max_blocks, **form)
            need = gpu.decode_attention_ex(**self.att, query_workspace=True)
            self.ws = dev(np.zeros(max(need, 256), np.uint8))

        def launch(self):
            gpu.rope_append_q8(**self.app)
            gpu.decode_attention_ex(**self.att, workspace=self.ws)

        def state(self):
            return [x.read(y.dtype, y.shape) for x, y in self.pools]

        def outputs(self):
            return [x.read(t, s) for x, t, s in zip(self.out, (np.float16, np.float32, np.float32), ((b, hq, d), (b, hq, d), (b, hq)))]

        def restore(self, state):
            for (x, _), y in zip(self.pools, state):
                x.write(y)
            for x in self.out:
                x.fill(0)

    steps = [Step(0), Step(600)]
    for s in steps:  # kernels loaded before anything is recorded
        s.launch()
    gpu.sync()
    graphs = [Captured(gpu, s.launch) for s in steps]
    for i in range(4):
        before = []
        for s in steps:
            for x in s.inputs:
                x.write(rng.standard_normal(x.nbytes // 4).astype(np.float32))
            s.pos.write(lens + i)
            s.n.write(lens + i + 1)
            before.append(s.state())
        replayed = []
        for s, g in zip(steps, graphs):
            g.replay()
        for s in steps:
            replayed.append(s.state() + s.outputs())
        for s, old, got in zip(steps, before, replayed):
            s.restore(old)
            s.launch()
            gpu.sync()
            for r, e in zip(got, s.state() + s.outputs()):
                assert np.array_equal(r.view(np.uint8), e.view(np.uint8)), f"replay {i}"
            assert np.isfinite(got[-1]).all() and np.isfinite(got[-2]).all()
    for g in graphs:
        g.close()


def test_another_stream(gpu):
    """A caller's stream gets the launches, in order with what went before on the library's."""
    hip = C.CDLL("libamdhip64.so")
    stream = C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    cache = Cache(np.random.default_rng(17), [5000, 40], 16, 2, 128, F8E4M3).upload()
    want, _ = run_decode(gpu, cache, 8, F16)
    _capi.check(gpu.lib.granite_hip_set_stream(stream), "set_stream")
    try:
        got, _ = run_decode(gpu, cache, 8, F16)
        run_prefill(gpu, cache, 40, 4960, 8, F16, F16, window=300, sinks=4)
    finally:
        _capi.check(gpu.lib.granite_hip_set_stream(None), "set_stream")
    assert np.array_equal(got, want)
    gpu.sync()
    assert hip.hipStreamDestroy(stream) == 0
