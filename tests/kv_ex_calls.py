"""Calls of the 8-bit / windowed attention entry points with given queries, and float64 references whose error bound goes
with what a result is made of, sum(p |v|), not with the largest value in the cache."""
from __future__ import annotations

import copy
import functools

import numpy as np

import kv8
from granite_amd import F16, F32, F8E4M3, MASK_CAUSAL
from gpu_util import dev
from test_gpu_kv_ex import Cache


def decode(gpu, cache, q, window=0, sinks=0, scale=None, **more):
    """One step, q [batch, heads, D]; results and log-sum-exps."""
    b, hq, d = q.shape
    out, lse = dev(np.full(q.shape, 7.0, np.float32)), dev(np.full((b, hq), 7.0, np.float32))
    dq, dl = dev(q), dev(np.asarray(cache.lens, np.int32))
    args = dict(q=dq, q_dtype=F16 if q.dtype == np.float16 else F32, out=out, lse=lse, batch_size=b, num_heads=hq,
                scale=d ** -0.5 if scale is None else scale, block_tables=cache.dev[4], seq_lens=dl,
                max_blocks_per_seq=cache.max_blocks, window=window, num_sinks=sinks, **cache.kwargs())
    args.update(more)
    gpu.decode_attention_ex(**args)
    gpu.sync()
    return out.read(np.float32, q.shape), lse.read(np.float32, (b, hq))


def prefill(gpu, cache, q, start, out_dtype, window=0, sinks=0, scale=None, mask=MASK_CAUSAL, cache_len=None, **more):
    """q [queries, heads, D] at positions start ...; results and log-sum-exps [queries, heads]."""
    n, hq, d = q.shape
    odt = np.float16 if out_dtype == F16 else np.float32
    out, lse, dq = dev(np.full(q.shape, 7.0, odt)), dev(np.full((hq, n), 7.0, np.float32)), dev(q)
    args = dict(q=dq, q_dtype=F16 if q.dtype == np.float16 else F32, q_tok_stride=hq * d, q_head_stride=d, out=out,
                out_dtype=out_dtype, out_tok_stride=hq * d, out_head_stride=d, seq_q=n, num_heads=hq,
                scale=d ** -0.5 if scale is None else scale, cache_len=cache.lens[0] if cache_len is None else cache_len,
                block_table=cache.dev[4], mask_mode=mask, start_pos=start, lse=lse, window=window, num_sinks=sinks,
                **cache.kwargs())
    args.update(more)
    gpu.attention_ex(**args)
    gpu.sync()
    return out.read(odt, q.shape), lse.read(np.float32, (hq, n)).T


def reference(cache, seq, q, positions, window, sinks, scale, tiles=False, half=False):
    """out, lse and bounds of both for queries q [n, heads, D] of sequence `seq` at the given positions.

    A score is a float sum of d products of at most (d + 4) 2^-24 of the terms' magnitudes away, one more rounding of
    its own size where it is taken to the log2 domain, and its exponential within 2^-22: a factor 1 +- ds on every
    probability, in the numerator and in the denominator, whose sums of n terms add n 2^-24.  A probability times
    its V scale enters the second product as a half and a half remainder, 2^-22 of itself, at the least 2^-37 (tiles: 2^-25)
    of the largest such product of the row, for a value of at most 448 times the scale.  Half results: the tiles' one
    half 2^-11, and the result's rounding."""
    length = cache.lens[seq]
    (k, v), valid = cache.rows(seq, length)
    vis = kv8.visible(positions, length, window, sinks, valid)
    if cache.bs and cache.kv == F8E4M3:
        entry = np.asarray(cache.table[seq])[np.arange(length) // cache.bs].astype(np.int64)
        vs = np.asarray(cache.vs, np.float64)[np.where(valid, entry, 0)]
    else:
        vs = np.ones((length, cache.hkv))
    q = np.asarray(q, np.float64)
    n, hq, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    group = hq // k.shape[1]
    out, lse = np.zeros((n, hq, d)), np.full((n, hq), -np.inf)
    tol, tol_lse = np.zeros((n, hq, d)), np.zeros((n, hq))
    for i in range(n):
        at = np.nonzero(vis[i])[0]
        if not len(at):
            continue
        for h in range(hq):
            kk, vv, sc = k[at, h // group], v[at, h // group], vs[at, h // group]
            x = kk @ q[i, h] * scale
            m = x.max()
            e = np.exp(x - m)
            p = e / e.sum()
            out[i, h], lse[i, h] = p @ vv, m + np.log(e.sum())
            ds = ((d + 4) * (np.abs(kk) @ np.abs(q[i, h])) * abs(scale) + np.abs(x)) * 2.0 ** -24 + 2.0 ** -22
            rel = p @ ds + 2 * (min(len(at), 4096) * 2.0 ** -24 + 2.0 ** -22)
            assert rel < 0.05, "inputs whose scores float arithmetic cannot tell apart"
            tail = len(at) * 448 * (2.0 ** -25 if tiles else 2.0 ** -37) * (p * sc).max()
            tol[i, h] = (p * ds) @ np.abs(vv) + rel * (p @ np.abs(vv)) + tail
            if half:
                tol[i, h] += 2.0 ** -11 * (p @ np.abs(vv)) + 2.0 ** -11 * np.abs(out[i, h]) + 2.0 ** -25
            tol_lse[i, h] = rel + 2.0 ** -22 * (1 + abs(lse[i, h]))
    return out, lse, tol, tol_lse


def compare(got, got_lse, want, what):
    out, lse, tol, tol_lse = want
    assert np.isfinite(got).all(), f"{what}: not finite at {np.argwhere(~np.isfinite(got))[0]}"
    with np.errstate(invalid="ignore"):
        off, off_lse = np.abs(np.asarray(got, np.float64) - out), np.where(lse == got_lse, 0, np.abs(got_lse - lse))
    bad = np.argwhere(off > tol)
    assert len(bad) == 0, f"{what}: {len(bad)} of {out.size} off, first {bad[0]}: {got[tuple(bad[0])]} for {out[tuple(bad[0])]}, allowed {tol[tuple(bad[0])]}"
    bad = np.argwhere(off_lse > tol_lse)
    assert len(bad) == 0, f"{what}: lse {bad[0]}: {got_lse[tuple(bad[0])]} for {lse[tuple(bad[0])]}"


# (kv, block size, heads, KV heads, head size, lengths, window and sinks, sequences that are looked at): decode steps of the row
# kernel (with and without runs of 16 tokens), of the persistent one over 8-bit pools, and of the one over half pools
STEPS = {
    "rows": (F8E4M3, 16, 8, 2, 128, [700, 33, 600], (0, 0), (0, 1, 2)),
    "rows any block": (F8E4M3, 20, 8, 2, 64, [700, 33, 600], (0, 0), (0, 1, 2)),
    "rows half": (F16, 16, 8, 2, 128, [700, 33, 600], (500, 4), (0, 1, 2)),
    "rows half any block": (F16, 12, 8, 2, 64, [700, 33, 600], (500, 4), (0, 2)),
    "persistent 8-bit": (F8E4M3, 16, 16, 16, 64, [2500, 31, 32, 33] + [600] * 20, (0, 0), (0, 1, 2, 3, 23)),
    "persistent 8-bit 128": (F8E4M3, 64, 32, 8, 128, [2900, 31, 2899, 33] + [300] * 20, (0, 0), (0, 1, 2, 3, 23)),
    "persistent half": (F16, 16, 16, 8, 128, [4000, 31, 3999, 33] + [300] * 12, (3900, 4), (0, 1, 2, 3)),
}
# (kv, block size, heads, KV heads, head size, queries, first position, window and sinks, queries that are looked at, tiles kernel)
RUNS = {
    "rows": (F8E4M3, 16, 8, 2, 128, 5, 595, (0, 0), (0, 1, 4), False),
    "rows any block": (F8E4M3, 5, 8, 2, 64, 5, 595, (0, 0), (0, 1, 4), False),
    "rows half": (F16, 0, 8, 2, 128, 5, 595, (400, 4), (0, 1, 4), False),
    "persistent": (F8E4M3, 48, 16, 2, 128, 3, 8100, (0, 0), (0, 1, 2), False),
    "tiles": (F8E4M3, 16, 96, 1, 64, 420, 480, (0, 0), (0, 33, 34, 419), True),
    "tiles 128": (F8E4M3, 16, 96, 1, 128, 420, 480, (0, 0), (0, 419), True),
    "tiles any block": (F8E4M3, 20, 96, 1, 64, 420, 480, (300, 4), (0, 33, 419), True),
    "tiles half": (F16, 16, 96, 1, 128, 420, 480, (300, 4), (0, 33, 419), True),
    "tiles contiguous": (F16, 0, 96, 1, 64, 420, 480, (300, 4), (0, 419), True),
    "tiles cut": (F8E4M3, 16, 8, 1, 64, 400, 5000, (0, 0), (0, 399), True),
}


@functools.lru_cache(maxsize=20)
def made(kv, bs, hkv, d, lens):
    return Cache(np.random.default_rng(1), lens, bs, hkv, d, kv)


def step_cache(name):
    kv, bs, hq, hkv, d, lens, window, some = STEPS[name]
    return copy.deepcopy(made(kv, bs, hkv, d, tuple(lens))), (len(lens), hq, d), window, some


def run_cache(name):
    kv, bs, hq, hkv, d, n, start, window, some, tiles = RUNS[name]
    return copy.deepcopy(made(kv, bs, hkv, d, (start + n,))), (n, hq, d), start, window, some, tiles


def check_step(gpu, cache, q, window, some, scale=None, what=""):
    got, lse = decode(gpu, cache, q, *window, scale=scale)
    for i in some:
        want = reference(cache, i, q[i:i + 1], [cache.lens[i] - 1], *window, scale)
        compare(got[i:i + 1], lse[i:i + 1], want, f"{what} sequence {i}")
    return got, lse


def check_run(gpu, cache, q, start, window, some, tiles, out_dtype, scale=None, what=""):
    some = np.asarray(some)
    got, lse = prefill(gpu, cache, q, start, out_dtype, *window, scale=scale)
    want = reference(cache, 0, q[some], start + some, *window, scale, tiles=tiles, half=out_dtype == F16)
    compare(got[some], lse[some], want, what)
    return got, lse
