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
