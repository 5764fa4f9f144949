"""Numpy side of the 8-bit cache and windowed attention tests: the e4m3 format, the block scales and the
attention, in float64 and from their definitions."""
from __future__ import annotations

import numpy as np


def _e4m3_values() -> np.ndarray:
    code = np.arange(256)
    sign, e, m = np.where(code & 0x80, -1.0, 1.0), (code >> 3) & 15, code & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[(code & 0x7F) == 0x7F] = np.nan
    return sign * v


E4M3 = _e4m3_values()


def decode8(codes: np.ndarray) -> np.ndarray:
    return E4M3[codes]


def encode8(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 code, ties to even, saturating at 448, NaN kept."""
    x = np.asarray(x, np.float64)
    mag = np.minimum(np.abs(x), 448.0)
    pos = E4M3[:127]
    hi = np.clip(np.searchsorted(pos, np.nan_to_num(mag)), 0, 126)
    lo = np.maximum(hi - 1, 0)
    d_hi, d_lo = pos[hi] - mag, mag - pos[lo]
    code = np.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)
    code = np.where(mag == pos[hi], hi, code)
    code = code | np.where(np.signbit(x), 0x80, 0)
    return np.where(np.isnan(x), 0x7F, code).astype(np.uint8)


def scale_for(top: float) -> float:
    e = -96
    while e < 120 and top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append8(x, pool, scale, table, start, bs, num_blocks):
    """Appends x [n, H, D] (float32 values) to one sequence, in place: the blocks one after another."""
    n = x.shape[0]
    i = 0
    while i < n:
        p = start + i
        take = min(bs - p % bs, n - i)
        block, row = int(table[p // bs]), p % bs
        fresh = x[i:i + take].astype(np.float64)
        i += take
        if not 0 <= block < num_blocks:
            continue
        lo = block * bs
        for h in range(x.shape[1]):
            finite = np.abs(fresh[:, h][np.isfinite(fresh[:, h])])
            need = scale_for(float(finite.max(initial=0.0)))
            old = float(scale[block, h])
            new = max(old, need) if row else need
            if row and new > old:
                pool[lo:lo + row, h] = encode8(decode8(pool[lo:lo + row, h]) * (old / new))
            pool[lo + row:lo + row + take, h] = encode8(fresh[:, h] / new)
            scale[block, h] = new


def rows_of(pool, scale, table, bs, num_blocks, length):
    """[length, H, D] float64 of one sequence, and which tokens lie in a block of the pool."""
    at = np.arange(length)
    entry = np.asarray(table)[at // bs].astype(np.int64)
    valid = (entry >= 0) & (entry < num_blocks)
    entry = np.where(valid, entry, 0)
    rows = entry * bs + at % bs
    if pool.dtype == np.uint8:
        return decode8(pool[rows]) * np.asarray(scale, np.float64)[entry][:, :, None], valid
    return pool[rows].astype(np.float64), valid


def visible(positions, length, window, sinks, valid=None, causal=True):
    p, k = np.asarray(positions)[:, None], np.arange(length)[None]
    v = k <= p if causal else np.ones((len(p), length), bool)
    if window:
        v = v & ((k > p - window) | (k < sinks))
    return v if valid is None else v & valid[None]


def attend(q, k, v, vis, scale):
    """q [n, Hq, D], k and v [T, Hkv, D], vis [n, T].  Keys a query does not see take no part at all, whatever they
    hold.  Returns out, lse and, per (query, head), a bound on what float arithmetic may change a score by."""
    q = np.asarray(q, np.float64)
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out, lse, ds = np.zeros((n, hq, d)), np.full((n, hq), -np.inf), np.zeros((n, hq))
    patterns, which = np.unique(vis, axis=0, return_inverse=True)
    which = np.asarray(which).reshape(-1)
    for i, pattern in enumerate(patterns):
        at, rows = np.nonzero(pattern)[0], np.nonzero(which == i)[0]
        if not len(at):
            continue
        for h in range(hq):
            kk, vv, qq = k[at, h // group], v[at, h // group], q[rows, h]
            s = qq @ kk.T * scale
            m = s.max(1, keepdims=True)
            e = np.exp(s - m)
            z = e.sum(1, keepdims=True)
            out[rows, h], lse[rows, h] = (e / z) @ vv, (m + np.log(z))[:, 0]
            # products of d terms accumulated in float (d roundings of at most 2^-24 of the terms'
            # magnitudes), the scale and the change of base rounded once each, exp2 within 2^-22
            ds[rows, h] = (d + 4) * 2.0 ** -24 * (np.abs(qq) @ np.abs(kk).T).max(1) * abs(scale) + 2.0 ** -22
    return out, lse, ds


def bounds(out, lse, ds, v_top, tokens, half):
    """How far results may be from attend()'s.  A score off by ds changes a probability by a factor 1 +- ds, the
    sums of up to `tokens` terms add at most tokens * 2^-24; numerator and denominator both, on values of at most
    v_top.  The probabilities' half and remainder keep 2^-22 of them.  With half output they are rounded to half
    (half a step, 2^-11) in the numerator and the result once more."""
    rel = 2 * (ds + min(tokens, 4096) * 2.0 ** -24 + 2.0 ** -22)
    o = rel[..., None] * v_top
    if half:
        o = o + 2.0 ** -11 * v_top + 2.0 ** -11 * np.abs(out) + 2.0 ** -25
    return o, rel + 2.0 ** -22 * (1 + np.abs(np.where(np.isfinite(lse), lse, 0)))
