"""GPU parity of granite_hip_rope_append_q8: the rotation bit for bit as RoPECache::apply's, codes and scales as the
definition in kv8.py, everything else in the pools untouched."""
import numpy as np
import pytest

import kv8
from granite_amd import F16, F32
from gpu_util import dev, say

pytestmark = pytest.mark.gpu
SENT, SENT_SCALE = 0x5A, np.float32(2.0 ** -3)


class Pools:
    def __init__(self, rng, num_blocks, bs, hkv, d, lengths, spare=0):
        """Sequences of `lengths` tokens' room over a shuffled pool; unused rows hold a sentinel."""
        self.bs, self.num_blocks, self.hkv, self.d = bs, num_blocks, hkv, d
        used = [-(-n // bs) for n in lengths]
        order = rng.permutation(num_blocks)[:sum(used)].astype(np.int32)
        self.max_blocks = max(used) + spare
        self.table = np.full((len(lengths), self.max_blocks), -1, np.int32)
        at = 0
        for i, u in enumerate(used):
            self.table[i, :u] = order[at:at + u]
            at += u
        self.k = np.full((num_blocks * bs, hkv, d), SENT, np.uint8)
        self.v = self.k.copy()
        self.ks = np.full((num_blocks, hkv), SENT_SCALE, np.float32)
        self.vs = self.ks.copy()
        self.upload()

    def upload(self):
        self.dev = [dev(x) for x in (self.k, self.v, self.ks, self.vs, self.table)]

    def kwargs(self):
        k, v, ks, vs, table = self.dev
        return dict(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, block_table=table, block_size=self.bs,
                    num_blocks=self.num_blocks, max_blocks_per_seq=self.max_blocks, table_stride=self.max_blocks)

    def check(self, what):
        got = [b.read(x.dtype, x.shape) for b, x in zip(self.dev, (self.k, self.v, self.ks, self.vs))]
        for name, g, w in zip(("K codes", "V codes", "K scales", "V scales"), got, (self.k, self.v, self.ks, self.vs)):
            if g.dtype == np.uint8:  # any NaN code is a NaN
                nan = (w & 0x7F) == 0x7F
                assert np.array_equal(nan, (g & 0x7F) == 0x7F), (what, name, "NaN")
                g, w = np.where(nan, 0, g), np.where(nan, 0, w)
            bad = np.argwhere(g != w)[:1]
            assert len(bad) == 0, f"{what}: {name}: differ, first at {bad[0]}: {g[tuple(bad[0])]} for {w[tuple(bad[0])]}"


def _src(rng, n, h, d, src, spread=1.0):
    x = (rng.standard_normal((n, h, d)) * spread * np.exp(rng.standard_normal((1, h, 1)))).astype(np.float32)
    return x.astype(np.float16) if src == F16 else x


def _check_q(got, want, dtype):
    if dtype == F16:
        assert np.array_equal(got.view(np.uint16), want.astype(np.float16).view(np.uint16))
    else:
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("src,q_out", [(F32, F16), (F16, F32), (F32, F32), (F16, F16)])
@pytest.mark.parametrize("n,start,bs,hq,hkv,d", [
    (1, 0, 16, 8, 2, 128), (1, 15, 16, 4, 4, 64), (1, 16, 16, 8, 2, 128), (16, 0, 16, 6, 3, 64),
    (37, 5, 16, 8, 2, 128), (5, 3, 1, 4, 1, 128), (33, 7, 8, 12, 4, 64), (200, 130, 64, 8, 2, 128),
    (300, 45, 128, 4, 1, 64), (500, 100, 400, 4, 2, 128), (61, 19, 20, 8, 8, 128), (700, 0, 256, 2, 2, 64)])
def test_run(gpu, oracle, n, start, bs, hq, hkv, d, src, q_out):
    say(f"append8 run n={n} start={start} bs={bs} hq={hq} hkv={hkv} d={d} src={src} q_out={q_out}")
    rng = np.random.default_rng(n * 31 + start)
    pools = Pools(rng, -(-(start + n) // bs) + 3, bs, hkv, d, [start + n])
    q, k, v = (_src(rng, n, h, d, src) for h in (hq, hkv, hkv))
    cos, sin = oracle.rope_table(start + n + 2, d, 10000.0)
    rot = [oracle.rope_apply(x.astype(np.float32), start, cos, sin) for x in (q, k)]
    old_k = _src(rng, start, hkv, d, F32, 0.1)
    for x, pool, scale in ((old_k, pools.k, pools.ks), (old_k, pools.v, pools.vs)):
        kv8.append8(x, pool, scale, pools.table[0], 0, bs, pools.num_blocks)
    pools.upload()
    dq, dk, dv, dcos, dsin = dev(q), dev(k), dev(v), dev(cos), dev(sin)
    out = dev(np.zeros((n, hq, d), np.float32 if q_out == F32 else np.float16))
    gpu.rope_append_q8(seq_len=n, head_dim=d, src_dtype=src, q=dq, q_out=out, q_out_dtype=q_out, num_heads_q=hq, k=dk,
                       v=dv, num_heads_k=hkv, start_pos=start, cos_table=dcos, sin_table=dsin,
                       table_positions=len(cos), **pools.kwargs())
    gpu.sync()
    kv8.append8(rot[1], pools.k, pools.ks, pools.table[0], start, bs, pools.num_blocks)
    kv8.append8(v.astype(np.float32), pools.v, pools.vs, pools.table[0], start, bs, pools.num_blocks)
    _check_q(out.read(np.float32 if q_out == F32 else np.float16, (n, hq, d)), rot[0], q_out)
    pools.check("run")


@pytest.mark.parametrize("src", [F32, F16])
@pytest.mark.parametrize("batch,bs,hq,hkv,d", [(1, 16, 8, 2, 128), (7, 16, 12, 3, 64), (64, 20, 8, 8, 128), (33, 1, 4, 2, 64)])
def test_steps_of_a_batch(gpu, oracle, batch, bs, hq, hkv, d, src):
    """Three steps in a row, each token through its own table; values that grow move the scales."""
    say(f"append8 steps batch={batch} bs={bs} hq={hq} hkv={hkv} d={d} src={src}")
    rng = np.random.default_rng(batch + bs)
    lengths = rng.integers(0, 70, batch)
    pools = Pools(rng, int(sum(-(-(n + 4) // bs) for n in lengths)) + 5, bs, hkv, d, [n + 4 for n in lengths], spare=2)
    cos, sin = oracle.rope_table(80, d, 10000.0)
    dcos, dsin = dev(cos), dev(sin)
    for step in range(3):
        q, k, v = (_src(rng, batch, h, d, src, 4.0 ** step) for h in (hq, hkv, hkv))
        pos = (lengths + step).astype(np.int32)
        dpos, dq, dk, dv, out = dev(pos), dev(q), dev(k), dev(v), dev(np.zeros((batch, hq, d), np.float32))
        gpu.rope_append_q8(seq_len=batch, head_dim=d, src_dtype=src, q=dq, q_out=out, q_out_dtype=F32, num_heads_q=hq,
                           k=dk, v=dv, num_heads_k=hkv, positions=dpos, cos_table=dcos, sin_table=dsin,
                           table_positions=80, **pools.kwargs())
        gpu.sync()
        got = out.read(np.float32, (batch, hq, d))
        for b in range(batch):
            rot = [oracle.rope_apply(x[b:b + 1].astype(np.float32), int(pos[b]), cos, sin) for x in (q, k)]
            kv8.append8(rot[1], pools.k, pools.ks, pools.table[b], int(pos[b]), bs, pools.num_blocks)
            kv8.append8(v[b:b + 1].astype(np.float32), pools.v, pools.vs, pools.table[b], int(pos[b]), bs, pools.num_blocks)
            _check_q(got[b:b + 1], rot[0], F32)
        pools.check(f"step {step}")


def test_values_at_the_edges(gpu, oracle):
    """Zeros, subnormals, the largest floats, infinities and NaN; ties of the code; a block of zeros that grows."""
    d, hkv, bs = 64, 2, 16
    rng = np.random.default_rng(5)
    pools = Pools(rng, 6, bs, hkv, d, [3 * bs])
    v = np.zeros((20, hkv, d), np.float32)
    v[0, 0, :8] = [np.inf, -np.inf, np.nan, 1.0, -448.0, 17.0, 18.0, 2.0 ** -9]
    v[1, 1, :4] = [1e-44, -1e-40, 3e-39, 0.0]
    v[16, 0, :6] = [1.6e38, -1e30, 2.0 ** -120, np.nan, 1.0, -0.0]
    v[17, 1, :6] = [448.0, 447.9, 232.0, 248.0, 1.0625, 1.1875]
    k = np.zeros((20, hkv, d), np.float32)  # rotating zeros leaves zeros, some of them negative
    cos, sin = oracle.rope_table(48, d, 10000.0)
    kw = dict(head_dim=d, src_dtype=F32, num_heads_k=hkv, cos_table=dev(cos), sin_table=dev(sin), table_positions=48)
    dk, dv = dev(k), dev(v)
    gpu.rope_append_q8(seq_len=20, k=dk, v=dv, start_pos=0, **kw, **pools.kwargs())
    kv8.append8(oracle.rope_apply(k, 0, cos, sin), pools.k, pools.ks, pools.table[0], 0, bs, 6)
    kv8.append8(v, pools.v, pools.vs, pools.table[0], 0, bs, 6)
    gpu.sync()
    pools.check("edges")
    assert pools.ks[pools.table[0, 0], 0] == np.float32(2.0 ** -96)
    more = np.full((3, hkv, d), 100.0, np.float32)  # grows the second block's scales from the middle
    dm = dev(more)
    gpu.rope_append_q8(seq_len=3, k=dm, v=dm, start_pos=20, **kw, **pools.kwargs())
    rot = oracle.rope_apply(more, 20, cos, sin)
    kv8.append8(rot, pools.k, pools.ks, pools.table[0], 20, bs, 6)
    kv8.append8(more, pools.v, pools.vs, pools.table[0], 20, bs, 6)
    gpu.sync()
    pools.check("grown")


def test_bad_pages_and_positions_store_nothing(gpu, oracle):
    d, hq, hkv, bs = 128, 4, 2, 16
    rng = np.random.default_rng(6)
    pools = Pools(rng, 9, bs, hkv, d, [2 * bs] * 4)
    pools.table[1, 1], pools.table[2, 0], pools.table[3, 0] = -1, 9, 2147483647
    pools.upload()
    cos, sin = oracle.rope_table(40, d, 10000.0)
    pos = np.array([-1, 20, 3, 40, 33, 7], np.int32)  # negative; bad entries; beyond the tables; beyond the table's blocks; good
    table = np.concatenate([pools.table, pools.table[:1], pools.table[:1]])
    table = np.ascontiguousarray(table[[0, 1, 2, 3, 4, 5]])
    q, k, v = (_src(rng, 6, h, d, F32) for h in (hq, hkv, hkv))
    out = dev(np.full((6, hq, d), 9.0, np.float32))
    keep = [dev(x) for x in (q, k, v, pos, cos, sin, table)]
    kw = pools.kwargs()
    kw["block_table"] = keep[6]
    gpu.rope_append_q8(seq_len=6, head_dim=d, src_dtype=F32, q=keep[0], q_out=out, q_out_dtype=F32, num_heads_q=hq,
                       k=keep[1], v=keep[2], num_heads_k=hkv, positions=keep[3], cos_table=keep[4], sin_table=keep[5],
                       table_positions=40, **kw)
    gpu.sync()
    got = out.read(np.float32, (6, hq, d))
    for i in (0, 3):
        assert (got[i] == 9.0).all()
    for i in (1, 2, 4, 5):
        assert np.array_equal(got[i], oracle.rope_apply(q[i:i + 1], int(pos[i]), cos, sin)[0])
    kv8.append8(oracle.rope_apply(k[5:6], 7, cos, sin), pools.k, pools.ks, pools.table[0], 7, bs, 9)
    kv8.append8(v[5:6], pools.v, pools.vs, pools.table[0], 7, bs, 9)
    pools.check("bad pages, steps")
    # a run that crosses a bad page stores the rest
    pools = Pools(rng, 9, bs, hkv, d, [3 * bs])
    pools.table[0, 1] = -5
    pools.upload()
    k, v = _src(rng, 40, hkv, d, F32), _src(rng, 40, hkv, d, F32)
    keep = [dev(k), dev(v), dev(cos), dev(sin)]
    gpu.rope_append_q8(seq_len=40, head_dim=d, src_dtype=F32, k=keep[0], v=keep[1], num_heads_k=hkv, cos_table=keep[2],
                       sin_table=keep[3], table_positions=40, **pools.kwargs())
    gpu.sync()
    kv8.append8(oracle.rope_apply(k, 0, cos, sin), pools.k, pools.ks, pools.table[0], 0, bs, 9)
    kv8.append8(v, pools.v, pools.vs, pools.table[0], 0, bs, 9)
    pools.check("bad pages, run")


def test_rotation_evaluated_on_the_device(gpu):
    """Without tables: an angle of up to 600 rad in float is off by at most 600 * (2^-23 for the product and the
    frequency) and cos, sin by 2^-22 more, so a rotated element by that times the pair's length."""
    n, start, hq, d = 9, 590, 3, 128
    rng = np.random.default_rng(8)
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    out, dq = dev(np.zeros((n, hq, d), np.float32)), dev(q)
    gpu.rope_append_q8(seq_len=n, head_dim=d, src_dtype=F32, q=dq, q_out=out, q_out_dtype=F32, num_heads_q=hq,
                       start_pos=start, freq_base=10000.0)
    gpu.sync()
    ang = (start + np.arange(n))[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = q[..., 0::2].astype(np.float64), q[..., 1::2].astype(np.float64)
    want = np.stack((a * c - b * s, a * s + b * c), -1).reshape(n, hq, d)
    # powf of the frequency: within 16 roundings
    tol = (600 * (16 + 2) * 2.0 ** -24 + 2.0 ** -22) * np.repeat(np.hypot(a, b), 2, -1)
    got = out.read(np.float32, (n, hq, d))
    assert (np.abs(got - want) <= tol).all()


def test_q_in_place(gpu, oracle):
    n, hq, d = 5, 3, 64
    q = np.random.default_rng(1).standard_normal((n, hq, d)).astype(np.float32)
    cos, sin = oracle.rope_table(9, d, 10000.0)
    dq, dc, ds = dev(q), dev(cos), dev(sin)
    gpu.rope_append_q8(seq_len=n, head_dim=d, src_dtype=F32, q=dq, q_out=dq, q_out_dtype=F32, num_heads_q=hq, start_pos=4,
                       cos_table=dc, sin_table=ds, table_positions=9)
    gpu.sync()
    assert np.array_equal(dq.read(np.float32, q.shape), oracle.rope_apply(q, 4, cos, sin))
