"""granite_hip_rope_append_q8 into large blocks, with few and with many of them: codes and scales against kv8.append8, one
block in pieces (old rows in front, a scale that grows) and runs that end inside a block."""
import numpy as np
import pytest

import kv8
from granite_amd import F16, F32
from gpu_util import dev, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs,n,start,hkv,d", [(64, 500, 17, 4, 128), (128, 700, 100, 4, 128), (96, 333, 5, 3, 128), (256, 900, 37, 2, 128),
                                              (1024, 1500, 1000, 1, 128), (128, 700, 100, 4, 64), (160, 2000, 3, 40, 128), (128, 127, 1, 8, 128)])
@pytest.mark.parametrize("src", [F16, F32])
def test_large_blocks(gpu, bs, n, start, hkv, d, src):
    say(f"append bs={bs} n={n} start={start} hkv={hkv} d={d} src={src}")
    rng = np.random.default_rng(n)
    blocks = -(-(start + n) // bs)
    num_blocks = blocks + 2
    table = rng.permutation(num_blocks)[:blocks].astype(np.int32)
    dt = np.float16 if src == F16 else np.float32
    pools = [np.full((num_blocks * bs, hkv, d), 0x55, np.uint8) for _ in range(2)]
    scales = [np.full((num_blocks, hkv), 2.0 ** -9, np.float32) for _ in range(2)]
    want_pools, want_scales = [p.copy() for p in pools], [s.copy() for s in scales]
    dp, ds, dt_ = [dev(p) for p in pools], [dev(s) for s in scales], dev(table)
    # identity rotation: cos 1, sin 0
    cos, sin = dev(np.ones((start + n, d // 2), np.float32)), dev(np.zeros((start + n, d // 2), np.float32))
    for first, count, gain in ((start, n // 3, 1.0), (start + n // 3, n - n // 3, 40.0)):
        k, v = (rng.standard_normal((2, count, hkv, d)) * gain).astype(dt)
        k[count // 2, 0, 3], v[count - 1, hkv - 1, 5] = np.inf, np.nan
        q = rng.standard_normal((count, 2, d)).astype(dt)
        dk, dv, dq, qo = dev(k), dev(v), dev(q), dev(np.zeros((count, 2, d), np.float32))
        gpu.rope_append_q8(seq_len=count, head_dim=d, src_dtype=src, q=dq, q_out=qo, q_out_dtype=F32, num_heads_q=2, k=dk, v=dv,
                           num_heads_k=hkv, k_cache=dp[0], v_cache=dp[1], k_scale=ds[0], v_scale=ds[1], block_table=dt_, block_size=bs,
                           num_blocks=num_blocks, max_blocks_per_seq=blocks, start_pos=first, cos_table=cos, sin_table=sin,
                           table_positions=start + n)
        gpu.sync()
        assert np.array_equal(qo.read(np.float32, q.shape), q.astype(np.float32))
        with np.errstate(invalid="ignore"):
            kr = k.astype(np.float32)
            kr[count // 2, 0, 2:4] = [np.nan, np.nan]  # (inf * 0 in the rotation's other product)
            kr[count // 2, 0, 3] = np.inf
            kr[count // 2, 0, 2] = np.nan
        for x, pool, scale in ((kr, want_pools[0], want_scales[0]), (v.astype(np.float32), want_pools[1], want_scales[1])):
            kv8.append8(x, pool, scale, table, first, bs, num_blocks)
        for name, got, want in (("K", dp[0].read(np.uint8, pools[0].shape), want_pools[0]), ("V", dp[1].read(np.uint8, pools[1].shape), want_pools[1])):
            nan = (want & 0x7F) == 0x7F
            assert np.array_equal((got & 0x7F) == 0x7F, nan), f"{name}: NaN"
            same = (got == want) | nan | (((got | want) & 0x7F) == 0)  # (the sign of a zero through the rotation's sum)
            assert same.all(), f"{name}: {np.argwhere(~same)[:3]}"
        for name, got, want in (("K", ds[0], want_scales[0]), ("V", ds[1], want_scales[1])):
            assert np.array_equal(got.read(np.float32, want.shape), want), f"{name} scales"
