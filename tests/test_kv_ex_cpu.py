"""CPU-side checks of the 8-bit / windowed attention entry points: the arithmetic that decides which keys are
visited, and every refusal.  Arguments are checked before the device is asked for, so a call that is refused
answers with its reason here too, and one that would run answers ENOTINIT (or does nothing: the sizes here are
zero where everything else is right)."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from granite_amd import _capi
from granite_amd._capi import (EINVAL, ENOTINIT, ENULL, EOVERFLOW, EUNSUPPORTED, F16, F32, F8E4M3, MASK_CAUSAL,
                               MASK_NONE, MASK_TREE, OK)

ROOT = Path(__file__).resolve().parent.parent
P = 1 << 20  # a pointer that is only tested


def host_test(tmp_path, name):
    exe = tmp_path / name
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-I", str(ROOT / "granite_amd" / "csrc"),
                    str(ROOT / "granite_amd" / "host" / "tests" / f"{name}.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip().endswith("ok"), out.stdout


def test_visible_tiles_against_single_keys(tmp_path):
    host_test(tmp_path, "kv_visible_test")


def test_choice_of_kernel(tmp_path):
    host_test(tmp_path, "kv_choice_test")


def decode(form=(), **changes):
    a = dict(q=P, q_dtype=F16, k_cache=P, v_cache=P, block_tables=P, seq_lens=P, out=P, lse=None, batch_size=0,
             num_heads=8, num_kv_heads=2, head_dim=128, block_size=16, max_blocks_per_seq=4, scale=1.0)
    a.update(changes)
    f = dict(kv_dtype=F8E4M3, k_scale=P, v_scale=P, num_blocks=8)
    f.update(form)
    return _capi.load().granite_hip_decode_attention_ex(C.byref(_capi.DecodeArgs(**a)), C.byref(_capi.KvForm(**f)), None, 0)


def prefill(form=(), **changes):
    a = dict(q=P, q_dtype=F16, q_tok_stride=1024, q_head_stride=128, out=P, out_dtype=F16, out_tok_stride=1024,
             out_head_stride=128, k_cache=P, v_cache=P, block_table=P, block_size=16, cache_len=64, seq_q=0,
             mask_mode=MASK_CAUSAL, num_heads=8, num_kv_heads=2, head_dim=128, scale=1.0)
    a.update(changes)
    f = dict(kv_dtype=F8E4M3, k_scale=P, v_scale=P, num_blocks=8)
    f.update(form)
    return _capi.load().granite_hip_attention_ex(C.byref(_capi.AttentionArgs(**a)), C.byref(_capi.KvForm(**f)), None, 0)


def append(**changes):
    a = dict(q=P, q_out=2 * P, k=P, v=P, src_dtype=F32, q_out_dtype=F16, k_cache=P, v_cache=P, k_scale=P, v_scale=P,
             block_table=P, freq_base=10000.0, num_heads_q=8, num_heads_k=2, seq_len=0, head_dim=128, block_size=16,
             num_blocks=8, max_blocks_per_seq=4)
    a.update(changes)
    return _capi.load().granite_hip_rope_append_q8(C.byref(_capi.RopeQ8Args(**a)))


def test_accepted_calls_reach_the_device():
    window = dict(kv_dtype=F16, k_scale=None, v_scale=None, window=5, num_sinks=4)
    for rc in (decode(), decode(window), decode(dict(window, num_blocks=0), block_tables=None, max_seq=9), prefill(),
               prefill(window), prefill(mask_mode=MASK_NONE), append(), append(q=None, q_out=None),
               append(k=None, v=None, block_table=None), append(positions=P, table_stride=4)):
        assert rc in (ENOTINIT, OK)


@pytest.mark.parametrize("want,call", [
    (ENULL, lambda: decode(q=None)), (ENULL, lambda: decode(k_cache=None)), (ENULL, lambda: decode(v_cache=None)),
    (ENULL, lambda: decode(out=None)), (ENULL, lambda: decode(dict(k_scale=None))),
    (ENULL, lambda: decode(dict(v_scale=None))),
    (EUNSUPPORTED, lambda: decode(head_dim=96)), (EUNSUPPORTED, lambda: decode(block_tables=None, max_seq=64)),
    (EINVAL, lambda: decode(num_heads=7)), (EINVAL, lambda: decode(num_kv_heads=0)), (EINVAL, lambda: decode(q_dtype=2)),
    (EINVAL, lambda: decode(dict(kv_dtype=F32))), (EINVAL, lambda: decode(dict(kv_dtype=3))),
    (EINVAL, lambda: decode(block_size=0)), (EINVAL, lambda: decode(dict(num_blocks=0))),
    (EINVAL, lambda: decode(max_blocks_per_seq=0)), (EINVAL, lambda: decode(k_cache=P + 8)),
    (EINVAL, lambda: decode(q=P + 4)), (EINVAL, lambda: decode(out=P + 4)),
    (EINVAL, lambda: decode(dict(num_blocks=1 << 31))), (EINVAL, lambda: decode(max_blocks_per_seq=1 << 30)),
    (EINVAL, lambda: decode(seq_lens=None)), (EINVAL, lambda: decode(seq_lens=None, fixed_seq_len=65)),
    (EINVAL, lambda: decode(dict(kv_dtype=F16, window=3), block_tables=None, max_seq=0)),
    (EINVAL, lambda: decode(dict(kv_dtype=F16, window=3), block_tables=None, max_seq=8, batch_size=2)),
])
def test_decode_refusals(want, call):
    assert call() == want


@pytest.mark.parametrize("want,call", [
    (ENULL, lambda: prefill(q=None)), (ENULL, lambda: prefill(out=None)), (ENULL, lambda: prefill(k_cache=None)),
    (ENULL, lambda: prefill(dict(k_scale=None))), (EUNSUPPORTED, lambda: prefill(head_dim=80)),
    (EUNSUPPORTED, lambda: prefill(block_table=None, max_seq=64)), (EUNSUPPORTED, lambda: prefill(mask_mode=MASK_TREE)),
    (EUNSUPPORTED, lambda: prefill(extra_len=4)), (EUNSUPPORTED, lambda: prefill(dict(window=4), mask_mode=MASK_NONE)),
    (EINVAL, lambda: prefill(mask_mode=9)), (EINVAL, lambda: prefill(cache_len=0)), (EINVAL, lambda: prefill(num_heads=7)),
    (EINVAL, lambda: prefill(out_dtype=F8E4M3)), (EINVAL, lambda: prefill(q_dtype=F8E4M3)),
    (EINVAL, lambda: prefill(q_tok_stride=1023)), (EINVAL, lambda: prefill(out_head_stride=4)),
    (EINVAL, lambda: prefill(block_size=0)), (EINVAL, lambda: prefill(dict(num_blocks=0))),
    (EINVAL, lambda: prefill(start_pos=0xFFFFFFFF)), (EINVAL, lambda: prefill(cache_len=1 << 31)),
    (EINVAL, lambda: prefill(dict(kv_dtype=F16, window=3), block_table=None, max_seq=63)),
])
def test_attention_refusals(want, call):
    assert call() == want


@pytest.mark.parametrize("want,call", [
    (ENULL, lambda: append(q=None, q_out=None, k=None, v=None)), (ENULL, lambda: append(q_out=None)),
    (ENULL, lambda: append(v=None)), (ENULL, lambda: append(k=None)), (ENULL, lambda: append(k_cache=None)),
    (ENULL, lambda: append(v_scale=None)), (ENULL, lambda: append(block_table=None)),
    (ENULL, lambda: append(cos_table=P)), (EUNSUPPORTED, lambda: append(head_dim=32)),
    (EINVAL, lambda: append(src_dtype=F8E4M3)), (EINVAL, lambda: append(q_out_dtype=F8E4M3)),
    (EINVAL, lambda: append(num_heads_q=0)), (EINVAL, lambda: append(num_heads_k=0)),
    (EINVAL, lambda: append(freq_base=0.0)),
    (EINVAL, lambda: append(block_size=0)), (EINVAL, lambda: append(num_blocks=0)),
    (EINVAL, lambda: append(max_blocks_per_seq=0)), (EINVAL, lambda: append(k=P + 4)), (EINVAL, lambda: append(q_out=P + 8)),
    (EINVAL, lambda: append(start_pos=0x7FFFFFFF, seq_len=1)), (EINVAL, lambda: append(num_blocks=1 << 31)),
    (EINVAL, lambda: append(positions=P, seq_len=2, table_stride=3)),
    (EOVERFLOW, lambda: append(seq_len=65)), (EOVERFLOW, lambda: append(start_pos=60, seq_len=5)),
    (EOVERFLOW, lambda: append(cos_table=P, sin_table=P, table_positions=9, seq_len=10)),
])
def test_append_refusals(want, call):
    assert call() == want


def test_q_in_place_needs_one_type():
    """Half output over float input would overlap rows that are still to be read."""
    assert append(q=P, q_out=P, src_dtype=F32, q_out_dtype=F16) == EINVAL
    assert append(q=P, q_out=P, src_dtype=F32, q_out_dtype=F32) in (ENOTINIT, OK)


def test_null_structures():
    lib = _capi.load()
    assert lib.granite_hip_decode_attention_ex(None, None, None, 0) == ENULL
    assert lib.granite_hip_attention_ex(None, None, None, 0) == ENULL
    assert lib.granite_hip_rope_append_q8(None) == ENULL
    assert lib.granite_hip_decode_ex_workspace_required(None, None, None) == ENULL
    assert lib.granite_hip_attention_ex_workspace_required(None, None, None) == ENULL


def test_new_structures_match_the_header():
    import re
    text = (ROOT / "include" / "granite_hip.h").read_text()
    for cname, cls in (("granite_hip_kv_form", _capi.KvForm), ("granite_hip_rope_q8_args", _capi.RopeQ8Args)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [part.strip().split()[-1].lstrip("*") for d in body.split(";") if d.strip() for part in d.strip().split(",")]
        assert fields == [f[0] for f in cls._fields_], cname


@pytest.mark.parametrize("cls", [_capi.DecodeArgs, _capi.AttentionArgs, _capi.KvForm, _capi.RopeQ8Args])
def test_packed_arguments_are_the_structures(cls):
    """HipCompute hands these structures over as bytes."""
    block = _capi.packed(cls)
    plain = [(0.5 if t is C.c_float else 3 * i + 1) for i, (_, t) in enumerate(cls._fields_)]
    odd = [(-2.5 if t is C.c_float else -1) for _, t in cls._fields_]  # wraps where a field has no sign
    for values in (plain, odd):
        got, want = cls.from_buffer_copy(block(*values)), cls(*values)
        assert [getattr(got, n) for n, _ in cls._fields_] == [getattr(want, n) for n, _ in cls._fields_]


def test_more_rows_than_an_index_holds_are_refused():
    assert prefill(seq_q=1 << 30, num_heads=8, num_kv_heads=2) == EINVAL
    assert prefill(seq_q=0, num_heads=8, num_kv_heads=2) in (ENOTINIT, OK)
