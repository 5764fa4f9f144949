"""Which kernel the calls of test_gpu_kv_ex_behind.py go to, from the sizes alone."""
from test_kv_ex_cpu import host_test


def test_calls_without_a_visible_tile(tmp_path):
    host_test(tmp_path, "kv_behind_test")
