"""The C++ host layer over 8-bit pools (granite_amd/host/tests/host_kv8_test.cpp, built by granite_amd.build)."""
import subprocess
from pathlib import Path

import pytest

BIN = Path(__file__).resolve().parents[1] / "granite_amd" / "bin" / "host_kv8_test"


@pytest.mark.gpu
def test_host_layer_kv8_cases():
    assert BIN.exists(), f"{BIN} is missing: run `python -m granite_amd.build` first"
    res = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "0 failed checks" in res.stdout, res.stdout[-3000:] + res.stderr[-1000:]
