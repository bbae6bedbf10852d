"""The C++ layer over caches that rows were evicted from, on the GPU: runs the
self-checking binary tests/cpp/test_kv_cut (built by __graft_entry__.build())."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_kv_cut")


@pytest.mark.gpu
def test_cut_selfcheck(gpu):
    """Prompts, steps and shared layers of the turn after an eviction."""
    if not os.path.exists(BIN):
        pytest.fail(f"{BIN} not built (run __graft_entry__.build())")
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    print(r.stdout[-4000:])
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr
    assert "PASSED" in r.stdout
