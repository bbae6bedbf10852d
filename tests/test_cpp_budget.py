"""A cache held to a budget through the C++ layer on the GPU: runs the
self-checking binary tests/cpp/test_kv_budget (built by __graft_entry__.build())."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_kv_budget")


@pytest.mark.gpu
def test_budget_selfcheck(gpu):
    """Scored prompts and steps with weights, cuts, blocks reused; refusals."""
    if not os.path.exists(BIN):
        pytest.fail(f"{BIN} not built (run __graft_entry__.build())")
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    print(r.stdout[-4000:])
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr
    assert "PASSED" in r.stdout


def test_budget_binary_links():
    if not os.path.exists(BIN):
        pytest.skip("budget self-check not built in this tree")
    out = subprocess.run(["ldd", BIN], capture_output=True, text=True).stdout
    assert "not found" not in out, out
    assert "libmolot_amd.so" in out
