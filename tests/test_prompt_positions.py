"""Prompts whose positions or slots would pass 2^31: refused before any launch (no GPU)."""
import ctypes
import os

import pytest

from molot_amd import lib as _lib

if not os.path.exists(_lib.LIB_PATH):
    pytest.skip("native library not built", allow_module_level=True)

_buf = (ctypes.c_char * 4096)()
P = ctypes.c_void_p((ctypes.addressof(_buf) + 63) & ~63)
N = ctypes.c_void_p(None)
TOP = 2 ** 31 - 1


def plain(pos0, slot0, M):
    return _lib.load().molot_hip_attn_prefill_gqa(P, P, P, P, 8, 4, M, 9, 64, 1.0, pos0, 0, 0, N)


def scored(pos0, slot0, M):
    return _lib.load().molot_hip_attn_prefill_scored(P, P, P, P, 8, 4, M, 9, 64, 1.0, pos0, 0, 50.0, N, N, N,
                                                     0, N)


def plain_step(pos0, slot0, M):
    return _lib.load().molot_hip_prefill_step(P, P, P, P, P, P, 8, 4, 64, M, slot0, pos0, N, N, 0, 0.0, N,
                                              1.0, 0, 0, N)


def scored_step(pos0, slot0, M):
    return _lib.load().molot_hip_prefill_step_scored(P, P, P, P, P, P, 8, 4, 64, M, slot0, pos0, N, N, 0, 0.0,
                                                     N, 1.0, 0, 50.0, N, N, N, 0, N)


def queries(pos0, slot0, M):
    return _lib.load().molot_hip_prefill_q(P, 8, 64, M, pos0, P, 0.0, N, N)


@pytest.mark.parametrize("entry", [plain, scored, plain_step, scored_step, queries])
def test_positions_past_an_int(entry):
    for pos0, M in ((TOP, 1), (TOP - 3, 4), (TOP - 69999, 70000)):
        assert entry(pos0, 0, M) == _lib.EINVAL
    assert entry(TOP, 0, 0) == 0


@pytest.mark.parametrize("entry", [plain_step, scored_step])
def test_slots_past_an_int(entry):
    assert entry(0, TOP - 3, 4) == _lib.EINVAL
