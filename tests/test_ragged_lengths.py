"""The longest sequences of the ragged entries, without a GPU (batches of no rows launch
nothing): the kernels' keys, up to 511 past a sequence's last in a tile's look ahead, are 31-bit."""
from __future__ import annotations

import ctypes
import os

import pytest

from molot_amd import lib as _lib

if not os.path.exists(_lib.LIB_PATH):
    pytest.skip("native library not built", allow_module_level=True)

_buf = (ctypes.c_char * 4096)()
_at = (ctypes.addressof(_buf) + 63) & ~63
P, O, N = ctypes.c_void_p(_at), ctypes.c_void_p(_at + 64), ctypes.c_void_p(None)
MOST = 2 ** 31 - 1 - 1024


def attend(most, width, page, T):
    return _lib.load().molot_hip_attn_ragged(P, P, P, O, P, P, P, T, 1, width, 9, most, 8, 4, 64, page, 1.0, 64,
                                             0.0, N, 0, N)


def step(most, width, page, T):
    return _lib.load().molot_hip_step_ragged(P, P, P, P, P, O, P, P, P, P, P, T, 1, width, 9, most, 8, 4, 64,
                                             page, N, N, 0, 0.0, N, 1.0, 64, 0.0, N, 0, N)


@pytest.mark.parametrize("fn", (attend, step))
@pytest.mark.parametrize("page", (1, 16, 128))
def test_lengths_near_31_bits(fn, page):
    width = (2 ** 31 - 1) // page
    for T in (0, 1):
        for most in (MOST + 1, width * page):
            assert fn(most, width, page, T) == _lib.ENOTSUP
    assert fn(MOST, width, page, 0) == 0
    assert fn(0, width, page, 0) == 0
