"""Refusals of the ragged entries: all before any launch, so they run without a GPU.
Pointers are of host memory that is never read."""
from __future__ import annotations

import ctypes
import os

import pytest

from molot_amd import lib as _lib

if not os.path.exists(_lib.LIB_PATH):
    pytest.skip("native library not built", allow_module_level=True)

_buf = (ctypes.c_char * 4096)()
_at = (ctypes.addressof(_buf) + 63) & ~63
P = ctypes.c_void_p(_at)       # 16-byte aligned
P2 = ctypes.c_void_p(_at + 64)
ODD = ctypes.c_void_p(_at + 4)
N = ctypes.c_void_p(None)
F32, BF16, Q8 = 0, 1, 2
NAN, INF = float("nan"), float("inf")


def plan(counts=P, done=N, pos=N, lens=P, kv=P, table=P, free=P, count=P, left=P, B=2, width=4, page=16,
         num=9, rows=3, start=P, seq=P, rpos=P, slot=P, status=P):
    return _lib.load().molot_hip_ragged_plan(counts, done, pos, lens, kv, table, free, count, left, B,
                                             width, page, num, rows, start, seq, rpos, slot, status, N)


def append(q=P, k=P, v=P, K=P, V=P, pos=P, slot=P, T=3, num=9, nq=8, nkv=4, d=64, page=16, eps=0.0, kv=F32):
    return _lib.load().molot_hip_rope_append_ragged(q, k, v, K, V, pos, slot, T, num, nq, nkv, d, page, N,
                                                    N, 0, eps, N, kv, N)


def attend(Q=P, K=P, V=P, O=P2, table=P, lens=P, start=P, T=3, B=2, width=4, num=9, most=50, nq=8, nkv=4,
           d=64, page=16, cap=0.0, kv=F32):
    return _lib.load().molot_hip_attn_ragged(Q, K, V, O, table, lens, start, T, B, width, num, most, nq,
                                             nkv, d, page, 1.0, 0, cap, N, kv, N)


def step(q=P, k=P, v=P, K=P, V=P, O=P2, table=P, lens=P, start=P, pos=P, slot=P, T=3, B=2, width=4, num=9,
         most=50, nq=8, nkv=4, d=64, page=16, eps=0.0, cap=0.0, kv=F32):
    return _lib.load().molot_hip_step_ragged(q, k, v, K, V, O, table, lens, start, pos, slot, T, B, width,
                                             num, most, nq, nkv, d, page, N, N, 0, eps, N, 1.0, 0, cap, N,
                                             kv, N)


@pytest.mark.parametrize("bad", [
    dict(counts=N), dict(lens=N), dict(kv=N), dict(table=N), dict(start=N), dict(seq=N), dict(rpos=N),
    dict(slot=N), dict(status=N), dict(count=N), dict(left=N), dict(free=N, done=P), dict(B=-1),
    dict(width=0), dict(page=0), dict(page=12), dict(num=0), dict(rows=-1), dict(num=1 << 28),
    dict(width=1 << 28, page=16)])
def test_plan_refusals(bad):
    assert plan(**bad) == _lib.EINVAL


@pytest.mark.parametrize("bad", [dict(B=(1 << 20) + 1), dict(rows=(1 << 20) + 1), dict(width=(1 << 20) + 1)])
def test_plan_sizes(bad):
    assert plan(**bad) == _lib.ENOTSUP


SHAPES = [dict(nq=0), dict(nkv=0), dict(nq=6), dict(kv=3), dict(kv=-1), dict(page=0), dict(page=24),
          dict(num=0), dict(num=1 << 27), dict(kv=Q8, nkv=1, nq=1, page=2), dict(T=-1)]
DIMS = [dict(d=0), dict(d=63), dict(d=514), dict(d=66, kv=Q8), dict(nkv=5000, nq=5000)]


@pytest.mark.parametrize("bad", SHAPES + [
    dict(q=N), dict(pos=N), dict(slot=N), dict(k=N), dict(v=N), dict(K=N), dict(V=N), dict(eps=-1.0),
    dict(eps=NAN), dict(eps=INF)])
def test_append_refusals(bad):
    assert append(**bad) == _lib.EINVAL


@pytest.mark.parametrize("bad", SHAPES + [
    dict(Q=N), dict(K=N), dict(V=N), dict(O=N), dict(table=N), dict(lens=N), dict(start=N), dict(B=-1),
    dict(width=0), dict(most=-1), dict(most=65), dict(width=1 << 28), dict(Q=ODD), dict(K=ODD), dict(V=ODD),
    dict(O=ODD), dict(O=P), dict(cap=-1.0), dict(cap=1e-31), dict(cap=NAN), dict(cap=INF)])
def test_attend_refusals(bad):
    assert attend(**bad) == _lib.EINVAL


@pytest.mark.parametrize("bad", [
    dict(q=N), dict(k=N), dict(v=N), dict(K=N), dict(O=N), dict(O=P), dict(pos=N), dict(slot=N),
    dict(table=N), dict(eps=NAN), dict(cap=NAN), dict(most=65), dict(page=24), dict(kv=3), dict(q=ODD)])
def test_step_refusals(bad):
    assert step(**bad) == _lib.EINVAL


@pytest.mark.parametrize("bad", DIMS)
def test_sizes_the_kernels_are_not_built_for(bad):
    assert append(**bad) == _lib.ENOTSUP
    assert attend(**bad) == _lib.ENOTSUP
    assert step(**bad) == _lib.ENOTSUP


def test_more_rows_than_the_grid():
    assert attend(T=1 << 30, nq=64, nkv=4) == _lib.ENOTSUP
    most = 1 << 20  # rows, and sequences
    for fn in (attend, step):
        assert fn(T=most + 1) == _lib.ENOTSUP and fn(B=most + 1) == _lib.ENOTSUP
        # tiles * KV heads * threads past 2^32
        assert fn(T=most, B=most, nq=64, nkv=64) == _lib.ENOTSUP
    assert append(T=most + 1) == _lib.ENOTSUP


def test_nothing_to_do():
    assert append(T=0) == 0 and append(T=0, k=N, v=N, K=N, V=N) == 0
    assert attend(T=0) == 0 and attend(B=0) == 0 and step(T=0) == 0 and step(B=0) == 0


def test_python_arguments():
    """The Python layer refuses what is not a device tensor, before the library is asked."""
    import torch

    from molot_amd import attn

    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        attn.ragged_plan(i, i, i, i, 2, 2, 16, 4, 4, i, i, i, i, i)
    f = torch.zeros(64)
    with pytest.raises(ValueError, match="device tensor"):
        attn.attn_ragged(f, f, f, f, i, i, i, 1, 1, 1, 1, 1, 1, 1, 64, 16, 1.0)
    with pytest.raises(ValueError, match="go together"):
        attn.rope_append_ragged(f, None, f, None, None, i, i, 1, 1, 1, 1, 64, 16, None)
