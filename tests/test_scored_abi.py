"""Refusals of the scored and the budget entries: all before any launch, so they
run without a GPU.  Pointers are of host memory that is never read."""
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
ODD = ctypes.c_void_p(_at + 4)
N = ctypes.c_void_p(None)
F32, BF16, Q8 = 0, 1, 2
NAN, INF = float("nan"), float("inf")


def decode(Q=P, K=P, V=P, O=P, nq=8, nkv=4, n=10, d=64, scale=1.0, pos=9, window=0, cap=50.0, slopes=N,
           acc=N, acc_cap=0, kv=F32):
    return _lib.load().molot_hip_attn_decode_scored(Q, K, V, O, nq, nkv, n, d, scale, pos, window, cap,
                                                    slopes, acc, acc_cap, kv, N)


def step(q=P, k=P, v=P, K=P, V=P, O=P, nq=8, nkv=4, d=64, slot=3, pos=3, eps=0.0, cap=50.0, acc=N,
         slot_pos=N, acc_cap=0, kv=F32):
    return _lib.load().molot_hip_decode_step_scored(q, k, v, K, V, O, nq, nkv, d, slot, pos, N, N, 0, eps,
                                                    N, 1.0, 0, cap, N, acc, slot_pos, acc_cap, kv, N)


def paged(table=P, lens=P, B=2, max_blocks=4, max_len=30, page=16, cap=50.0, acc=N, nkv=4, d=64, kv=F32):
    return _lib.load().molot_hip_attn_decode_paged_scored(P, P, P, P, table, lens, N, B, max_blocks,
                                                          max_len, 8, nkv, d, page, 1.0, 0, cap, N, acc,
                                                          kv, N)


def paged_step(k=P, acc=N, slot_pos=N, page=16, cap=50.0, eps=0.0, B=2):
    return _lib.load().molot_hip_decode_step_paged_scored(P, k, P, P, P, P, P, P, N, B, 4, 30, 8, 4, 64,
                                                          page, N, N, 0, eps, N, 1.0, 0, cap, N, acc,
                                                          slot_pos, F32, N)


def prefill(Q=P, K=P, O=P, nq=8, nkv=4, M=5, Nk=9, d=64, pos0=4, cap=50.0, kv=F32):
    return _lib.load().molot_hip_attn_prefill_scored(Q, K, P, O, nq, nkv, M, Nk, d, 1.0, pos0, 0, cap, N, N,
                                                     N, kv, N)


def prefill_paged(row=P, max_blocks=2, page=16, Nk=20, cap=50.0):
    return _lib.load().molot_hip_attn_prefill_paged_scored(P, P, P, P, row, max_blocks, page, 8, 4, 5, Nk,
                                                           64, 1.0, 4, 0, cap, N, N, N, F32, N)


def prefill_step(q=P, M=5, slot0=4, pos0=4, eps=0.0, cap=50.0, d=64, kv=F32):
    return _lib.load().molot_hip_prefill_step_scored(q, P, P, P, P, P, 8, 4, d, M, slot0, pos0, N, N, 0, eps,
                                                     N, 1.0, 0, cap, N, N, N, kv, N)


def prefill_step_paged(row=P, max_blocks=2, page=16, M=5, slot0=4, cap=50.0):
    return _lib.load().molot_hip_prefill_step_paged_scored(P, P, P, P, P, P, row, max_blocks, page, 8, 4,
                                                           64, M, slot0, 4, N, N, 0, 0.0, N, 1.0, 0, cap,
                                                           N, N, N, F32, N)


def track(acc=P, sp=P, nkv=4, n=10, M=3, cap=12):
    return _lib.load().molot_hip_kv_track(acc, sp, nkv, n, M, 9, cap, N)


def track_paged(acc=P, table=P, lens=P, B=2, max_blocks=4, max_len=30, M=3, nkv=4, page=16):
    return _lib.load().molot_hip_kv_track_paged(acc, P, table, lens, N, B, max_blocks, max_len, M, nkv,
                                                page, N)


def evict(K=P, V=P, acc=P, sp=P, nkv=4, n=10, d=64, keep=5, recent=2, cap=12, kv=F32):
    return _lib.load().molot_hip_kv_evict(K, V, acc, sp, nkv, n, d, keep, recent, 9, cap, kv, N)


def evict_paged(K=P, acc=P, sp=P, table=P, lens=P, B=2, max_blocks=4, max_len=30, nkv=4, d=64, page=16,
                keep=5, recent=2, kv=F32):
    return _lib.load().molot_hip_kv_evict_paged(K, P, acc, sp, table, lens, N, B, max_blocks, max_len, nkv,
                                                d, page, keep, recent, kv, N)


EINVAL = [
    (decode, dict(Q=N)), (decode, dict(O=N)), (decode, dict(K=N)), (decode, dict(V=N)),
    (decode, dict(n=-1)), (decode, dict(nq=7)), (decode, dict(nkv=0)), (decode, dict(kv=3)),
    (decode, dict(K=ODD)), (decode, dict(Q=ODD)), (decode, dict(cap=-1.0)), (decode, dict(cap=NAN)),
    (decode, dict(cap=INF)), (decode, dict(cap=1e-31)), (decode, dict(cap=2e30)),
    (decode, dict(acc=P, acc_cap=9)),
    (step, dict(q=N)), (step, dict(k=N)), (step, dict(slot=-1)), (step, dict(eps=-1.0)),
    (step, dict(cap=NAN)), (step, dict(slot_pos=P)), (step, dict(acc=P, acc_cap=3)), (step, dict(O=ODD)),
    (paged, dict(table=N)), (paged, dict(lens=N)), (paged, dict(B=-1)), (paged, dict(max_blocks=0)),
    (paged, dict(max_len=65)), (paged, dict(page=12)), (paged, dict(page=0)), (paged, dict(cap=-2.0)),
    (paged, dict(kv=Q8, nkv=1, page=2)),
    (paged_step, dict(k=N)), (paged_step, dict(slot_pos=P)), (paged_step, dict(cap=INF)),
    (paged_step, dict(eps=NAN)), (paged_step, dict(page=3)),
    (prefill, dict(Q=N)), (prefill, dict(O=N)), (prefill, dict(K=N)), (prefill, dict(M=-1)),
    (prefill, dict(Nk=-1)), (prefill, dict(pos0=-1)), (prefill, dict(cap=NAN)), (prefill, dict(Q=ODD)),
    (prefill, dict(nq=6)), (prefill, dict(kv=9)),
    (prefill_paged, dict(row=N)), (prefill_paged, dict(max_blocks=0)), (prefill_paged, dict(Nk=33)),
    (prefill_paged, dict(cap=-1.0)),
    (prefill_step, dict(q=N)), (prefill_step, dict(M=-1)), (prefill_step, dict(slot0=-1)),
    (prefill_step, dict(pos0=-1)), (prefill_step, dict(eps=INF)), (prefill_step, dict(cap=NAN)),
    (prefill_step_paged, dict(row=N)), (prefill_step_paged, dict(slot0=28)),
    (prefill_step_paged, dict(page=24)), (prefill_step_paged, dict(cap=INF)),
    (track, dict(acc=N)), (track, dict(n=-1)), (track, dict(M=-1)), (track, dict(M=11)),
    (track, dict(cap=9)), (track, dict(nkv=0)),
    (track_paged, dict(acc=N)), (track_paged, dict(table=N)), (track_paged, dict(lens=N)),
    (track_paged, dict(B=-1)), (track_paged, dict(max_len=65)), (track_paged, dict(M=-1)),
    (track_paged, dict(page=6)), (track_paged, dict(nkv=0)),
    (evict, dict(K=N)), (evict, dict(V=N)), (evict, dict(acc=N)), (evict, dict(sp=N)),
    (evict, dict(K=ODD)), (evict, dict(V=ODD)), (evict, dict(keep=-1)), (evict, dict(recent=-1)),
    (evict, dict(n=-1)), (evict, dict(cap=9)), (evict, dict(kv=3)), (evict, dict(nkv=0)),
    (evict_paged, dict(K=N)), (evict_paged, dict(acc=N)), (evict_paged, dict(sp=N)),
    (evict_paged, dict(table=N)), (evict_paged, dict(lens=N)), (evict_paged, dict(B=-1)),
    (evict_paged, dict(page=24)), (evict_paged, dict(max_len=65)), (evict_paged, dict(keep=-1)),
    (evict_paged, dict(recent=-2)), (evict_paged, dict(kv=Q8, nkv=1, page=2)),
    (evict_paged, dict(K=ODD)), (evict_paged, dict(kv=-1)),
]
ENOTSUP = [
    (decode, dict(d=63)), (decode, dict(d=514)), (decode, dict(d=66, kv=Q8)), (prefill, dict(d=0)),
    (prefill_step, dict(d=7)), (prefill_step, dict(M=70000, slot0=0)), (evict, dict(d=63)),
    (evict, dict(d=514)), (evict, dict(d=6, kv=Q8)), (evict_paged, dict(d=1)),
    (evict_paged, dict(B=70000)), (track_paged, dict(B=70000)),
]
NOTHING = [  # nothing to do: no launch either
    (paged, dict(B=0)), (paged_step, dict(B=0)), (prefill, dict(M=0)), (prefill_step, dict(M=0)),
    (track, dict(M=0)), (track_paged, dict(M=0)), (track_paged, dict(B=0)), (evict, dict(keep=10)),
    (evict, dict(keep=50)), (evict, dict(keep=0)), (evict, dict(n=0)), (evict_paged, dict(B=0)),
    (evict_paged, dict(keep=30)), (evict_paged, dict(keep=0)),
]


@pytest.mark.parametrize("status,cases", [(_lib.EINVAL, EINVAL), (_lib.ENOTSUP, ENOTSUP), (0, NOTHING)],
                         ids=["EINVAL", "ENOTSUP", "nothing"])
def test_status(status, cases):
    for fn, kw in cases:
        got = fn(**kw)
        assert got == status, f"{fn.__name__}({kw}): {got}"


def test_alibi_slopes():
    from molot_amd import attn
    assert attn.alibi_slopes(8).tolist() == [2.0 ** -(h + 1) for h in range(8)]
    got = attn.alibi_slopes(12)
    assert got.dtype.is_floating_point and got.tolist() == pytest.approx(
        [2.0 ** (-8 * (h + 1) / 12) for h in range(12)], rel=2.0 ** -23)


def test_document_starts():
    from molot_amd import attn
    assert attn.document_starts([3, 0, 1, 2], 10).tolist() == [10, 10, 10, 13, 14, 14]
    assert attn.document_starts([]).tolist() == []
    with pytest.raises(ValueError):
        attn.document_starts([2, -1])
