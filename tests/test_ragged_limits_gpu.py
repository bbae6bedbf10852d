"""Ragged batches at the bounds of their work lists, on the GPU."""
from __future__ import annotations

import math

import pytest
import torch

import ragged_ref as rr
from molot_amd import attn

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def close(got, want, tol):
    assert torch.isfinite(got).all()
    err = float((got.double() - want).abs().max())
    assert err <= tol, f"error {err:.3g}, bound {tol:.3g}"


@pytest.mark.parametrize("B", (2, 400, 4500))
@pytest.mark.parametrize("kv,d", [("f32", 128), ("bf16", 256), ("q8", 64), ("bf16", 512)])
def test_starts_that_do_not_ascend(gpu, kv, d, B):
    """Ranges that overlap come to more tiles than the lists hold for T rows (200 and 2250 of
    64 rows): none is attended, by either entry, and the next call is right."""
    nkv, nq, T, n = 2, 8, 64, 1000
    g = gen(B)
    b = rr.Batch(g, kv, nkv, d, [T], [n - T])
    i32 = dict(dtype=torch.int32, device="cuda")
    table = b.table[:1].expand(B, -1).contiguous()
    lens = torch.full((B,), n, **i32)
    lens[::7] = n - 32  # tiles of several sizes
    q = torch.randn(T, nq, d, device="cuda", generator=g)
    freq = attn.rope_inv_freq(1e4, d).cuda()
    none = torch.full((T,), -1, **i32)
    every = torch.arange(B + 1, device="cuda")
    starts = [torch.where(every % 2 == 0, 0, T), torch.where(every % 2 == 0, -5, 2 ** 31 - 1)]
    down = torch.full((B + 1,), T, device="cuda")
    down[-1] = T - 1  # the last alone
    for start in starts + [down]:
        start = start.to(torch.int32)
        O = torch.full((T, nq, d), math.nan, device="cuda")
        attn.attn_ragged(q, b.K, b.V, O, table, lens, start, T, B, b.width, b.blocks, n, nq, nkv, d, 16, 0.1)
        Q = q.clone()
        attn.step_ragged(Q, None, None, b.K, b.V, O, table, lens, start, none, none, T, B, b.width, b.blocks, n,
                         nq, nkv, d, 16, freq, 0.1)
        torch.cuda.synchronize()
        assert torch.isnan(O).all() and torch.equal(Q, q)
    O = torch.full((T, nq, d), math.nan, device="cuda")
    attn.attn_ragged(q, b.K, b.V, O, *b.args(), nq, nkv, d, 16, 0.1)
    want, tol = b.attend(q, 0.1)
    close(O, want, tol)
