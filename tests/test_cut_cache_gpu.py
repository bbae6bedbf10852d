"""Prompts over a cache that rows were evicted from: positions run ahead of the
slots, and a row still sees no row appended after it (64-bit reference over the
rows stored)."""
from __future__ import annotations

import math

import pytest
import torch

import scored_ref as ref
from molot_amd import attn

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# (kv, nq, nkv, d, m, slot0, pos0, window): each prefill kernel, by head dim and by work
STEPS = [
    ("f32", 8, 4, 128, 40, 25, 300, 0),
    ("f32", 8, 4, 128, 40, 25, 30, 0),        # some of the rows behind only
    ("f32", 8, 4, 64, 1, 0, 900, 0),
    ("bf16", 32, 8, 128, 600, 33, 700, 0),    # the pieces
    ("f32", 32, 8, 128, 600, 0, 1, 0),
    ("q8", 32, 8, 128, 600, 70, 5000, 0),
    ("f32", 8, 4, 256, 150, 20, 170, 0),
    ("q8", 8, 4, 256, 65, 10, 400, 0),
    ("bf16", 8, 2, 512, 300, 40, 4000, 0),
    ("f32", 8, 2, 512, 20, 40, 100, 0),       # rows streamed one by one
    ("f32", 6, 2, 34, 50, 9, 200, 0),
    ("f32", 8, 4, 128, 200, 25, 300, 64),     # a window goes by the slots
    ("f32", 8, 4, 256, 150, 90, 400, 64),
]


@pytest.mark.parametrize("presplit", [True, False])
@pytest.mark.parametrize("kv,nq,nkv,d,m,slot0,pos0,window", STEPS)
def test_plain_prompt_is_causal(gpu, kv, nq, nkv, d, m, slot0, pos0, window, presplit):
    g = gen(d + m)
    n, page, scale = slot0 + m, 16, 1 / math.sqrt(d)
    q, k, v = (torch.randn(m, h, d, device="cuda", generator=g) for h in (nq, nkv, nkv))
    x, y = (torch.randn(n, nkv, d, device="cuda", generator=g) for _ in range(2))
    inv = attn.rope_inv_freq(10000.0, d).cuda()
    Kc, Vc = ref.make_cache(x, kv)[0], ref.make_cache(y, kv)[0]
    blocks = (n + page - 1) // page
    table = torch.arange(blocks, dtype=torch.int32).flip(0)
    Kp, Vp = (ref.make_pages(z, kv, blocks, table.tolist(), page) for z in (x, y))
    q1, q2 = q.clone(), q.clone()
    O, Op = (torch.full((m, nq, d), math.nan, device="cuda") for _ in range(2))
    attn.set_prefill_presplit(presplit)
    try:
        attn.prefill_step(q1, k, v, Kc, Vc, O, nq, nkv, d, m, slot0, pos0, inv, scale, window)
        attn.prefill_step_paged(q2, k, v, Kp, Vp, Op, table.cuda(), blocks, page, nq, nkv, d, m, slot0,
                                pos0, inv, scale, window)
    finally:
        attn.set_prefill_presplit(True)
    assert torch.equal(q1, q2)
    K, V = ref.cache_values(Kc, kv, nkv, d), ref.cache_values(Vc, kv, nkv, d)
    i = slot0 + torch.arange(m, device="cuda")
    lo = (i - window + 1).clamp(min=0) if window else torch.zeros_like(i)
    want, _ = ref.attend(q1, K, V, scale, i, lo, i + 1)
    tol = ref.tolerance(q1, K, V, scale, 0.0, None, n)
    for got in (O, Op):
        err = float((got.double() - want).abs().max())
        assert err <= tol, f"error {err:.3g}, bound {tol:.3g}"
