"""Evictions of long caches whose chunks are 8192 slots: more workgroups than the chip
holds at once, and many chunks of one head, against the rule slot by slot."""
from __future__ import annotations

import pytest
import torch

import scored_ref as ref
from molot_amd import attn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["smooth", "ties", "equal", "zeros", "near"])
@pytest.mark.parametrize("nkv,n,keep,recent", [(32, 33000, 24577, 700), (1, 340001, 300001, 5000),
                                               (1, 340000, 4096, 0)])
def test_rule(gpu, nkv, n, keep, recent, kind):
    d, pos = 2, n - 1
    g = torch.Generator(device="cuda")
    g.manual_seed(n + keep)
    rand = lambda: torch.rand(nkv, n, device="cuda", generator=g)  # noqa: E731
    acc = {"smooth": lambda: torch.exp(2 * torch.randn(nkv, n, device="cuda", generator=g)),
           "ties": lambda: (4 * rand()).floor(),
           "equal": lambda: torch.full((nkv, n), 0.25, device="cuda"),
           "zeros": lambda: torch.where(rand() < 0.9, torch.zeros(nkv, n, device="cuda"), rand()),
           "near": lambda: 1 + (4000 * rand()).floor() * 2.0 ** -23}[kind]()
    sp = torch.stack([torch.randperm(n, device="cuda", generator=g) for _ in range(nkv)]).int()
    K, V = (torch.randn(n, nkv * d, device="cuda", generator=g) for _ in range(2))
    want = [x.clone() for x in (K, V, acc, sp)]
    for h, moves in enumerate(ref.evict(acc.cpu(), sp.cpu(), n, keep, recent, pos)):
        if not moves:
            continue
        to, at = (torch.tensor([m[i] for m in moves], device="cuda") for i in (0, 1))
        for x in want[:2]:
            rows = x.view(-1, nkv, d)
            rows[to, h] = rows[at, h]
        for x in want[2:]:
            x[h, to] = x[h, at]
    attn.kv_evict(K, V, acc, sp, nkv, n, d, keep, recent, pos)
    for got, exp in zip((K, V, acc, sp), want):
        assert torch.equal(got, exp)
