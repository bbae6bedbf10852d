"""Calls of the scored entries at the limits they document: bounds of the lengths,
batches and prompts past a launch's grid or a workspace."""
from __future__ import annotations

import math

import pytest
import torch

import scored_ref as ref
from molot_amd import attn
from molot_amd import lib as _lib

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, sigma=1.0):
    return torch.randn(*shape, device="cuda", generator=g) * sigma


def check_out(got, want, tol):
    assert torch.isfinite(got).all()
    err = float((got.double() - want).abs().max())
    assert err <= tol, f"error {err:.3g}, bound {tol:.3g}"


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("kv,nq,nkv,d", [("f32", 8, 4, 128), ("bf16", 16, 4, 128), ("q8", 16, 4, 128),
                                         ("q8", 8, 4, 256)])
@pytest.mark.parametrize("bound,over", [(64, 1), (64, 7), (65, 3), (301, 2)])
def test_rows_past_the_bound_keep_their_weight(gpu, kv, nq, nkv, d, bound, over, step):
    """Sequences longer than max_seq_len: what lies past it may be left out, and its acc
    is left as it is (a step's new row: set); nothing is read from earlier calls' scores."""
    g, page, B = gen(bound + over), 16, 3
    n = bound + over
    width = (n + page - 1) // page
    table = torch.arange(B * width, dtype=torch.int32).view(B, width)
    x = randn(g, n, nkv, d)
    pools = []
    for _ in range(2):
        pool = ref.make_pages(randn(g, 0, nkv, d), kv, B * width, [], page)
        for b in range(B):
            ref.put_pages(pool, x, kv, table[b].tolist(), page)
        pools.append(pool)
    acc = torch.rand(B * width, nkv, page, device="cuda", generator=g)
    sp = torch.full((B * width, nkv, page), -5, dtype=torch.int32, device="cuda")
    O = torch.empty(B, nq, d, device="cuda")
    new = randn(g, B, nkv, d)
    lens, tb = torch.full((B,), n, dtype=torch.int32, device="cuda"), table.cuda()
    kvd = {"f32": 0, "bf16": 1, "q8": 2}[kv]
    P, S = attn._ptr, attn._stream()
    L = _lib.load()

    def call(q, limit, to):
        if step:
            st = L.molot_hip_decode_step_paged_scored(
                P(q), P(new), P(new), P(pools[0]), P(pools[1]), P(O), P(tb), P(lens), P(None), B, width,
                limit, nq, nkv, d, page, P(None), P(None), 0, 0.0, P(None), 0.1, 0, 0.0, P(None), P(to),
                P(sp), kvd, S)
        else:
            st = L.molot_hip_attn_decode_paged_scored(
                P(q), P(pools[0]), P(pools[1]), P(O), P(tb), P(lens), P(None), B, width, limit, nq, nkv, d,
                page, 0.1, 0, 0.0, P(None), P(to), kvd, S)
        assert st == 0

    call(randn(g, B, nq, d, sigma=900.0), n, acc.clone())  # scores of another size in the workspace
    before = acc.clone()
    call(randn(g, B, nq, d), bound, acc)
    rows = lambda z: z[tb.long()].permute(0, 2, 1, 3).reshape(B, nkv, -1)[:, :, :n]  # noqa: E731
    a, b4, G = rows(acc), rows(before), nq // nkv
    last = n - 1 if step else n
    assert torch.equal(a[:, :, bound:last], b4[:, :, bound:last])
    grown = a[:, :, :bound] - b4[:, :, :bound]
    assert bool((grown >= -1e-6).all()) and float(grown.sum(-1).max()) <= G * (1 + 1e-4)
    if step:
        assert bool((a[:, :, n - 1] >= 0).all()) and float(a[:, :, n - 1].max()) <= G * (1 + 1e-4)
        assert (rows(sp)[:, :, n - 1] == n - 1).all() and (rows(sp)[:, :, :n - 1] == -5).all()


# (kv, nq, nkv, d, m, window, ranges, presplit): past 65536 (row, head group) slots
ROWS = [("bf16", 8, 8, 128, 10000, 8, True, True), ("bf16", 8, 8, 64, 9000, 0, True, False),
        ("f32", 8, 4, 34, 17000, 40, False, False), ("q8", 16, 8, 256, 8300, 30, True, True)]


@pytest.mark.parametrize("kv,nq,nkv,d,m,window,ranges,presplit", ROWS)
def test_prompt_rows_past_a_grid(gpu, kv, nq, nkv, d, m, window, ranges, presplit):
    """Prompts that stream each row's own keys, of more rows than one launch takes: a
    window with key_hi past it, and the pieces switched off."""
    g, scale = gen(m), 1 / math.sqrt(d)
    q = randn(g, m, nq, d, sigma=3.0)
    Kc, K = ref.make_cache(randn(g, m, nkv, d), kv)
    Vc, V = ref.make_cache(randn(g, m, nkv, d), kv)
    i = torch.arange(m, device="cuda")
    lo = hi = None
    start, end = (i - window + 1).clamp(min=0) if window else torch.zeros_like(i), i + 1
    if ranges:
        lo = (i - 50).clamp(min=0).int()
        hi = (i + 20).int()
        start, end = torch.maximum(start, lo.long()), hi.long().clamp(max=m)
    sl = attn.alibi_slopes(nq).cuda()
    O = torch.full((m, nq, d), math.nan, device="cuda")
    attn.set_prefill_presplit(presplit)
    try:
        attn.attn_prefill_scored(q, Kc, Vc, O, nq, nkv, m, m, d, scale, 0, window, 50.0, sl, lo, hi)
    finally:
        attn.set_prefill_presplit(True)
    assert bool(torch.isfinite(O).all())
    part = 65536 // nkv  # (ends of the launches' parts, whatever the heads of a group)
    some = sorted({t for e in (0, part // 2, part, 2 * part, m) for t in range(e - 4, e + 4) if 0 <= t < m})
    some = torch.tensor(some, device="cuda")
    want, _ = ref.attend(q[some], K, V, scale, some, start[some], end[some], 50.0, sl)
    check_out(O[some], want, ref.tolerance(q[some], K, V, scale, 50.0, sl, 100))


def test_weights_of_many_short_sequences(gpu):
    """8200 sequences of 8 KV heads in one launch each: more (sequence, head) pairs than a
    merge takes, and nothing to merge."""
    nq, nkv, d, page, B = 8, 8, 4, 4, 8200
    g = gen(70)
    K, V = (randn(g, B, nkv, page, d) for _ in range(2))
    table = torch.randperm(B, device="cuda", generator=g).int().view(B, 1)
    lens = (torch.arange(B, device="cuda") % 5).int()
    q, O = randn(g, B, nq, d, sigma=3.0), torch.empty(B, nq, d, device="cuda")
    acc = torch.zeros(B, nkv, page, device="cuda")
    attn.attn_decode_paged_scored(q, K.view(B, -1), V.view(B, -1), O, table, lens, None, B, 1, nq, nkv, d,
                                  page, 0.5, 0, 20.0, None, acc)
    kb, vb = (z[table[:, 0].long()].double() for z in (K, V))  # [B][head][slot][d]
    s = 20 * ((q.double()[:, :, None] * kb).sum(-1) * 0.5 / 20).tanh()
    s.masked_fill_(torch.arange(page, device="cuda") >= lens[:, None, None], -math.inf)
    p = torch.nan_to_num(s.softmax(-1))
    tol = ref.tolerance(q[0][None], kb[0].transpose(0, 1), vb[0].transpose(0, 1), 0.5, 20.0, None, page)
    tol = 4 * tol  # (one sequence's largest |q||k| and |V| stand for all: 8200 of 4 elements each)
    check_out(O, (p[..., None] * vb).sum(2), tol)
    assert float((acc[table[:, 0].long()].double() - p).abs().max()) <= tol


@pytest.mark.parametrize("step", [False, True])
def test_weights_of_a_ragged_batch_past_the_workspace(gpu, step):
    """One sequence of a million rows among 39 short ones under 64 heads: the scores of
    40 such sequences would be 10 GiB, what the workspace holds at most is 8."""
    nq, nkv, d, page, B, n = 64, 1, 2, 16, 40, 1 << 20
    g, width = gen(71), n // page
    lens = [17 + b for b in range(B)]
    lens[23] = n
    table = torch.zeros(B, width, dtype=torch.int32)
    at = 0
    for b, m in enumerate(lens):
        k = (m + page - 1) // page
        table[b, :k] = torch.arange(at, at + k, dtype=torch.int32)
        at += k
    K, V = (randn(g, at, page * d) for _ in range(2))
    acc, sp = torch.zeros(at, nkv, page, device="cuda"), torch.zeros(at, nkv, page, dtype=torch.int32,
                                                                     device="cuda")
    q, O = randn(g, B, nq, d), torch.empty(B, nq, d, device="cuda")
    new = [randn(g, B, nkv, d) for _ in range(2)]
    L, tb = torch.tensor(lens, dtype=torch.int32, device="cuda"), table.cuda()
    pos = (L + 4) if step else None
    if step:
        attn.decode_step_paged_scored(q, *new, K, V, O, tb, L, pos, B, width, nq, nkv, d, page, None, 0.7, 0,
                                      50.0, None, acc, sp)
    else:
        attn.attn_decode_paged_scored(q, K, V, O, tb, L, None, B, width, nq, nkv, d, page, 0.7, 0, 50.0,
                                      None, acc)
    for b in (0, 22, 23, 24, B - 1):
        m = lens[b]
        blk = tb[b, :(m + page - 1) // page].long()
        Kb, Vb = (z[blk].view(-1, nkv, d)[:m].double() for z in (K, V))
        if step:
            assert torch.equal(Kb[-1].float(), new[0][b]) and torch.equal(Vb[-1].float(), new[1][b])
            assert int(sp[blk[-1], 0, (m - 1) % page]) == m + 4
        end = torch.tensor([m], device="cuda")
        want, p = ref.attend(q[b:b + 1], Kb, Vb, 0.7, end - 1, end * 0, end, 50.0)
        tol = ref.tolerance(q[b:b + 1], Kb, Vb, 0.7, 50.0, None, m)
        check_out(O[b], want[0], tol)
        got = acc[blk].view(-1)[:m].double()
        # (a head's weights each to the bound of an output of V = 1; 64 of them)
        one = ref.tolerance(q[b:b + 1], Kb, torch.ones_like(Vb), 0.7, 50.0, None, m)
        assert float((got - p[0].sum(0)).abs().max()) <= nq * one


def test_empty_and_partial_batches(gpu):
    """No sequence: nothing to do.  Lengths and tables of more sequences than the batch's
    are not looked at past it."""
    nq, nkv, d, page, width = 4, 2, 8, 4, 2
    K, V = (torch.randn(4, nkv * page * d, device="cuda") for _ in range(2))
    acc, sp = torch.zeros(4, nkv, page, device="cuda"), torch.zeros(4, nkv, page, dtype=torch.int32, device="cuda")
    lens = torch.tensor([5, -1], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1], [99, 0]], dtype=torch.int32, device="cuda")
    q, new = torch.randn(1, nq, d, device="cuda"), torch.randn(1, nkv, d, device="cuda")
    for B in (0, 1):
        O = torch.full((1, nq, d), 7.0, device="cuda")
        attn.attn_decode_paged(q, K, V, O, table, lens, None, B, width, nq, nkv, d, page, 0.3)
        O2 = torch.full((1, nq, d), 7.0, device="cuda")
        attn.attn_decode_paged_scored(q, K, V, O2, table, lens, None, B, width, nq, nkv, d, page, 0.3, acc=acc)
        assert bool((O == 7).all()) == (B == 0) and float((O - O2).abs().max()) < 1e-6
        attn.decode_step_paged_scored(q.clone(), new, new, K, V, O, table, lens, None, B, width, nq, nkv, d,
                                      page, None, 0.3, acc=acc, slot_pos=sp)
        attn.kv_track_paged(acc, sp, table, lens, None, B, width, 3, nkv, page)
        attn.kv_evict_paged(K, V, acc, sp, table, lens, None, B, width, nkv, d, page, 4, 1)
    assert torch.isfinite(O).all()


@pytest.mark.parametrize("kv,nq,nkv,d", [("f32", 8, 4, 128), ("bf16", 16, 4, 128), ("q8", 16, 4, 128),
                                         ("q8", 8, 4, 256), ("f32", 6, 2, 34)])
def test_paged_step_outside_its_window(gpu, kv, nq, nkv, d):
    """New rows outside the windows of their positions, beside others inside: appended,
    o = 0, their acc 0 and their positions kept."""
    page, window, lens, pos = 16, 9, (40, 1, 17, 300, 33), (48, 9, 25, 400, 33)
    B, width = len(lens), (max(lens) + page - 1) // page
    g = gen(72)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(3)).int().view(B, width)
    pools = [ref.make_pages(randn(g, 0, nkv, d), kv, B * width, [], page) for _ in range(2)]
    for pool in pools:
        for b, n in enumerate(lens):
            ref.put_pages(pool, randn(g, n, nkv, d), kv, table[b].tolist(), page)
    acc = torch.rand(B * width, nkv, page, device="cuda", generator=g)
    sp = torch.full((B * width, nkv, page), -5, dtype=torch.int32, device="cuda")
    before, tb = acc.clone(), table.cuda()
    q, O = randn(g, B, nq, d), torch.full((B, nq, d), 7.0, device="cuda")
    new = [randn(g, B, nkv, d) for _ in range(2)]
    L, P = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lens, pos))
    attn.decode_step_paged_scored(q, *new, *pools, O, tb, L, P, B, width, nq, nkv, d, page, None, 0.1, window,
                                  50.0, None, acc, sp)
    rows = lambda z, b: z[tb[b].long()].permute(1, 0, 2).reshape(nkv, -1)[:, :lens[b]]  # noqa: E731
    for b, (n, p) in enumerate(zip(lens, pos)):
        a, a0, s = rows(acc, b), rows(before, b), rows(sp, b)
        assert (s[:, -1] == p).all() and (s[:, :-1] == -5).all()
        inside = p - window + 1 < n  # the window still holds slot n - 1
        assert bool((O[b] != 0).any()) == inside
        first = max(0, p - window + 1)
        assert torch.equal(a[:, :min(first, n - 1)], a0[:, :min(first, n - 1)])
        G = nq // nkv
        grown = a[:, -1] + (a[:, :-1] - a0[:, :-1]).sum(-1)  # (fp32 sums of at most 9 rows of weights up to G)
        assert float((grown - (G if inside else 0)).abs().max()) <= (2e-5 * G if inside else 0.0)


def test_plain_prompt_rows_past_a_grid(gpu):
    """The same path without scores, at a head dim that no prefill kernel tiles."""
    nq, nkv, d, m = 8, 4, 34, 17000
    g, scale = gen(73), 1 / math.sqrt(d)
    q = randn(g, m, nq, d, sigma=3.0)
    Kc, K = ref.make_cache(randn(g, m, nkv, d), "f32")
    Vc, V = ref.make_cache(randn(g, m, nkv, d), "f32")
    O = torch.full((m, nq, d), math.nan, device="cuda")
    attn.set_prefill_presplit(False)
    try:
        attn.attn_prefill_gqa(q, Kc, Vc, O, nq, nkv, m, m, d, scale, 0)
    finally:
        attn.set_prefill_presplit(True)
    assert bool(torch.isfinite(O).all())
    some = torch.tensor([0, 1, 16383, 16384, 16385, m - 1], device="cuda")
    want, _ = ref.attend(q[some], K, V, scale, some, torch.zeros_like(some), some + 1)
    check_out(O[some], want, ref.tolerance(q[some], K, V, scale, 0.0, None, m))
