"""Scored attention on the GPU: capped scores, distance bias, key ranges and
weights, against 64 bits (tests/scored_ref.py)."""
from __future__ import annotations

import math

import pytest
import torch

import scored_ref as ref
from molot_amd import attn
from molot_amd import lib as _lib

pytestmark = pytest.mark.gpu

KVS = ("f32", "bf16", "q8")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, sigma=1.0):
    return torch.randn(*shape, device="cuda", generator=g) * sigma


def slopes_of(nq):
    return attn.alibi_slopes(nq).cuda()


def rel(got, want):
    top = float(want.abs().max())
    return float((got.double() - want).abs().max()) / (top if top else 1.0)


def check_out(got, want, tol):
    assert torch.isfinite(got).all()
    err = float((got.double() - want).abs().max()) if want.numel() else 0.0
    assert err <= tol, f"error {err:.3g}, bound {tol:.3g}"


# (kv, nq, nkv, d, n, window, softcap, alibi)
DECODE = [
    ("f32", 32, 8, 128, 300, 0, 50.0, False),
    ("f32", 32, 8, 128, 4097, 0, 50.0, True),
    ("f32", 8, 8, 64, 1, 0, 30.0, True),
    ("f32", 8, 8, 64, 2, 0, 0.0, True),
    ("f32", 6, 2, 34, 65, 0, 5.0, True),
    ("f32", 12, 4, 96, 1025, 0, 50.0, True),
    ("f32", 8, 4, 256, 2500, 1024, 50.0, False),
    ("f32", 8, 2, 512, 777, 0, 20.0, True),
    ("f32", 16, 1, 128, 513, 100, 0.0, True),
    ("bf16", 64, 8, 128, 5000, 0, 0.0, True),
    ("bf16", 32, 8, 128, 33, 0, 50.0, True),
    ("bf16", 16, 1, 64, 2049, 0, 30.0, False),
    ("bf16", 3, 1, 64, 31, 7, 30.0, True),
    ("bf16", 8, 4, 256, 2500, 1024, 50.0, True),
    ("bf16", 8, 2, 512, 300, 0, 50.0, False),
    ("bf16", 5, 5, 80, 129, 0, 10.0, True),
    ("q8", 32, 8, 128, 2999, 0, 30.0, True),
    ("q8", 8, 4, 64, 64, 0, 50.0, False),
    ("q8", 8, 4, 256, 1500, 512, 50.0, True),
    ("q8", 8, 2, 512, 300, 0, 0.0, True),
    ("q8", 4, 2, 36, 70, 0, 50.0, True),
    ("bf16", 16, 2, 128, 131075, 0, 50.0, False),
    ("q8", 4, 1, 64, 131072, 0, 50.0, True),
]


def decode_problem(kv, nq, nkv, d, n, alibi, seed=11, sigma_q=3.0):
    g = gen(seed)
    q = randn(g, 1, nq, d, sigma=sigma_q)
    Kc, K = ref.make_cache(randn(g, n, nkv, d), kv)
    Vc, V = ref.make_cache(randn(g, n, nkv, d), kv)
    return q, Kc, Vc, K, V, slopes_of(nq) if alibi else None


def span(n, pos, window):
    lo = max(0, pos - window + 1) if window > 0 else 0
    return (torch.tensor([min(lo, n)], device="cuda"), torch.tensor([n], device="cuda"),
            torch.tensor([pos], device="cuda"))


@pytest.mark.parametrize("kv,nq,nkv,d,n,window,softcap,alibi", DECODE)
def test_decode(gpu, kv, nq, nkv, d, n, window, softcap, alibi):
    q, Kc, Vc, K, V, sl = decode_problem(kv, nq, nkv, d, n, alibi)
    O = torch.full((1, nq, d), math.nan, device="cuda")
    scale = 1 / math.sqrt(d)
    attn.attn_decode_scored(q, Kc, Vc, O, nq, nkv, n, d, scale, n - 1, window, softcap, sl)
    lo, hi, pos = span(n, n - 1, window)
    want, _ = ref.attend(q, K, V, scale, pos, lo, hi, softcap, sl)
    check_out(O, want, ref.tolerance(q, K, V, scale, softcap, sl, n))


@pytest.mark.parametrize("kv,nq,nkv,d,n,window,softcap,alibi", DECODE)
def test_decode_weights(gpu, kv, nq, nkv, d, n, window, softcap, alibi):
    """acc of the attended slots grows by the heads' weights, no other changes."""
    q, Kc, Vc, K, V, sl = decode_problem(kv, nq, nkv, d, n, alibi, seed=12)
    O = torch.empty(1, nq, d, device="cuda")
    scale, cap = 1 / math.sqrt(d), n + 5
    acc = torch.rand(nkv, cap, device="cuda", generator=gen(3))
    before = acc.clone()
    attn.attn_decode_scored(q, Kc, Vc, O, nq, nkv, n, d, scale, n - 1, window, softcap, sl, acc)
    lo, hi, pos = span(n, n - 1, window)
    want, p = ref.attend(q, K, V, scale, pos, lo, hi, softcap, sl)
    check_out(O, want, ref.tolerance(q, K, V, scale, softcap, sl, n))
    grown = before.double()
    grown[:, :n] += p.view(nkv, nq // nkv, n).sum(1)
    one = torch.ones_like(V)
    tol = ref.tolerance(q, K, one, scale, softcap, sl, n) * (nq // nkv) + 2 * ref.EPS32 * (nq // nkv + 1)
    assert float((acc.double() - grown).abs().max()) <= tol
    assert torch.equal(acc[:, n:], before[:, n:]) and torch.equal(acc[:, :int(lo)], before[:, :int(lo)])


@pytest.mark.parametrize("merge", [-1, 0, 1])
@pytest.mark.parametrize("kv,nq,nkv,d,n", [("f32", 32, 8, 128, 300), ("f32", 32, 8, 128, 9001),
                                           ("bf16", 32, 8, 128, 700), ("q8", 32, 8, 128, 50)])
def test_decode_weights_by_each_merge(gpu, kv, nq, nkv, d, n, merge):
    q, Kc, Vc, K, V, sl = decode_problem(kv, nq, nkv, d, n, True)
    O, acc = torch.empty(1, nq, d, device="cuda"), torch.zeros(nkv, n, device="cuda")
    _lib.load().molot_hip_set_merge(merge)
    try:
        attn.attn_decode_scored(q, Kc, Vc, O, nq, nkv, n, d, 0.09, n - 1, 0, 50.0, sl, acc)
    finally:
        _lib.load().molot_hip_set_merge(-1)
    lo, hi, pos = span(n, n - 1, 0)
    want, p = ref.attend(q, K, V, 0.09, pos, lo, hi, 50.0, sl)
    check_out(O, want, ref.tolerance(q, K, V, 0.09, 50.0, sl, n))
    w = p.view(nkv, nq // nkv, n).sum(1)
    # (the tolerance of test_two_streams_at_once for one step)
    assert float((acc.double() - w).abs().max()) < 1e-4 * float(w.max())


def test_decode_empty_ranges(gpu):
    """No slot, or a window past them all: o = 0, acc left alone."""
    nq, nkv, d, n = 8, 4, 64, 40
    for kv in KVS:
        q, Kc, Vc, K, V, sl = decode_problem(kv, nq, nkv, d, n, True)
        for rows, pos, window in ((0, 0, 0), (n, 500, 8)):
            O = torch.full((1, nq, d), 7.0, device="cuda")
            acc = torch.ones(nkv, n, device="cuda")
            attn.attn_decode_scored(q, Kc, Vc, O, nq, nkv, rows, d, 0.125, pos, window, 50.0, sl, acc)
            assert torch.count_nonzero(O) == 0 and torch.equal(acc, torch.ones_like(acc))


@pytest.mark.parametrize("softcap", [1e-30, 1e-3, 2.0, 1e30])
def test_caps_of_any_size(gpu, softcap):
    """Far below the scores (all capped), about them, and far above (none)."""
    nq, nkv, d, n = 8, 4, 128, 700
    for kv in KVS:
        q, Kc, Vc, K, V, _ = decode_problem(kv, nq, nkv, d, n, False, seed=5)
        O = torch.empty(1, nq, d, device="cuda")
        scale = 1 / math.sqrt(d)
        attn.attn_decode_scored(q, Kc, Vc, O, nq, nkv, n, d, scale, n - 1, 0, softcap)
        lo, hi, pos = span(n, n - 1, 0)
        want, _ = ref.attend(q, K, V, scale, pos, lo, hi, softcap)
        check_out(O, want, ref.tolerance(q, K, V, scale, softcap, None, n))


def test_infinite_products_end_at_the_cap(gpu):
    """A key whose product overflows has score +cap (or -cap): with a cap the others
    keep their weight.  The rows: +inf, -inf, finite."""
    nq, nkv, d, n, cap = 4, 4, 64, 200, 4.0
    q, Kc, Vc, K, V, _ = decode_problem("f32", nq, nkv, d, n, False, seed=6)
    q = q.abs() + 0.5
    x = K.float().clone()
    x[17] = 3e38
    x[90] = -3e38
    Kc, K = ref.make_cache(x, "f32")
    O = torch.empty(1, nq, d, device="cuda")
    attn.attn_decode_scored(q, Kc, Vc, O, nq, nkv, n, d, 1.0, n - 1, 0, cap)
    lo, hi, pos = span(n, n - 1, 0)
    want, _ = ref.attend(q, K.clamp(-1e6, 1e6), V, 1.0, pos, lo, hi, cap)
    x[17], x[90] = 0.0, 0.0  # (the bound is the finite rows'; the two are at the cap)
    check_out(O, want, ref.tolerance(q, x.double(), V, 1.0, cap, None, n))


def test_no_cap_no_slopes_is_the_plain_step(gpu):
    """The scored entry with neither is attn_decode_gqa_cache to rounding."""
    for kv in KVS:
        q, Kc, Vc, K, V, _ = decode_problem(kv, 32, 8, 128, 3000, False)
        a, b = torch.empty(2, 1, 32, 128, device="cuda").unbind(0)
        attn.attn_decode_gqa_cache(q, Kc, Vc, a, 32, 8, 3000, 128, 0.09, 2999, 0)
        attn.attn_decode_scored(q, Kc, Vc, b, 32, 8, 3000, 128, 0.09, 2999)
        assert rel(a, b.double()) < 2e-6


STEP = [("f32", 32, 8, 128, 700, 0, True), ("bf16", 32, 8, 128, 2500, 0, True),
        ("q8", 32, 8, 128, 1300, 0, True), ("f32", 8, 4, 256, 1200, 512, False),
        ("q8", 8, 2, 512, 40, 0, False), ("bf16", 12, 4, 96, 0, 0, True),
        ("bf16", 16, 1, 64, 3, 2, True), ("f32", 7, 7, 50, 90, 0, False)]


@pytest.mark.parametrize("kv,nq,nkv,d,slot,window,alibi", STEP)
def test_step(gpu, kv, nq, nkv, d, slot, window, alibi):
    """The fused step: rows and q as the unscored step leaves them, the attention of
    the rows stored, acc and position of the new slot set."""
    g = gen(21)
    n, pos, scale, cap = slot + 1, slot + 9, 1 / math.sqrt(d), slot + 4
    q, k, v = randn(g, nq, d, sigma=3.0), randn(g, nkv, d), randn(g, nkv, d)
    Kc, _ = ref.make_cache(randn(g, n, nkv, d), kv)
    Vc, _ = ref.make_cache(randn(g, n, nkv, d), kv)
    wq, wk = 1 + 0.2 * randn(g, d), 1 + 0.2 * randn(g, d)
    inv = attn.rope_inv_freq(10000.0, d).cuda()
    sl = slopes_of(nq) if alibi else None
    acc = torch.rand(nkv, cap, device="cuda", generator=g)
    sp = torch.full((nkv, cap), -5, dtype=torch.int32, device="cuda")
    acc0 = acc.clone()
    q1, K1, V1, q2, K2, V2 = (x.clone() for x in (q, Kc, Vc) * 2)
    O = torch.empty(nq, d, device="cuda")
    # (window past the slot: nothing attended is covered by test_step_outside_its_window)
    pos_w = slot if window else pos
    attn.decode_step_scored(q1, k, v, K1, V1, O, nq, nkv, d, slot, pos_w, inv, scale, window, 40.0,
                            sl, acc, sp, wq, wk, True, 1e-6)
    attn.decode_step(q2, k, v, K2, V2, torch.empty_like(O), nq, nkv, d, slot, pos_w, inv, scale,
                     window, wq, wk, True, 1e-6)
    assert torch.equal(q1, q2) and torch.equal(K1, K2) and torch.equal(V1, V2)
    K, V = ref.cache_values(K1, kv, nkv, d), ref.cache_values(V1, kv, nkv, d)
    lo, hi, p0 = span(n, pos_w, window)
    want, p = ref.attend(q1.view(1, nq, d), K, V, scale, p0, lo, hi, 40.0, sl)
    check_out(O, want[0], ref.tolerance(q1.view(1, nq, d), K, V, scale, 40.0, sl, n + 9))
    grown = acc0.double()
    grown[:, slot] = 0.0
    grown[:, :n] += p.view(nkv, nq // nkv, n).sum(1)
    G = nq // nkv
    tol = ref.tolerance(q1.view(1, nq, d), K, torch.ones_like(V), scale, 40.0, sl, n + 9) * G
    assert float((acc.double() - grown).abs().max()) <= tol + 2 * ref.EPS32 * (G + 1)
    assert (sp[:, slot] == pos_w).all() and (sp[:, :slot] == -5).all() and (sp[:, n:] == -5).all()
    assert torch.equal(acc[:, n:], acc0[:, n:])


def test_step_outside_its_window(gpu):
    """The new row itself outside the window: appended, o = 0, its acc 0."""
    nq, nkv, d, slot, pos = 8, 4, 64, 10, 400
    for kv in KVS:
        g = gen(22)
        q, k, v = randn(g, nq, d), randn(g, nkv, d), randn(g, nkv, d)
        Kc, _ = ref.make_cache(randn(g, 12, nkv, d), kv)
        Vc, _ = ref.make_cache(randn(g, 12, nkv, d), kv)
        acc, sp = torch.ones(nkv, 12, device="cuda"), torch.zeros(nkv, 12, dtype=torch.int32, device="cuda")
        O = torch.ones(nq, d, device="cuda")
        attn.decode_step_scored(q, k, v, Kc, Vc, O, nq, nkv, d, slot, pos, None, 0.125, 16, 50.0, None,
                                acc, sp)
        assert torch.count_nonzero(O) == 0
        assert (acc[:, slot] == 0).all() and (sp[:, slot] == pos).all()
        assert (acc[:, :slot] == 1).all() and (acc[:, 11] == 1).all() and (sp[:, :slot] == 0).all()


PAGED = [("bf16", 32, 8, 128, (1, 700, 33, 2048, 16, 0), 16, 0, True),
         ("q8", 32, 8, 128, (2999, 1, 500), 16, 0, True),
         ("f32", 8, 2, 128, (65, 0, 17), 8, 0, False),
         ("f32", 8, 4, 256, (300, 1500), 32, 200, True),
         ("q8", 8, 2, 512, (40, 5), 16, 0, False),
         ("bf16", 12, 4, 96, (90, 130, 7), 4, 50, True)]


def paged_problem(kv, nq, nkv, d, lens, page, seed=31):
    g = gen(seed)
    need = [(n + page - 1) // page for n in lens]
    blocks = sum(need) + 3
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(1, max(need))
    table = torch.full((len(lens), width), 10 ** 6, dtype=torch.int32)  # unused entries: never read
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = torch.tensor(perm[at:at + k], dtype=torch.int32)
        at += k
    pools, values = [], []
    for _ in range(2):
        fill = 0.0 if kv == "q8" else math.nan  # pages and rows of nobody
        pool = ref.make_pages(randn(g, 0, nkv, d), kv, blocks, [], page, fill)
        vals = []
        for b, n in enumerate(lens):
            x = randn(g, n, nkv, d)
            ref.put_pages(pool, x, kv, table[b].tolist(), page)
            vals.append(ref.make_cache(x, kv)[1])
        pools.append(pool)
        values.append(vals)
    q = randn(g, len(lens), nq, d, sigma=3.0)
    return q, pools, values, table, blocks


@pytest.mark.parametrize("kv,nq,nkv,d,lens,page,window,alibi", PAGED)
def test_paged_with_weights(gpu, kv, nq, nkv, d, lens, page, window, alibi):
    q, (Kp, Vp), (Ks, Vs), table, blocks = paged_problem(kv, nq, nkv, d, lens, page)
    B, G, scale = len(lens), nq // nkv, 1 / math.sqrt(d)
    sl = slopes_of(nq) if alibi else None
    acc = torch.rand(blocks, nkv, page, device="cuda", generator=gen(4))
    grown = acc.double()
    O = torch.full((B, nq, d), math.nan, device="cuda")
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    attn.attn_decode_paged_scored(q, Kp, Vp, O, table.cuda(), L, None, B, table.shape[1], nq, nkv, d,
                                  page, scale, window, 50.0, sl, acc)
    tol_w = 0.0
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.count_nonzero(O[b]) == 0
            continue
        lo, hi, pos = span(n, n - 1, window)
        qb = q[b:b + 1]
        want, p = ref.attend(qb, Ks[b], Vs[b], scale, pos, lo, hi, 50.0, sl)
        check_out(O[b], want[0], ref.tolerance(qb, Ks[b], Vs[b], scale, 50.0, sl, n))
        w = p.view(nkv, G, n).sum(1)
        t = torch.arange(n)
        grown[table[b].long()[t // page].cuda(), :, (t % page).cuda()] += w.T
        tol_w = max(tol_w, ref.tolerance(qb, Ks[b], torch.ones_like(Vs[b]), scale, 50.0, sl, n) * G)
    assert float((acc.double() - grown).abs().max()) <= tol_w + 2 * ref.EPS32 * (G + 1)


@pytest.mark.parametrize("nq,n", [(4096, 140000), (4097, 10)])
def test_weights_refused(gpu, nq, n):
    """Scores of one KV head past 2 GiB, and more than 4096 heads on it: refused, nothing
    written; the same call without weights runs."""
    K, V = (torch.ones(n, 2, device="cuda") for _ in range(2))
    q, O = torch.ones(nq, 2, device="cuda"), torch.zeros(nq, 2, device="cuda")
    acc = torch.zeros(1, n, device="cuda")
    with pytest.raises(_lib.MolotHipError):
        attn.attn_decode_scored(q, K, V, O, nq, 1, n, 2, 1.0, n - 1, 0, 50.0, None, acc)
    torch.cuda.synchronize()
    assert torch.count_nonzero(acc) == 0 and torch.count_nonzero(O) == 0
    attn.attn_decode_scored(q, K, V, O, nq, 1, n, 2, 1.0, n - 1, 0, 50.0)
    assert float((O - 1).abs().max()) < 1e-5


def test_paged_weights_past_a_gigabyte(gpu):
    """64 sequences of 70000 rows under 64 heads: 1.15 GB of scores kept for the weights."""
    nq, nkv, d, page, B, n = 64, 1, 64, 16, 64, 70000
    g, G, width = gen(36), nq // nkv, n // page
    table = torch.randperm(B * width, device="cuda", generator=g).int().view(B, width)
    K, V = (randn(g, B * width, page * d).bfloat16() for _ in range(2))
    acc = torch.zeros(B * width, nkv, page, device="cuda")
    q, O = randn(g, B, nq, d, sigma=3.0), torch.empty(B, nq, d, device="cuda")
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    attn.attn_decode_paged_scored(q, K, V, O, table, lens, None, B, width, nq, nkv, d, page, 0.125, 0,
                                  50.0, None, acc)
    lo, hi, pos = span(n, n - 1, 0)
    for b in (0, 31, B - 1):
        Kb, Vb = (x[table[b].long()].view(n, nkv, d).double() for x in (K, V))
        want, p = ref.attend(q[b:b + 1], Kb, Vb, 0.125, pos, lo, hi, 50.0)
        check_out(O[b], want[0], ref.tolerance(q[b:b + 1], Kb, Vb, 0.125, 50.0, None, n))
        got = acc[table[b].long()].view(n).double()
        tol = ref.tolerance(q[b:b + 1], Kb, torch.ones_like(Vb), 0.125, 50.0, None, n) * G
        assert float((got - p.view(G, n).sum(0)).abs().max()) <= tol


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("lag", [0, 3, None])
def test_paged_step(gpu, kv, lag):
    """The fused paged step, positions told or not: rows as the unscored step's, and
    the new slots' acc and positions."""
    nq, nkv, d, page, lens = 16, 4, 128, 16, (1, 17, 260, 32)
    q, (Kp, Vp), _, table, blocks = paged_problem(kv, nq, nkv, d, lens, page, seed=33)
    B, G, scale = len(lens), nq // nkv, 1 / math.sqrt(d)
    g = gen(34)
    k, v = randn(g, B, nkv, d), randn(g, B, nkv, d)
    inv = attn.rope_inv_freq(10000.0, d).cuda()
    sl, L, tb = slopes_of(nq), torch.tensor(lens, dtype=torch.int32, device="cuda"), table.cuda()
    pos = None if lag is None else L - 1 + lag
    acc = torch.rand(blocks, nkv, page, device="cuda", generator=g)
    acc0 = acc.clone()
    sp = torch.full((blocks, nkv, page), -5, dtype=torch.int32, device="cuda")
    q1, K1, V1, q2, K2, V2 = (x.clone() for x in (q, Kp, Vp) * 2)
    O = torch.empty(B, nq, d, device="cuda")
    attn.decode_step_paged_scored(q1, k, v, K1, V1, O, tb, L, pos, B, table.shape[1], nq, nkv, d, page,
                                  inv, scale, 0, 30.0, sl, acc, sp)
    if pos is None:
        # (with positions the unscored step takes its unfused kernels, whose rotation
        # rounds its two products apart)
        attn.decode_step_paged(q2, k, v, K2, V2, torch.empty_like(O), tb, L, None, B, table.shape[1],
                               nq, nkv, d, page, inv, scale)
        assert torch.equal(q1, q2)
        for x, y in ((K1, K2), (V1, V2)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # the new rows against the rotation in 64 bits (the angle is the fp32 product): fp32
    # rounds two products and their sum, the cache types half a step of theirs
    ang = ((L - 1 + (lag or 0)).float()[:, None] * inv).double()[:, None]
    k0, k1 = k.double().chunk(2, -1)
    turned = torch.cat([k0 * ang.cos() - k1 * ang.sin(), k0 * ang.sin() + k1 * ang.cos()], -1)
    near = {"f32": 0.0, "bf16": 2.0 ** -8, "q8": 0.5 / 127}[kv] + 6 * ref.EPS32
    for b, n in enumerate(lens):
        pages = table[b, :(n + page - 1) // page].long().cuda()

        def rows(pool):
            x = pool[pages]
            if kv == "q8":
                cut = nkv * page * d
                c = x[:, :cut].contiguous().view(torch.int8).view(-1, nkv, page, d).double()
                x = c * x[:, cut:].contiguous().view(torch.float32).view(-1, nkv, page)[..., None].double()
            else:
                x = x.view(-1, nkv, page, d).double()
            return x.transpose(1, 2).reshape(-1, nkv, d)[:n]

        K, V = rows(K1), rows(V1)
        assert float((K[n - 1] - turned[b]).abs().max()) <= near * 2 * float(k[b].abs().max())
        p0 = torch.tensor([n - 1 + (lag or 0)], device="cuda")
        lo, hi, _ = span(n, n - 1, 0)
        want, p = ref.attend(q1[b:b + 1], K, V, scale, p0, lo, hi, 30.0, sl)
        check_out(O[b], want[0], ref.tolerance(q1[b:b + 1], K, V, scale, 30.0, sl, n + 3))
        t = torch.arange(n)
        at = (pages[(t // page).cuda()], slice(None), (t % page).cuda())
        base = acc0[at].double()
        base[n - 1] = 0.0
        tol = ref.tolerance(q1[b:b + 1], K, torch.ones_like(V), scale, 30.0, sl, n + 3) * G
        err = float((acc[at].double() - base - p.view(nkv, G, n).sum(1).T).abs().max())
        assert err <= tol + 2 * ref.EPS32 * (G + 1)
        got = sp[at]
        assert (got[n - 1] == n - 1 + (lag or 0)).all() and (got[:n - 1] == -5).all()


# --- prefill -----------------------------------------------------------------

# (kv, nq, nkv, d, m, n0, window, softcap, alibi, mask)
PREFILL = [
    ("f32", 32, 8, 128, 200, 0, 0, 50.0, False, "causal"),
    ("f32", 32, 8, 128, 77, 300, 0, 50.0, True, "causal"),
    ("f32", 8, 8, 64, 130, 0, 0, 0.0, True, "docs"),
    ("f32", 8, 4, 256, 150, 20, 64, 50.0, True, "causal"),
    ("f32", 8, 2, 512, 90, 0, 0, 50.0, False, "prefix"),
    ("f32", 12, 4, 96, 65, 33, 0, 30.0, True, "ranges"),
    ("f32", 6, 2, 34, 41, 0, 0, 5.0, True, "ranges"),
    ("bf16", 32, 8, 128, 300, 0, 0, 50.0, True, "docs"),
    ("bf16", 8, 4, 256, 300, 0, 0, 50.0, False, "docs"),
    ("bf16", 8, 4, 256, 70, 500, 128, 30.0, True, "ranges"),
    ("bf16", 16, 1, 64, 100, 0, 0, 30.0, True, "prefix"),
    ("bf16", 8, 2, 512, 33, 70, 0, 50.0, True, "ranges"),
    ("q8", 32, 8, 128, 129, 0, 0, 50.0, True, "docs"),
    ("q8", 8, 4, 256, 64, 64, 0, 50.0, True, "ranges"),
    ("q8", 4, 2, 36, 50, 0, 0, 30.0, True, "prefix"),
    ("q8", 8, 2, 512, 70, 10, 0, 20.0, False, "causal"),
    ("f32", 32, 8, 128, 1, 0, 0, 50.0, True, "causal"),
    ("bf16", 32, 8, 128, 2, 1000, 0, 50.0, True, "causal"),
    ("q8", 8, 8, 64, 3, 40, 0, 50.0, True, "ranges"),
    # enough query rows for the pieces; several key splits, and blocks of few keys with one
    ("f32", 16, 4, 64, 345, 0, 0, 50.0, True, "docs"),
    ("q8", 8, 8, 64, 150, 0, 0, 50.0, True, "ranges"),
    ("q8", 4, 2, 36, 211, 0, 0, 30.0, True, "prefix"),
    ("f32", 6, 2, 34, 601, 0, 0, 5.0, True, "docs"),
    ("bf16", 32, 8, 128, 175, 0, 0, 50.0, True, "ranges"),
    ("q8", 32, 8, 128, 101, 0, 0, 50.0, False, "prefix"),
    ("f32", 12, 4, 96, 301, 0, 0, 30.0, True, "ranges"),
    ("f32", 8, 4, 256, 351, 0, 0, 0.0, True, "docs"),
    ("bf16", 8, 4, 256, 700, 0, 0, 50.0, True, "docs"),
    ("bf16", 8, 4, 256, 65, 2000, 0, 50.0, False, "causal"),
    ("q8", 8, 4, 256, 301, 0, 0, 50.0, True, "ranges"),
    ("f32", 8, 2, 512, 401, 0, 0, 50.0, True, "docs"),
    ("bf16", 8, 2, 512, 699, 0, 0, 50.0, True, "docs"),
    ("bf16", 8, 2, 512, 33, 2000, 700, 50.0, True, "causal"),
    ("q8", 8, 2, 512, 399, 0, 0, 50.0, True, "ranges"),
]


def key_ranges(mask, m, n0, window, seed=9):
    """(lo, hi as given or None, lo, hi as attended) of every row."""
    N = n0 + m
    pos = n0 + torch.arange(m)
    start = (pos - window + 1).clamp(min=0) if window > 0 else torch.zeros(m, dtype=torch.long)
    lo = hi = None
    if mask == "docs":
        lens, left = [], m
        for k in (7, 50, 1, 64, 33):
            lens.append(min(k, left))
            left -= lens[-1]
        lo = attn.document_starts(lens + [left], n0)
    elif mask == "prefix":
        hi = torch.maximum(pos + 1, torch.full_like(pos, n0 + m // 2)).int()
    elif mask == "ranges":  # anything, empty ones and values outside the keys among them
        r = torch.Generator().manual_seed(seed)
        lo = torch.randint(-20, N + 20, (m,), generator=r, dtype=torch.int32)
        hi = torch.randint(-20, N + 40, (m,), generator=r, dtype=torch.int32)
        lo[::3] = 0
        hi[1::3] = N
    at = start if lo is None else torch.maximum(start, lo.long())
    end = (pos + 1 if hi is None else hi.long()).clamp(0, N)
    return lo, hi, at, end


@pytest.mark.parametrize("presplit", [True, False])
@pytest.mark.parametrize("kv,nq,nkv,d,m,n0,window,softcap,alibi,mask", PREFILL)
def test_prefill(gpu, kv, nq, nkv, d, m, n0, window, softcap, alibi, mask, presplit):
    g = gen(41)
    N, scale = n0 + m, 1 / math.sqrt(d)
    q = randn(g, m, nq, d, sigma=3.0)
    Kc, K = ref.make_cache(randn(g, N, nkv, d), kv)
    Vc, V = ref.make_cache(randn(g, N, nkv, d), kv)
    sl = slopes_of(nq) if alibi else None
    lo, hi, at, end = key_ranges(mask, m, n0, window)
    dev = lambda x: None if x is None else x.cuda()  # noqa: E731
    O = torch.full((m, nq, d), math.nan, device="cuda")
    attn.set_prefill_presplit(presplit)
    try:
        attn.attn_prefill_scored(q, Kc, Vc, O, nq, nkv, m, N, d, scale, n0, window, softcap, sl,
                                 dev(lo), dev(hi))
    finally:
        attn.set_prefill_presplit(True)
    pos = n0 + torch.arange(m, device="cuda")
    want, _ = ref.attend(q, K, V, scale, pos, at.cuda(), end.cuda(), softcap, sl)
    check_out(O, want, ref.tolerance(q, K, V, scale, softcap, sl, N))
    empty = (at >= end).cuda()
    assert torch.count_nonzero(O[empty]) == 0


@pytest.mark.parametrize("d", [64, 96, 128, 256, 512])
@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, "lowest"])
@pytest.mark.parametrize("m", [96, 500])  # rows streamed one by one; the pieces
def test_prefill_masked_rows_count_for_nothing(gpu, kv, d, bad, m):
    """What a masked key holds, in K, V or both, reaches no row that does not see it."""
    nq, nkv = 8, 4
    g = gen(43)
    q = randn(g, m, nq, d, sigma=3.0)
    xk, xv = randn(g, m, nkv, d), randn(g, m, nkv, d)
    if bad == "lowest":
        bad = float(torch.finfo(torch.float32 if kv == "f32" else torch.bfloat16).min)
    starts = attn.document_starts([30, 41, m - 71])
    for t in (33, 70):  # rows of the second document
        xk[t, 1] = bad
        xv[t, :, ::2] = bad
    Kc, K = ref.make_cache(xk, kv)
    Vc, V = ref.make_cache(xv, kv)
    O = torch.empty(m, nq, d, device="cuda")
    scale = 1 / math.sqrt(d)
    attn.attn_prefill_scored(q, Kc, Vc, O, nq, nkv, m, m, d, scale, 0, 0, 50.0, None, starts.cuda())
    keep = torch.tensor([i for i in range(m) if i < 33 or i >= 71], device="cuda")
    Kz, Vz = K.clone(), V.clone()
    Kz[[33, 70]], Vz[[33, 70]] = 0.0, 0.0
    pos = torch.arange(m, device="cuda")
    want, _ = ref.attend(q, Kz, Vz, scale, pos, starts.cuda().long(), pos + 1, 50.0)
    check_out(O[keep], want[keep], ref.tolerance(q, Kz, Vz, scale, 50.0, None, m))


@pytest.mark.parametrize("kv,d", [("f32", 128), ("bf16", 64), ("q8", 256), ("f32", 80), ("q8", 512)])
@pytest.mark.parametrize("slot0", [0, 21])
@pytest.mark.parametrize("m", [70, 500])  # rows streamed one by one; the pieces
def test_prefill_steps(gpu, kv, d, slot0, m):
    """The appending steps, contiguous and paged: rows and q as the unscored steps
    leave them, the attention of the rows stored."""
    nq, nkv, page = 8, 4, 16
    g = gen(45)
    N, scale = slot0 + m, 1 / math.sqrt(d)
    q, k, v = randn(g, m, nq, d, sigma=3.0), randn(g, m, nkv, d), randn(g, m, nkv, d)
    x, y = randn(g, N, nkv, d), randn(g, N, nkv, d)
    inv = attn.rope_inv_freq(10000.0, d).cuda()
    wq = 1 + 0.2 * randn(g, d)
    sl = slopes_of(nq)
    lo = attn.document_starts([40, m - 40], slot0).cuda()
    pos = slot0 + torch.arange(m, device="cuda")
    Kc, Vc = ref.make_cache(x, kv)[0], ref.make_cache(y, kv)[0]
    K2, V2, q1, q2 = Kc.clone(), Vc.clone(), q.clone(), q.clone()
    O = torch.empty(m, nq, d, device="cuda")
    attn.prefill_step_scored(q1, k, v, Kc, Vc, O, nq, nkv, d, m, slot0, slot0, inv, scale, 0, 50.0, sl,
                             lo, None, wq, None, True)
    attn.prefill_step(q2, k, v, K2, V2, torch.empty_like(O), nq, nkv, d, m, slot0, slot0, inv, scale, 0,
                      wq, None, True)
    assert torch.equal(q1, q2) and torch.equal(Kc, K2) and torch.equal(Vc, V2)
    K, V = ref.cache_values(Kc, kv, nkv, d), ref.cache_values(Vc, kv, nkv, d)
    want, _ = ref.attend(q1, K, V, scale, pos, lo.long(), pos + 1, 50.0, sl)
    tol = ref.tolerance(q1, K, V, scale, 50.0, sl, N)
    check_out(O, want, tol)
    blocks = (N + page - 1) // page
    table = torch.arange(blocks, dtype=torch.int32).flip(0)
    Kp = ref.make_pages(x, kv, blocks, table.tolist(), page)
    Vp = ref.make_pages(y, kv, blocks, table.tolist(), page)
    q3, O3 = q.clone(), torch.empty_like(O)
    attn.prefill_step_paged_scored(q3, k, v, Kp, Vp, O3, table.cuda(), blocks, page, nq, nkv, d, m,
                                   slot0, slot0, inv, scale, 0, 50.0, sl, lo, None, wq, None, True)
    assert torch.equal(q3, q1)
    check_out(O3, want, tol)
    O4 = torch.empty_like(O)
    attn.attn_prefill_paged_scored(q3, Kp, Vp, O4, table.cuda(), blocks, page, nq, nkv, m, N, d, scale,
                                   slot0, 0, 50.0, sl, lo, None)
    check_out(O4, want, tol)


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("slot0,behind,window", [(0, 0, 0), (21, 0, 300), (21, 400, 0), (130, 400, 200)])
def test_prefill_step_pieces(gpu, kv, d, slot0, behind, window):
    """A step whose append leaves the attention's operands gives what the attention over
    the stored rows does, rows among them that no operand holds: not finite, and past
    the operands' range.  behind: positions past the slots (rows were evicted)."""
    nq, nkv, m = 8, 4, 520
    g = gen(48)
    N, scale = slot0 + m, 1 / math.sqrt(d)
    q, k, v = randn(g, m, nq, d, sigma=3.0), randn(g, m, nkv, d), randn(g, m, nkv, d)
    if kv != "q8":
        k[100, 1] *= 1e25
        v[200, 2] *= 1e-33
        k[333, 0, 5] = math.nan
        v[333, 0, 7] = math.inf
    inv = attn.rope_inv_freq(10000.0, d).cuda()
    sl = slopes_of(nq)
    lo = attn.document_starts([90, 200, 100, m - 390], slot0).cuda()
    Kc, Vc = (ref.make_cache(randn(g, N, nkv, d), kv)[0] for _ in range(2))
    O, O2 = torch.empty(m, nq, d, device="cuda"), torch.empty(m, nq, d, device="cuda")
    _lib.load().molot_hip_set_block_order(0)  # (the small windows' rows are streamed: in one order both times)
    try:
        attn.prefill_step_scored(q, k, v, Kc, Vc, O, nq, nkv, d, m, slot0, slot0 + behind, inv, scale,
                                 window, 50.0, sl, lo)
        attn.attn_prefill_scored(q, Kc, Vc, O2, nq, nkv, m, N, d, scale, slot0, window, 50.0, sl, lo)
    finally:
        _lib.load().molot_hip_set_block_order(1)
    assert torch.equal(O.view(torch.int32), O2.view(torch.int32))
    clean = torch.ones(m, dtype=torch.bool, device="cuda")
    clean[90:290] = clean[333:390] = False  # documents with the rows that are not ordinary, from there on
    assert bool(torch.isfinite(O[clean]).all())


@pytest.mark.parametrize("kv,d", [("f32", 128), ("bf16", 64), ("f32", 256), ("bf16", 512)])
@pytest.mark.parametrize("below", [16.0, 21.0, 24.0])
def test_prefill_of_one_key_above_a_long_tail(gpu, kv, d, below):
    """One key, then 16383 that are e^-below of it each and together up to 2e-3 of the
    output: none of them may be dropped as small."""
    nq, nkv, m, N = 4, 1, 520, 16384
    g = gen(52)
    K, V = torch.zeros(N, nkv, d, device="cuda"), 1 + 0.01 * randn(g, N, nkv, d)
    K[5, 0, 0], V[5] = 1.0, -1.0
    q = torch.zeros(m, nq, d, device="cuda")
    q[:, :, 0] = below
    Kc, K = ref.make_cache(K, kv)
    Vc, V = ref.make_cache(V, kv)
    O = torch.empty(m, nq, d, device="cuda")
    sl = torch.zeros(nq, device="cuda")
    attn.attn_prefill_scored(q, Kc, Vc, O, nq, nkv, m, N, d, 1.0, N - m, 0, 0.0, sl)
    some = torch.tensor([0, 1, 31, 32, 300, 519], device="cuda")
    pos = N - m + some
    want, _ = ref.attend(q[some], K, V, 1.0, pos, torch.zeros_like(pos), pos + 1, 0.0)
    # Every score is one exact product (below * 1, or 0), so what moves is: the one key's
    # score in base 2 by three roundings of half an ulp of 32, 2^-20 each, and the tail
    # (mass w of the output, its V 2 away) with it; the sum (test_prefill's 2^-21 and
    # 8 2^-24 of |V|); what the pieces drop of 2^14 keys, 2^-20 of |V|; and half an ulp of
    # the one key's output, 2^-25 |V|, a tile of 32 keys added to it, all to one side
    # (a tile of the tail is less than that half ulp from below = 21 on): 512 of them.
    w = N * math.exp(-below)
    vmax = float(V.abs().max())
    tol = 2 * w * 3 * 2.0 ** -20 + (2.0 ** -21 + 8 * ref.EPS32 + 2.0 ** -20 + N / 32 * 2.0 ** -25) * vmax
    check_out(O[some], want, tol)


def test_prefill_of_more_rows_than_a_grid(gpu):
    """70001 rows in one call: every row its own keys, on either side of the parts' ends."""
    nq, nkv, d, m = 2, 1, 64, 70001
    g = gen(49)
    q = randn(g, m, nq, d, sigma=3.0)
    Kc, K = ref.make_cache(randn(g, m, nkv, d), "bf16")
    Vc, V = ref.make_cache(randn(g, m, nkv, d), "bf16")
    lo = attn.document_starts([700] * 100 + [1]).cuda()
    hi = (torch.arange(m, device="cuda") + 30).int()
    sl = slopes_of(nq)
    O = torch.full((m, nq, d), math.nan, device="cuda")
    attn.attn_prefill_scored(q, Kc, Vc, O, nq, nkv, m, m, d, 0.125, 0, 0, 50.0, sl, lo, hi)
    assert bool(torch.isfinite(O).all())
    some = torch.tensor([0, 1, 699, 700, *range(32760, 32776), *range(65528, 65544), m - 2, m - 1],
                        device="cuda")
    want, _ = ref.attend(q[some], K, V, 0.125, some, lo[some].long(), hi[some].long().clamp(max=m), 50.0, sl)
    check_out(O[some], want, ref.tolerance(q[some], K, V, 0.125, 50.0, sl, m))


def test_prefill_pieces_past_a_gigabyte(gpu):
    """A long fp32 cache: 1.15 GB of pieces."""
    nq, nkv, d, m, N = 8, 8, 128, 64, 140001
    g = gen(50)
    q = randn(g, m, nq, d, sigma=3.0)
    Kc, K = ref.make_cache(randn(g, N, nkv, d), "f32")
    Vc, V = ref.make_cache(randn(g, N, nkv, d), "f32")
    O = torch.empty(m, nq, d, device="cuda")
    attn.attn_prefill_scored(q, Kc, Vc, O, nq, nkv, m, N, d, 0.09, N - m, 0, 50.0)
    some = torch.tensor([0, 31, 63], device="cuda")
    pos = N - m + some
    want, _ = ref.attend(q[some], K, V, 0.09, pos, torch.zeros_like(pos), pos + 1, 50.0)
    check_out(O[some], want, ref.tolerance(q[some], K, V, 0.09, 50.0, None, N))


def test_prefill_step_behind_its_positions(gpu):
    """slot0 < pos0 (rows were evicted): a row sees no row appended after it."""
    nq, nkv, d, m, slot0, pos0 = 8, 4, 128, 40, 25, 300
    g = gen(46)
    q, k, v = randn(g, m, nq, d), randn(g, m, nkv, d), randn(g, m, nkv, d)
    Kc, _ = ref.make_cache(randn(g, slot0 + m, nkv, d), "f32")
    Vc, _ = ref.make_cache(randn(g, slot0 + m, nkv, d), "f32")
    O = torch.empty(m, nq, d, device="cuda")
    inv = attn.rope_inv_freq(10000.0, d).cuda()
    attn.prefill_step_scored(q, k, v, Kc, Vc, O, nq, nkv, d, m, slot0, pos0, inv, 0.09, 0, 50.0)
    K, V = ref.cache_values(Kc, "f32", nkv, d), ref.cache_values(Vc, "f32", nkv, d)
    i = slot0 + torch.arange(m, device="cuda")
    want, _ = ref.attend(q, K, V, 0.09, i, torch.zeros_like(i), i + 1, 50.0)
    check_out(O, want, ref.tolerance(q, K, V, 0.09, 50.0, None, slot0 + m))


# --- streams, graphs, refusals -------------------------------------------------


def test_graph_replays(gpu):
    """Steps with weights and a prefill with ranges, captured and replayed with eager
    calls between: every replay gives what the eager calls give."""
    nq, nkv, d, n, m = 32, 8, 128, 3000, 64
    q, Kc, Vc, K, V, sl = decode_problem("bf16", nq, nkv, d, n, True)
    qm = randn(gen(51), m, nq, d, sigma=3.0)
    lo = attn.document_starts([20, 44], n - m).cuda()
    O, Om = torch.empty(1, nq, d, device="cuda"), torch.empty(m, nq, d, device="cuda")
    acc = torch.zeros(nkv, n, device="cuda")

    def calls():
        attn.attn_decode_scored(q, Kc, Vc, O, nq, nkv, n, d, 0.09, n - 1, 0, 50.0, sl, acc)
        attn.attn_prefill_scored(qm, Kc, Vc, Om, nq, nkv, m, n, d, 0.09, n - m, 0, 50.0, sl, lo)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        calls()
        calls()
    torch.cuda.synchronize()
    want, want_m = O.clone(), Om.clone()
    one = acc.clone() / 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        calls()
    for i in range(3):
        acc.zero_()
        O.zero_()
        Om.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert rel(O, want.double()) < 2e-6 and rel(Om, want_m.double()) < 2e-6
        assert float((acc - one).abs().max()) < 1e-5
        calls()  # eager, on another stream's workspace
        torch.cuda.synchronize()


def test_two_streams_at_once(gpu):
    """Calls on two streams keep apart: each has its own workspaces."""
    nq, nkv, d, n = 32, 8, 128, 6000
    probs = [decode_problem(kv, nq, nkv, d, n, True, seed=60 + i) for i, kv in enumerate(("f32", "bf16"))]
    outs = [torch.empty(1, nq, d, device="cuda") for _ in probs]
    accs = [torch.zeros(nkv, n, device="cuda") for _ in probs]
    streams = [torch.cuda.Stream() for _ in probs]
    torch.cuda.synchronize()
    for _ in range(4):
        for (q, Kc, Vc, *_r, sl), O, acc, s in zip(probs, outs, accs, streams):
            with torch.cuda.stream(s):
                attn.attn_decode_scored(q, Kc, Vc, O, nq, nkv, n, d, 0.09, n - 1, 0, 50.0, sl, acc)
    torch.cuda.synchronize()
    for (q, Kc, Vc, K, V, sl), O, acc in zip(probs, outs, accs):
        lo, hi, pos = span(n, n - 1, 0)
        want, p = ref.attend(q, K, V, 0.09, pos, lo, hi, 50.0, sl)
        check_out(O, want, ref.tolerance(q, K, V, 0.09, 50.0, sl, n))
        w = 4 * p.view(nkv, nq // nkv, n).sum(1)
        assert float((acc.double() - w).abs().max()) < 4e-4 * float(w.max())


def test_capture_without_warmup_is_refused(gpu):
    """A capture cannot grow the weights' workspace: an error, nothing launched."""
    nq, nkv, d, n = 8, 4, 128, 5000
    q, Kc, Vc, *_ = decode_problem("f32", nq, nkv, d, n, False)
    O, acc = torch.empty(1, nq, d, device="cuda"), torch.zeros(nkv, n, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(_lib.MolotHipError):
        with torch.cuda.graph(graph, stream=s):
            one = torch.ones(1, device="cuda")  # (a graph of something)
            try:
                attn.attn_decode_scored(q, Kc, Vc, O, nq, nkv, n, d, 0.09, n - 1, 0, 50.0, None, acc)
            finally:
                one += 1
    torch.cuda.synchronize()
    assert torch.count_nonzero(acc) == 0
