"""Eviction from a cache by accumulated weight, against the rule slot by slot
(tests/scored_ref.py), and a stream that lives on a budget."""
from __future__ import annotations

import math

import pytest
import torch

import scored_ref as ref
from molot_amd import attn

pytestmark = pytest.mark.gpu

KVS = ("f32", "bf16", "q8")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def weights(g, kind, nkv, cap):
    if kind == "ties":
        return torch.randint(0, 4, (nkv, cap), device="cuda", generator=g).float()
    if kind == "equal":
        return torch.full((nkv, cap), 0.25, device="cuda")
    if kind == "near":  # equal in their first 20 bits, some in all
        return 1 + torch.randint(0, 4000, (nkv, cap), device="cuda", generator=g) * 2.0 ** -23
    x = torch.exp(2 * torch.randn(nkv, cap, device="cuda", generator=g))
    if kind == "odd":
        r = torch.rand(nkv, cap, device="cuda", generator=g)
        for lo, val in ((0.1, math.nan), (0.2, math.inf), (0.3, -math.inf), (0.4, -1.0), (0.5, -0.0),
                        (0.6, 0.0), (0.7, 1e-42)):
            x = torch.where((r < lo) & (r >= lo - 0.1), torch.full_like(x, val), x)
    return x


def raw(x):
    return x.view(torch.uint8) if x.dtype == torch.uint8 else x.view(
        {4: torch.int32, 2: torch.int16}[x.element_size()])


def cache_bits(c, kv, nkv, d):
    """[n][nkv][bytes] of a token-major cache's head rows, a Q8 row's scale with it."""
    n = c.shape[0]
    if kv != "q8":
        return c.view(n, nkv, d).view(torch.uint8).view(n, nkv, -1)
    codes = c[:, :nkv * d].reshape(n, nkv, d)
    sc = c[:, nkv * d:nkv * d + 4 * nkv].reshape(n, nkv, 4)
    return torch.cat([codes, sc], -1)


# (n, keep, recent)
CUTS = [(1, 0, 0), (1, 1, 3), (2, 1, 0), (5, 4, 2), (64, 63, 5), (65, 64, 64), (300, 200, 50),
        (1023, 1000, 0), (1024, 1, 1), (1025, 1024, 10), (2500, 2000, 300), (4352, 4096, 512),
        (3000, 100, 2999), (3000, 100, 5000), (7000, 3500, 1), (500, 500, 3), (500, 600, 3)]


@pytest.mark.parametrize("kind", ["smooth", "ties", "equal", "odd"])
@pytest.mark.parametrize("n,keep,recent", CUTS)
def test_rule(gpu, n, keep, recent, kind):
    """Positions in any order; the slots past n and outside the moves stay as they were."""
    nkv, d, cap, pos = 3, 34, n + 6, 5 * n
    g = gen(n + keep)
    acc = weights(g, kind, nkv, cap)
    sp = torch.stack([torch.randperm(cap, device="cuda", generator=g) for _ in range(nkv)]).int()
    sp += pos - cap + 1
    K, _ = ref.make_cache(torch.randn(n + 4, nkv, d, device="cuda", generator=g), "f32")
    V, _ = ref.make_cache(torch.randn(n + 4, nkv, d, device="cuda", generator=g), "f32")
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
    left = attn.kv_evict(K, V, acc, sp, nkv, n, d, keep, recent, pos)
    assert left == min(n, keep)
    for got, exp in zip((K, V, acc, sp), want):
        assert torch.equal(raw(got), raw(exp))


@pytest.mark.parametrize("kind", ["smooth", "ties", "equal", "odd", "zeros", "near"])
@pytest.mark.parametrize("n,keep,recent", [(16384, 16000, 500), (16385, 16000, 500), (20001, 8192, 3),
                                           (40000, 39999, 0), (40000, 1, 0), (60000, 24576, 40000),
                                           (33333, 30000, 2500), (131073, 120001, 5000)])
def test_rule_long(gpu, n, keep, recent, kind):
    """Caches past one workgroup's: chunks on both sides of keep, up to one bin of them."""
    nkv, d, pos = 2, 2, n - 1
    g = gen(n + keep)
    acc = weights(g, "smooth" if kind == "zeros" else kind, nkv, n)
    if kind == "zeros":  # most rows never seen
        acc = torch.where(torch.rand(nkv, n, device="cuda", generator=g) < 0.9, torch.zeros_like(acc), acc)
    sp = torch.stack([torch.randperm(n, device="cuda", generator=g) for _ in range(nkv)]).int()
    K = torch.randn(n, nkv * d, device="cuda", generator=g)
    V = torch.randn(n, nkv * d, device="cuda", generator=g)
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
        assert torch.equal(raw(got), raw(exp))


@pytest.mark.parametrize("pos,recent", [(-5, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31 - 1, 3),
                                        (-2 ** 31, 7)])
def test_extreme_positions(gpu, pos, recent):
    nkv, n, keep = 2, 50, 40
    acc = weights(gen(4), "smooth", nkv, n)
    sp = torch.tensor([-2 ** 31, -2 ** 31 + 1, -5, 0, 2 ** 31 - 1] * 10, device="cuda").int().repeat(nkv, 1)
    K, V = (torch.randn(n, nkv * 2, device="cuda", generator=gen(i)) for i in (5, 6))
    want = acc.clone()
    for h, moves in enumerate(ref.evict(acc.cpu(), sp.cpu(), n, keep, recent, pos)):
        for to, at in moves:
            want[h, to] = acc[h, at]
    attn.kv_evict(K, V, acc, sp, nkv, n, 2, keep, recent, pos)
    assert torch.equal(acc, want)


def test_shared_blocks_are_refused(gpu):
    """Every slot's acc has one writer: two sequences of a call, or one of them twice
    over, may not name the same block."""
    nkv, d, page, blocks = 2, 4, 8, 6
    K, V = (torch.zeros(blocks, nkv * page * d, device="cuda") for _ in range(2))
    acc = torch.zeros(blocks, nkv, page, device="cuda")
    sp = torch.zeros(blocks, nkv, page, dtype=torch.int32, device="cuda")
    q, o = torch.zeros(2, 4, d, device="cuda"), torch.zeros(2, 4, d, device="cuda")
    new = torch.zeros(2, nkv, d, device="cuda")
    inv = torch.ones(d // 2, device="cuda")
    for rows in ([[0, 1], [2, 0]], [[3, 3], [1, 2]]):
        table = torch.tensor(rows, dtype=torch.int32, device="cuda")
        lens = torch.tensor([16, 9], dtype=torch.int32, device="cuda")
        for call in (
                lambda: attn.attn_decode_paged_scored(q, K, V, o, table, lens, None, 2, 2, 4, nkv, d, page,
                                                      1.0, acc=acc),
                lambda: attn.decode_step_paged_scored(q, new, new, K, V, o, table, lens, None, 2, 2, 4, nkv,
                                                      d, page, inv, 1.0, acc=acc, slot_pos=sp),
                lambda: attn.kv_track_paged(acc, sp, table, lens, None, 2, 2, 3, nkv, page),
                lambda: attn.kv_evict_paged(K, V, acc, sp, table, lens, None, 2, 2, nkv, d, page, 5, 1)):
            with pytest.raises(ValueError):
                call()
        # without acc a block may serve several, as in the plain attention
        attn.attn_decode_paged_scored(q, K, V, o, table, lens, None, 2, 2, 4, nkv, d, page, 1.0)
    table = torch.tensor([[0, 1], [2, 0]], dtype=torch.int32, device="cuda")  # (its second entry unused)
    lens = torch.tensor([16, 8], dtype=torch.int32, device="cuda")
    attn.kv_track_paged(acc, sp, table, lens, None, 2, 2, 3, nkv, page)


def test_paged_long(gpu):
    """Sequences on either side of the one-workgroup limit in a batch."""
    kv, nkv, d, page, lens, keep, recent = "f32", 2, 4, 32, (17000, 20, 9000, 30001), 8000, 100
    g = gen(8)
    table, blocks, pools = paged(g, kv, nkv, d, lens, page)
    acc = weights(g, "smooth", blocks, nkv * page).view(blocks, nkv, page)
    sp = torch.randint(0, 30000, (blocks, nkv, page), device="cuda", generator=g).int()
    want_acc, want_sp, want = acc.clone(), sp.clone(), [p.clone() for p in pools]
    for b, n in enumerate(lens):
        if n <= keep:
            continue
        t = torch.arange(n)
        blk, sl = table[b].long()[t // page].cuda(), (t % page).cuda()
        a, p = acc[blk, :, sl].T.cpu(), sp[blk, :, sl].T.cpu()
        for h, moves in enumerate(ref.evict(a, p, n, keep, recent, n - 1)):
            to, at = (torch.tensor([m[i] for m in moves], device="cuda") for i in (0, 1))
            for x in [want_acc, want_sp] + [w.view(blocks, nkv, page, d) for w in want]:
                x[blk[to], h, sl[to]] = x[blk[at], h, sl[at]]
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    attn.kv_evict_paged(*pools, acc, sp, table.cuda(), L, None, len(lens), table.shape[1], nkv, d, page,
                        keep, recent)
    assert torch.equal(raw(acc), raw(want_acc)) and torch.equal(sp, want_sp)
    for x, y in zip(pools, want):
        assert torch.equal(raw(x), raw(y))


@pytest.mark.parametrize("kv,nkv,d", [("f32", 8, 128), ("bf16", 8, 128), ("q8", 8, 128), ("bf16", 5, 6),
                                      ("q8", 3, 4), ("q8", 2, 512), ("f32", 1, 2), ("f32", 2, 510)])
def test_rows(gpu, kv, nkv, d):
    """Whole rows move, Q8 scales with them; the rest of the cache keeps its bits."""
    n, keep, recent, pos = 777, 600, 100, 776
    g = gen(d)
    acc, sp = weights(g, "smooth", nkv, n), torch.arange(n, device="cuda").int().repeat(nkv, 1)
    caches = [ref.make_cache(torch.randn(n, nkv, d, device="cuda", generator=g), kv)[0] for _ in range(2)]
    before = [cache_bits(c, kv, nkv, d).clone() for c in caches]
    moves = ref.evict(acc.cpu(), sp.cpu(), n, keep, recent, pos)
    attn.kv_evict(*caches, acc, sp, nkv, n, d, keep, recent, pos)
    for c, b in zip(caches, before):
        for h in range(nkv):
            to, at = (torch.tensor([m[i] for m in moves[h]], device="cuda") for i in (0, 1))
            b[to, h] = b[at, h]
        assert torch.equal(cache_bits(c, kv, nkv, d), b)


def paged(g, kv, nkv, d, lens, page, spare=4):
    need = [(n + page - 1) // page for n in lens]
    blocks = sum(need) + spare
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(blocks)).int()
    table = torch.full((len(lens), max(1, max(need))), 10 ** 6, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at:at + k]
        at += k
    size = nkv * page * (d + 4 if kv == "q8" else d)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "q8": torch.uint8}[kv]
    if kv == "q8":
        pools = [torch.randint(0, 255, (blocks, size), device="cuda", generator=g).to(dt) for _ in range(2)]
    else:
        pools = [torch.randn(blocks, size, device="cuda", generator=g).to(dt) for _ in range(2)]
    return table, blocks, pools


@pytest.mark.parametrize("kv,nkv,d,page", [("f32", 4, 64, 16), ("bf16", 8, 128, 16), ("q8", 8, 128, 16),
                                           ("q8", 4, 20, 1), ("bf16", 3, 34, 64)])
def test_paged(gpu, kv, nkv, d, page):
    """Sequences of every kind at once: none, one row, under the budget, over it."""
    lens, keep, recent = (0, 1, 100, 257, 64, 400, 99, 101), 100, 20
    g = gen(7)
    table, blocks, pools = paged(g, kv, nkv, d, lens, page)
    B = len(lens)
    acc = weights(g, "ties", blocks, nkv * page).view(blocks, nkv, page)
    sp = torch.randint(0, 500, (blocks, nkv, page), device="cuda", generator=g).int()
    pos = torch.tensor([n + 3 * b for b, n in enumerate(lens)], dtype=torch.int32)
    want_acc, want_sp, want = acc.clone(), sp.clone(), [p.clone() for p in pools]
    for b, n in enumerate(lens):
        if n <= keep:
            continue
        t = torch.arange(n)
        blk, sl = table[b].long()[t // page], t % page
        a, p = acc[blk.cuda(), :, sl.cuda()].T.cpu(), sp[blk.cuda(), :, sl.cuda()].T.cpu()
        for h, moves in enumerate(ref.evict(a, p, n, keep, recent, int(pos[b]))):
            for to, at in moves:
                T, A = (int(blk[to]), h, int(sl[to])), (int(blk[at]), h, int(sl[at]))
                want_acc[T], want_sp[T] = want_acc[A], want_sp[A]
                for x in want:
                    rows = x[:, :nkv * page * d].view(blocks, nkv, page, d)
                    rows[T] = rows[A]
                    if kv == "q8":
                        sc = x[:, nkv * page * d:].view(blocks, nkv, page, 4)
                        sc[T] = sc[A]
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    attn.kv_evict_paged(*pools, acc, sp, table.cuda(), L, pos.cuda(), B, table.shape[1], nkv, d, page,
                        keep, recent)
    assert torch.equal(raw(acc), raw(want_acc)) and torch.equal(sp, want_sp)
    for x, y in zip(pools, want):
        assert torch.equal(raw(x), raw(y))


def test_track(gpu):
    nkv, cap, n, M, pos = 5, 90, 80, 13, 444
    acc, sp = torch.ones(nkv, cap, device="cuda"), torch.full((nkv, cap), -1, dtype=torch.int32, device="cuda")
    attn.kv_track(acc, sp, nkv, n, M, pos)
    t = torch.arange(cap, device="cuda")
    new = (t >= n - M) & (t < n)
    assert torch.equal(acc, torch.where(new, 0.0, 1.0).expand(nkv, cap))
    assert torch.equal(sp, torch.where(new, pos - (n - 1 - t), -1).int().expand(nkv, cap))
    attn.kv_track(acc, None, nkv, n, n, pos)  # positions are optional
    assert torch.count_nonzero(acc[:, :n]) == 0 and (acc[:, n:] == 1).all()


def test_track_paged(gpu):
    nkv, page, lens, M = 3, 8, (0, 1, 8, 30, 5), 9
    table, blocks, _ = paged(gen(3), "f32", nkv, 2, lens, page)
    acc = torch.ones(blocks, nkv, page, device="cuda")
    sp = torch.full((blocks, nkv, page), -1, dtype=torch.int32, device="cuda")
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pos = L + 70
    want_a, want_p = acc.clone(), sp.clone()
    for b, n in enumerate(lens):
        for t in range(max(0, n - M), n):
            want_a[table[b, t // page], :, t % page] = 0.0
            want_p[table[b, t // page], :, t % page] = n + 70 - (n - 1 - t)
    attn.kv_track_paged(acc, sp, table.cuda(), L, pos, len(lens), table.shape[1], M, nkv, page)
    assert torch.equal(acc, want_a) and torch.equal(sp, want_p)


def test_long_cache_offsets(gpu):
    """Row offsets past 2^31 bytes."""
    nkv, d, n = 8, 512, 140000  # 4.3 GB fp32 (offsets past 2^32)
    K = torch.zeros(n, nkv * d, device="cuda")
    K[:, 0] = torch.arange(n, device="cuda")
    V = torch.full((n, nkv * d), 2.0, device="cuda")
    V[:, -1] = torch.arange(n, device="cuda")
    g = gen(1)
    acc, sp = weights(g, "smooth", nkv, n), torch.arange(n, device="cuda").int().repeat(nkv, 1)
    keep, recent = n - 700, 700
    moves = ref.evict(acc.cpu(), sp.cpu(), n, keep, recent, n - 1)
    attn.kv_evict(K, V, acc, sp, nkv, n, d, keep, recent, n - 1)
    for h, x, col in ((0, K, 0), (nkv - 1, V, nkv * d - 1)):
        want = torch.arange(n, device="cuda").float()
        to, at = (torch.tensor([m[i] for m in moves[h]], device="cuda") for i in (0, 1))
        assert len(to) == 700
        want[to] = want[at]
        assert torch.equal(x[:, col], want)


def test_graph_replays(gpu):
    """Track and evict, captured: each replay does what the eager calls do."""
    nkv, d, n, keep, recent = 8, 128, 3000, 2500, 600
    g = gen(5)
    acc0, sp0 = weights(g, "ties", nkv, n), torch.arange(n, device="cuda").int().repeat(nkv, 1)
    K0 = torch.randn(n, nkv * d, device="cuda", generator=g)
    V0 = torch.randn(n, nkv * d, device="cuda", generator=g)
    bufs = [x.clone() for x in (K0, V0, acc0, sp0)]

    def reset():
        for x, y in zip(bufs, (K0, V0, acc0, sp0)):
            x.copy_(y)

    def calls():
        attn.kv_track(bufs[2], bufs[3], nkv, n, 500, n + 99)
        attn.kv_evict(*bufs, nkv, n, d, keep, recent, n + 99)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        calls()
    torch.cuda.synchronize()
    want = [x.clone() for x in bufs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        calls()
    for _ in range(3):
        reset()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(bufs, want):
            assert torch.equal(x, y)
        reset()
        calls()
        torch.cuda.synchronize()
        for x, y in zip(bufs, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("kv", KVS)
def test_a_stream_on_a_budget(gpu, kv):
    """A prompt, then steps whose weights drive evictions, then more steps: every
    step's output is the attention over the tokens that are left, each at its own
    position, and the books (acc, positions) are those of the tokens."""
    nq, nkv, d, M, budget, slack, recent, steps = 8, 4, 64, 90, 64, 16, 12, 60
    G, scale, cap = nq // nkv, 0.125, M + 4
    g = gen(77)
    inv = attn.rope_inv_freq(10000.0, d).cuda()
    row = nkv * d if kv != "q8" else nkv * d + (4 * nkv + 15) // 16 * 16
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "q8": torch.uint8}[kv]
    K, V = (torch.zeros(cap, row, dtype=dt, device="cuda") for _ in range(2))
    acc, sp = torch.zeros(nkv, cap, device="cuda"), torch.zeros(nkv, cap, dtype=torch.int32, device="cuda")
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    O = torch.empty(M, nq, d, device="cuda")
    attn.prefill_step_scored(3 * rnd(M, nq, d), rnd(M, nkv, d), rnd(M, nkv, d), K, V, O, nq, nkv, d, M,
                             0, 0, inv, scale, 0, 50.0)
    attn.kv_track(acc, sp, nkv, M, M, M - 1)
    # the tokens of every KV head: position -> (k row, v row, weight), in 64 bits
    Kv, Vv = ref.cache_values(K, kv, nkv, d), ref.cache_values(V, kv, nkv, d)
    book = [{t: [Kv[t, h], Vv[t, h], 0.0] for t in range(M)} for h in range(nkv)]
    n, pos = M, M
    o = torch.empty(nq, d, device="cuda")
    for step in range(steps):
        if n >= budget + slack:
            attn.kv_evict(K, V, acc, sp, nkv, n, d, budget, recent, pos - 1)
            n = budget
            # the weights are the GPU's own: its choice is checked against the rule on them
            for h in range(nkv):
                left = set(sp[h, :n].tolist())
                gone = [t for t in book[h] if t not in left]
                assert len(left) == n and left <= set(book[h])
                kept = [book[h][t][2] for t in left if t <= pos - 1 - recent]
                assert all(t <= pos - 1 - recent for t in gone)
                if gone and kept:
                    assert max(book[h][t][2] for t in gone) <= min(kept) + 1e-4
                for t in gone:
                    del book[h][t]
        q = 3 * rnd(nq, d)
        attn.decode_step_scored(q, rnd(nkv, d), rnd(nkv, d), K, V, o, nq, nkv, d, n, pos, inv, scale, 0,
                                50.0, None, acc, sp)
        n += 1
        Kv, Vv = ref.cache_values(K, kv, nkv, d), ref.cache_values(V, kv, nkv, d)
        for h in range(nkv):
            book[h][pos] = [Kv[n - 1, h], Vv[n - 1, h], 0.0]
            assert sorted(sp[h, :n].tolist()) == sorted(book[h])
            toks = sorted(book[h])
            Kh = torch.stack([book[h][t][0] for t in toks])[:, None]
            Vh = torch.stack([book[h][t][1] for t in toks])[:, None]
            qh = q[h * G:(h + 1) * G][None]
            zero, end = torch.tensor([0], device="cuda"), torch.tensor([len(toks)], device="cuda")
            want, p = ref.attend(qh, Kh, Vh, scale, end - 1, zero, end, 50.0)
            tol = ref.tolerance(qh, Kh, Vh, scale, 50.0, None, n)
            err = float((o[h * G:(h + 1) * G].double() - want[0]).abs().max())
            assert err <= tol, (step, h, err, tol)
            for t, w in zip(toks, p[0].sum(0).tolist()):
                book[h][t][2] += w
            by_pos = {int(x): float(w) for x, w in zip(sp[h, :n], acc[h, :n])}
            assert max(abs(by_pos[t] - book[h][t][2]) for t in toks) < 2e-4
        pos += 1
