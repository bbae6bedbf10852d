"""Ragged batches on the GPU against 64 bits (tests/ragged_ref.py): attention of packed
rows, their norms, RoPE and append, and both as a layer's step."""
from __future__ import annotations

import math

import pytest
import torch

import ragged_ref as rr
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


def close(got, want, tol):
    assert torch.isfinite(got).all()
    err = float((got.double() - want).abs().max()) if want.numel() else 0.0
    assert err <= tol, f"error {err:.3g}, bound {tol:.3g}"


def attend(b, q, nq, scale, window=0, softcap=0.0, slopes=None, O=None):
    O = torch.full((b.T, nq, b.d), math.nan, device="cuda") if O is None else O
    attn.attn_ragged(q, b.K, b.V, O, *b.args(), nq, b.nkv, b.d, b.page, scale, window, softcap, slopes)
    return O


def run(kv, nq, nkv, d, counts, cached, page=16, window=0, softcap=0.0, alibi=False, pad=0, seed=5,
        fill=None, sigma=2.0):
    g = gen(seed)
    if kv == "q8" and (nkv * page) % 4:
        page = 4
    b = rr.Batch(g, kv, nkv, d, counts, cached, page, pad, fill=fill)
    q = randn(g, b.T, nq, d, sigma=sigma)
    sl = attn.alibi_slopes(nq).cuda() if alibi else None
    scale = 1 / math.sqrt(d)
    O = attend(b, q, nq, scale, window, softcap, sl)
    want, tol = b.attend(q, scale, window, softcap, sl)
    close(O[:b.rows], want, tol)
    assert torch.isnan(O[b.rows:]).all()  # rows behind the last are left as they were
    return b, q, O


# (nq, nkv, d, page): groups of 1 to 16, padded and odd head dims
LAYERS = [(32, 8, 128, 16), (8, 8, 64, 16), (12, 4, 96, 16), (8, 4, 256, 16), (64, 8, 128, 32), (16, 1, 64, 4),
          (6, 2, 128, 1), (5, 1, 72, 8), (7, 7, 200, 128)]
# counts, cached: one token each, drafts, prompts, all of them, empty ones between
MIXES = [
    ([1], [0]),
    ([1], [1]),
    ([1, 1, 1], [0, 31, 32]),
    ([1] * 9, [5, 700, 0, 33, 64, 1500, 1, 255, 256]),
    ([5, 5, 5, 5], [100, 3, 900, 0]),
    ([0, 3, 0, 0, 17, 1, 0], [40, 0, 0, 9, 500, 64, 2]),
    ([33], [0]),
    ([129], [70]),
    ([300, 1, 8, 1], [0, 1000, 90, 31]),
    ([64, 200, 31, 2], [513, 0, 0, 5]),
]


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("nq,nkv,d,page", LAYERS)
def test_mixes(gpu, kv, nq, nkv, d, page):
    for i, (counts, cached) in enumerate(MIXES):
        run(kv, nq, nkv, d, counts, cached, page, pad=i % 3, seed=i)


@pytest.mark.parametrize("kv,nq,nkv,d", [("f32", 4, 2, 34), ("bf16", 4, 2, 90), ("q8", 4, 2, 36),
                                         ("f32", 8, 2, 512), ("bf16", 8, 2, 512), ("q8", 8, 2, 512),
                                         ("bf16", 2, 1, 2), ("f32", 3, 1, 300), ("q8", 4, 4, 260)])
def test_other_head_dims(gpu, kv, nq, nkv, d):
    run(kv, nq, nkv, d, [1, 0, 40, 5], [300, 7, 0, 31], pad=2)
    run(kv, nq, nkv, d, [9, 1], [20, 3000], softcap=30.0, alibi=True, window=100)


@pytest.mark.parametrize("window,softcap,alibi", [(1, 0.0, False), (7, 0.0, False), (100, 50.0, False),
                                                  (64, 0.0, True), (0, 50.0, True), (0, 20.0, False),
                                                  (0, 0.0, True), (100000, 0.0, False)])
@pytest.mark.parametrize("kv,nq,nkv,d", [("f32", 32, 8, 128), ("bf16", 32, 8, 128), ("q8", 8, 8, 64),
                                         ("bf16", 8, 4, 256)])
def test_scores_and_windows(gpu, kv, nq, nkv, d, window, softcap, alibi):
    run(kv, nq, nkv, d, [1, 70, 4, 260, 1], [1200, 0, 333, 90, 0], window=window, softcap=softcap,
        alibi=alibi, sigma=6.0 if softcap else 2.0)


@pytest.mark.parametrize("kv,counts,cached", [("bf16", [1], [40000]), ("q8", [4, 1], [30000, 12]),
                                              ("f32", [1, 600], [20000, 0]), ("bf16", [17, 300], [33000, 50])])
def test_long_contexts_are_split(gpu, kv, counts, cached):
    run(kv, 16, 2, 128, counts, cached)


def test_a_batch_of_many_sequences(gpu):
    """More sequences than the plan's LDS holds, most of them of no rows or one."""
    counts = [i % 3 % 2 for i in range(4500)]
    counts[7], counts[4400] = 90, 40
    run("bf16", 4, 2, 64, counts, [i % 40 for i in range(4500)])


@pytest.mark.parametrize("kv", ("f32", "bf16"))
def test_slots_that_hold_no_row(gpu, kv):
    """Pages end inside a tile, and what lies past a sequence's rows counts for nothing."""
    for fill in (math.nan, math.inf, 3e38):
        run(kv, 8, 2, 128, [1, 40, 3], [70, 5, 500], fill=fill)
        run(kv, 8, 4, 256, [1, 40, 3], [70, 5, 500], fill=fill)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("kv,d", [("f32", 128), ("bf16", 128), ("bf16", 64), ("f32", 256), ("bf16", 512)])
def test_rows_before_one_that_is_not_finite(gpu, kv, d, value):
    """K or V of a slot holds infinities or NaN: the rows that do not attend it stay exact."""
    counts, cached = [200, 1, 1], [10, 300, 40]
    for which in ("K", "V"):
        g = gen(3)
        b = rr.Batch(g, kv, 2, d, counts, cached)
        q = randn(g, b.T, 8, d)
        t = 150  # a slot of the first sequence's own rows
        pool = getattr(b, which).view(b.blocks, 2, 16, d)
        pool[int(b.table[0, t // 16]), :, t % 16, 5] = value
        O = attend(b, q, 8, 0.1)
        want, tol = b.attend(q, 0.1)  # of the values as they were
        keep = torch.ones(b.rows, dtype=torch.bool, device="cuda")
        keep[t - 10:200] = False
        close(O[keep], want[keep], tol)
        if which == "V":
            assert not torch.isfinite(O[~keep][:, :, 5]).any()
            other = torch.arange(d, device="cuda") != 5
            close(O[~keep][:, :, other], want[~keep][:, :, other], tol)


def test_query_rows_that_are_not_finite(gpu):
    g = gen(4)
    for kv, cached in (("f32", 60), ("bf16", 60), ("bf16", 9000)):
        b = rr.Batch(g, kv, 2, 128, [70, 1], [cached, 5])
        q = randn(g, b.T, 8, 128)
        q[3, 1, 7] = math.nan
        O = attend(b, q, 8, 0.1)
        assert torch.isnan(O[3, 1]).all()
        q[3, 1, 7] = 0.0
        want, tol = b.attend(q, 0.1)
        keep = torch.ones(71, 8, dtype=torch.bool, device="cuda")
        keep[3, 1] = False
        close(O[keep], want[keep], tol)


@pytest.mark.parametrize("kv", KVS)
def test_scales_far_apart(gpu, kv):
    """Rows of K and V of very different sizes: each keeps its own precision."""
    g = gen(6)
    b = rr.Batch(g, kv, 2, 128, [90, 1, 4], [40, 300, 64])
    if kv == "q8":
        sc = b.V[:, 2 * 16 * 128:].view(torch.float32)
        sc *= torch.exp2(torch.randint(-20, 20, sc.shape, device="cuda", generator=g).float())
    else:
        v = b.V.view(-1, 128)
        v *= torch.exp2(torch.randint(-20, 20, (v.shape[0], 1), device="cuda", generator=g).float())
    q = randn(g, b.T, 8, 128)
    V = b.values(b.V)
    O = attend(b, q, 8, 0.1)
    want, tol = b.attend(q, 0.1, V=V)
    close(O, want, tol)


def test_lengths_past_the_bound(gpu):
    """Slots from max_len on are left out; a row behind them sees those before."""
    g = gen(7)
    b = rr.Batch(g, "bf16", 2, 64, [5, 40], [100, 0])
    q = randn(g, b.T, 4, 64)
    b.max_len = 30
    O = attend(b, q, 4, 0.1)
    b2 = rr.Batch(gen(7), "bf16", 2, 64, [5, 40], [100, 0])
    K = [x[:30] for x in b2.kval]
    V = [x[:30] for x in b2.vval]
    for s, (n, c) in enumerate(((100, 5), (0, 40))):
        pos = torch.arange(n, n + c, device="cuda")
        want, _ = ref.attend(q[b.starts[s]:b.starts[s + 1]], K[s], V[s], 0.1, pos, torch.zeros_like(pos),
                             (pos + 1).clamp(max=30))
        close(O[b.starts[s]:b.starts[s + 1]], want, ref.tolerance(q, K[s], V[s], 0.1, 0.0, None, 0))


def test_index_arrays_that_hold_anything(gpu):
    """Garbage lengths, starts and block ids are not followed out of the arrays."""
    g = gen(8)
    b = rr.Batch(g, "bf16", 2, 128, [3, 40, 1], [10, 100, 700])
    q = randn(g, b.T, 8, 128)
    keep = (b.table.clone(), b.kv_lens.clone(), b.row_start.clone())
    big = 2 ** 31 - 1
    for table, lens, start in ((big, None, None), (-1, None, None), (None, big, None), (None, -big, None),
                               (None, 2, None), (None, None, [0, big, 5, 44]), (None, None, [-9, 3, 2, 1]),
                               (None, None, [40, 40, 44, 60])):
        b.table, b.kv_lens, b.row_start = (x.clone() for x in keep)
        if table is not None:
            b.table.fill_(table)
        if lens is not None:
            b.kv_lens.fill_(lens)
        if start is not None:
            b.row_start.copy_(torch.tensor(start))
        attend(b, q, 8, 0.1)
    torch.cuda.synchronize()
    b.table, b.kv_lens, b.row_start = keep
    want, tol = b.attend(q, 0.1)
    close(attend(b, q, 8, 0.1), want, tol)


def test_offsets_past_32_bits(gpu):
    """Pages whose rows lie more than 2^32 bytes, and elements, into the pool."""
    nkv, d, page = 8, 128, 16
    blocks = 2 ** 32 // (nkv * d * page) + 40
    g = gen(9)
    K = torch.zeros(blocks, nkv * page * d, dtype=torch.bfloat16, device="cuda")
    V = torch.zeros_like(K)
    b = rr.Batch(g, "bf16", nkv, d, [40, 1, 3], [0, 200, 30], page, spare=0)
    n = b.blocks
    K[-n:], V[-n:] = b.K, b.V
    live = b.table >= 0
    b.table[live] += blocks - n
    b.K, b.V, b.blocks = K, V, blocks
    q = randn(g, b.T, 32, d)
    want, tol = b.attend(q, 0.1)
    close(attend(b, q, 32, 0.1), want, tol)


# --- norms, RoPE and append ---------------------------------------------------


def rotated(x, pos, freq, weight=None, eps=1e-6):
    """Rows [T][heads][d] normed and rotated in 64 bits (the angle a product in 32)."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    if freq is None:
        return x
    ang = (pos.float()[:, None, None] * freq).double()
    a, c = x.chunk(2, -1)
    return torch.cat([a * ang.cos() - c * ang.sin(), a * ang.sin() + c * ang.cos()], -1)


def slots_of(b):
    """Positions and places in the pool of the new rows."""
    pos, at = [], []
    for s in range(b.B):
        for t in range(b.cached[s], b.cached[s] + b.counts[s]):
            pos.append(t)
            at.append(int(b.table[s, t // b.page]) * b.page + t % b.page)
    more = b.T - b.rows
    i32 = dict(dtype=torch.int32, device="cuda")
    return torch.tensor(pos + [0] * more, **i32), torch.tensor(at + [-1] * more, **i32)


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("nq,nkv,d,page", LAYERS + [(4, 2, 36, 2), (8, 2, 512, 16), (9, 3, 4, 4)])
def test_append(gpu, kv, nq, nkv, d, page):
    if kv == "q8" and (nkv * page) % 4:
        page = 4
    g = gen(d)
    b = rr.Batch(g, kv, nkv, d, [1, 0, 37, 4], [0, 3, 61, 1000], page, pad=3)
    pos, at = slots_of(b)
    freq = (1e4 ** (-torch.arange(0, d, 2, device="cuda") / d)).float()
    q, kn, vn = randn(g, b.T, nq, d), randn(g, b.T, nkv, d), randn(g, b.T, nkv, d)
    qn, kw = 1 + 0.1 * randn(g, d), 1 + 0.1 * randn(g, d)
    for norms, table in ((False, freq), (True, freq), (True, None)):
        Q, K, V = q.clone(), b.K.clone(), b.V.clone()
        attn.rope_append_ragged(Q, kn, vn, K, V, pos, at, b.T, b.blocks, nq, nkv, d, page, table,
                                qn if norms else None, kw if norms else None, norms, 1e-6)
        want = rotated(q, pos, table, qn if norms else None)
        # a norm's factor, weight, and two products and their sum: 2^-24 each, and the sine's
        close(Q[:b.rows], want[:b.rows], 10 * ref.EPS32 * float(want.abs().max()))
        assert torch.equal(Q[b.rows:], q[b.rows:])
        k = rotated(kn, pos, table, kw if norms else None)[:b.rows]
        v = vn.double()[:b.rows]
        if norms:
            v = v / (v.pow(2).mean((-1, -2), keepdim=True) + 1e-6).sqrt()
        step = {"f32": 0.0, "bf16": 2.0 ** -8, "q8": 0.5 / 127 * (1 + 1e-5)}[kv]
        for pool, was, x in ((K, b.K, k), (V, b.V, v)):
            got = torch.cat([r[n:] for r, n in zip(b.values(pool), b.cached)])
            tol = 10 * ref.EPS32 * x.abs().amax(-1, keepdim=True)
            tol = tol + step * (x.abs() if kv == "bf16" else x.abs().amax(-1, keepdim=True))
            assert ((got - x).abs() <= tol).all()
            # nothing else of the pool is written
            put = torch.zeros(b.blocks * page, dtype=torch.bool, device="cuda")
            put[at[:b.rows].long()] = True
            keep = ~put.view(b.blocks, page)
            if kv == "q8":
                cut = nkv * page * d
                for c, w in ((slice(0, cut), d), (slice(cut, None), 4)):
                    x0, x1 = (p[:, c].reshape(b.blocks, nkv, page, w).transpose(1, 2)[keep] for p in (pool, was))
                    assert torch.equal(x0, x1)
            else:
                x0, x1 = (p.view(b.blocks, nkv, page, d).transpose(1, 2)[keep] for p in (pool, was))
                assert torch.equal(x0, x1)


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 128), (8, 4, 256), (8, 8, 64)])
def test_append_agrees_with_the_prompts_own(gpu, kv, nq, nkv, d):
    """prefill_step_paged's rows, to the roundings of either: a norm, a weight, two products
    and their sum in fp32, then the cache type's (which may fall to either side)."""
    g = gen(2)
    b = rr.Batch(g, kv, nkv, d, [33], [50])
    pos, at = slots_of(b)
    freq = attn.rope_inv_freq(1e4, d).cuda()
    q, kn, vn = randn(g, 33, nq, d), randn(g, 33, nkv, d), randn(g, 33, nkv, d)
    qn, kw = 1 + 0.1 * randn(g, d), 1 + 0.1 * randn(g, d)
    Q, K, V = q.clone(), b.K.clone(), b.V.clone()
    attn.rope_append_ragged(Q, kn, vn, K, V, pos, at, 33, b.blocks, nq, nkv, d, 16, freq, qn, kw, True, 1e-6)
    attn.prefill_step_paged(q, kn, vn, b.K, b.V, torch.empty_like(q), b.table[0].clamp(min=0), b.width, 16,
                            nq, nkv, d, 33, 50, 50, freq, 0.1, 0, qn, kw, True, 1e-6)
    close(Q, q.double(), 20 * ref.EPS32 * float(q.abs().max()))
    step = {"f32": 0.0, "bf16": 2.0 ** -7, "q8": 1.0 / 127 * (1 + 1e-5)}[kv] + 20 * ref.EPS32
    for mine, theirs in ((K, b.K), (V, b.V)):
        x, y = b.values(mine)[0], b.values(theirs)[0]
        assert ((x - y).abs() <= step * y.abs().amax(-1, keepdim=True)).all()
        assert torch.equal(x[:50], y[:50])


def test_queries_alone(gpu):
    g = gen(1)
    b = rr.Batch(g, "bf16", 2, 64, [4, 9], [20, 3], pad=2)
    pos, at = slots_of(b)
    freq = attn.rope_inv_freq(1e4, 64).cuda()
    q = randn(g, b.T, 8, 64)
    Q = q.clone()
    attn.rope_append_ragged(Q, None, None, None, None, pos, at, b.T, b.blocks, 8, 2, 64, 16, freq)
    close(Q[:13], rotated(q, pos, freq)[:13], 6 * ref.EPS32 * float(q.abs().max()) * 2)
    assert torch.equal(Q[13:], q[13:])


def test_slots_out_of_the_pool_are_not_stored(gpu):
    g = gen(1)
    b = rr.Batch(g, "f32", 2, 64, [5], [0])
    pos, at = slots_of(b)
    at[1], at[3] = b.blocks * 16, 2 ** 31 - 1
    q, kn = randn(g, 5, 4, 64), randn(g, 5, 2, 64)
    Q, K, V = q.clone(), b.K.clone(), b.V.clone()
    attn.rope_append_ragged(Q, kn, kn, K, V, pos, at, 5, b.blocks, 4, 2, 64, 16, None)
    was, got = b.values(b.K)[0], b.values(K)[0]
    for i in range(5):
        assert torch.equal(got[i], was[i] if i in (1, 3) else kn[i].double())


# --- a layer's step, and a run of all of them ---------------------------------


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("nq,nkv,d,window,softcap", [(32, 8, 128, 0, 0.0), (8, 4, 256, 64, 50.0),
                                                     (8, 8, 64, 0, 30.0), (8, 2, 512, 0, 0.0)])
def test_step(gpu, kv, nq, nkv, d, window, softcap):
    g = gen(13)
    b = rr.Batch(g, kv, nkv, d, [1, 60, 0, 5, 1], [700, 0, 4, 128, 31], pad=2)
    pos, at = slots_of(b)
    freq = attn.rope_inv_freq(1e4, d).cuda()
    q, kn, vn = randn(g, b.T, nq, d), randn(g, b.T, nkv, d), randn(g, b.T, nkv, d)
    qn, kw = 1 + 0.1 * randn(g, d), 1 + 0.1 * randn(g, d)
    O = torch.full((b.T, nq, d), math.nan, device="cuda")
    scale = 1 / math.sqrt(d)
    attn.step_ragged(q, kn, vn, b.K, b.V, O, *b.args()[:3], pos, at, *b.args()[3:], nq, nkv, d, 16, freq,
                     scale, window, softcap, None, qn, kw)
    want, tol = b.attend(q, scale, window, softcap, None, b.values(b.K), b.values(b.V))
    close(O[:b.rows], want, tol)
    assert torch.isnan(O[b.rows:]).all()


@pytest.mark.parametrize("kv", KVS)
def test_steps_of_a_sequence_alone_and_among_others(gpu, kv):
    """A row's result is that of its sequence by itself, to roundings."""
    nq, nkv, d = 16, 4, 128
    g = gen(21)
    b = rr.Batch(g, kv, nkv, d, [1, 150, 6], [900, 40, 77])
    q = randn(g, b.T, nq, d)
    O = attend(b, q, nq, 0.09)
    for s in range(3):
        rows = slice(b.starts[s], b.starts[s + 1])
        one = torch.empty(b.counts[s], nq, d, device="cuda")
        start = torch.tensor([0, b.counts[s]], dtype=torch.int32, device="cuda")
        attn.attn_ragged(q[rows].contiguous(), b.K, b.V, one, b.table[s:s + 1].contiguous(),
                         b.kv_lens[s:s + 1].contiguous(), start, b.counts[s], 1, b.width, b.blocks,
                         b.max_len, nq, nkv, d, 16, 0.09)
        _, tol = b.attend(q, 0.09)
        close(one, O[rows].double(), 2 * tol)


def test_decode_rows_agree_with_the_paged_decode(gpu):
    nq, nkv, d = 32, 8, 128
    for kv in KVS:
        g = gen(22)
        b = rr.Batch(g, kv, nkv, d, [1] * 12, [7, 100, 31, 32, 900, 2500, 0, 64, 63, 1, 333, 3])
        q = randn(g, b.T, nq, d)
        O, P = attend(b, q, nq, 0.09), torch.empty(12, nq, d, device="cuda")
        attn.attn_decode_paged(q, b.K, b.V, P, b.table.clamp(min=0), b.kv_lens, None, 12, b.width, nq, nkv, d,
                               16, 0.09)
        _, tol = b.attend(q, 0.09)
        close(O, P.double(), 2 * tol)


@pytest.mark.parametrize("kv", KVS)
def test_ticks_in_a_graph(gpu, kv):
    """Plan and two layers' steps captured once and replayed over growing sequences, one
    of them finished and begun anew, against the same sequences by themselves."""
    nq, nkv, d, page, width, B, T = 8, 2, 64, 4, 40, 4, 48
    num, i32 = 90, dict(dtype=torch.int32, device="cuda")
    g = gen(30)
    zeros = lambda *s: torch.zeros(*s, **i32)  # noqa: E731
    counts, done, lens, table = zeros(B), zeros(B), zeros(B), zeros(B, width)
    free, left = torch.arange(num, **i32), torch.tensor([num], **i32)
    start, seq, pos, at, status = zeros(B + 1), zeros(T), zeros(T), zeros(T), zeros(1)
    empty = rr.Batch(g, kv, nkv, d, [], [], page, spare=num)
    K, V = [empty.K.clone(), empty.K.clone()], [empty.K.clone(), empty.K.clone()]
    freq = attn.rope_inv_freq(1e4, d).cuda()
    x = randn(g, 2, T, nq + 2 * nkv, d)
    q, O = torch.empty(2, T, nq, d, device="cuda"), torch.empty(2, T, nq, d, device="cuda")

    def tick():
        attn.ragged_plan(counts, lens, lens, table, B, width, page, num, T, start, seq, pos, at, status, free,
                         left, left, done)
        for layer in range(2):
            q[layer].copy_(x[layer, :, :nq])
            kn, vn = (x[layer, :, nq + i * nkv:nq + (i + 1) * nkv].contiguous() for i in range(2))
            attn.step_ragged(q[layer], kn, vn, K[layer], V[layer], O[layer], table, lens, start, pos, at, T,
                             B, width, num, width * page, nq, nkv, d, page, freq, 0.125)

    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        tick()  # sizes the workspaces (no rows)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        tick()
    own = [0] * B
    for step, (new, off) in enumerate([([20, 1, 0, 9], [0] * 4), ([1, 1, 1, 1], [0] * 4),
                                       ([1, 30, 0, 4], [1, 0, 0, 0]), ([7, 1, 1, 0], [0, 0, 0, 1]),
                                       ([1, 1, 1, 1], [0] * 4), ([100, 0, 0, 0], [0] * 4), ([0, 2, 5, 1], [0] * 4)]):
        counts.copy_(torch.tensor(new, **i32))
        done.copy_(torch.tensor(off, **i32))
        x.copy_(randn(g, *x.shape))
        O.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        if sum(new) > T:
            assert int(status) == rr.E2BIG and torch.isnan(O).all() and lens.tolist() == own
            continue
        assert int(status) == 0
        own = [(0 if f else n) + c for n, c, f in zip(own, new, off)]
        assert lens.tolist() == own
        b = empty
        b.B, b.counts, b.cached = B, new, [n - c for n, c in zip(own, new)]
        b.table, b.starts = table, start.tolist()
        for layer in range(2):
            want, tol = b.attend(q[layer], 0.125, K=b.values(K[layer]), V=b.values(V[layer]))
            close(O[layer, :sum(new)], want, tol)
            assert torch.isnan(O[layer, sum(new):]).all()
            rows = rotated(x[layer, :, nq:nq + nkv], pos, freq)[:sum(new)]
            got = torch.cat([r[n - c:] for r, n, c in zip(b.values(K[layer]), own, new)])
            step_of = {"f32": 0.0, "bf16": 2.0 ** -8, "q8": 0.5 / 127 * (1 + 1e-5)}[kv]
            assert float((got - rows).abs().max()) <= (step_of + 6 * ref.EPS32) * float(rows.abs().max())


def test_capture_without_a_call_before_it_is_refused(gpu):
    g = gen(5)
    b = rr.Batch(g, "bf16", 2, 128, [1, 300], [70, 900])
    q = randn(g, b.T, 8, 128)
    O, s, graph = torch.empty_like(q), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with pytest.raises(_lib.MolotHipError) as e:
        with torch.cuda.graph(graph, stream=s):
            attend(b, q, 8, 0.1, O=O)
    assert e.value.status == _lib.ENOWS
    torch.cuda.synchronize()


def test_streams_at_once(gpu):
    """Calls on streams of their own, each with its own workspace, in turn and overlapping."""
    jobs = []
    for i in range(4):
        g = gen(40 + i)
        b = rr.Batch(g, "bf16", 2, 128, [1, 90 + i, 3], [5000, 20 * i, 64])
        q = randn(g, b.T, 8, 128)
        jobs.append((b, q, torch.cuda.Stream(), torch.empty_like(q)))
    torch.cuda.synchronize()
    for _ in range(5):
        for b, q, s, O in jobs:
            with torch.cuda.stream(s):
                attend(b, q, 8, 0.1, O=O)
    torch.cuda.synchronize()
    for b, q, s, O in jobs:
        want, tol = b.attend(q, 0.1)
        close(O, want, tol)


def test_two_graphs_of_one_stream(gpu):
    """Graphs captured one after the other share the stream's workspace and replay in turn."""
    jobs = []
    s = torch.cuda.Stream()
    for i, counts in enumerate(([1, 200], [40, 1, 1])):
        g = gen(50 + i)
        b = rr.Batch(g, "f32", 2, 128, counts, [3000, 40, 9][:len(counts)])
        jobs.append((b, randn(g, b.T, 8, 128), torch.empty(b.T, 8, 128, device="cuda"), torch.cuda.CUDAGraph()))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for b, q, O, _ in jobs:
            attend(b, q, 8, 0.1, O=O)
    torch.cuda.synchronize()
    for b, q, O, graph in jobs:
        with torch.cuda.graph(graph, stream=s):
            attend(b, q, 8, 0.1, O=O)
    with torch.cuda.stream(s):
        for _ in range(3):
            for b, q, O, graph in jobs:
                O.fill_(math.nan)
                graph.replay()
            for b, q, O, graph in jobs:
                want, tol = b.attend(q, 0.1)
                close(O, want, tol)
    torch.cuda.synchronize()


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 128), (4, 4, 64), (10, 2, 96), (8, 4, 256)])
def test_rows_about_a_narrow_tile(gpu, kv, nq, nkv, d):
    """Sequences whose rows just fill a narrow tile of 16 or 32, or two, or pass it: alone (partials of
    that many rows), long enough to be split, and beside others and wide tiles."""
    G = nq // nkv
    for R in (15, 16, 17, 31, 32, 33, 63, 64, 65):
        n = -(-R // G)
        run(kv, nq, nkv, d, [n], [5000])
        run(kv, nq, nkv, d, [n], [3], softcap=30.0, alibi=True)
        run(kv, nq, nkv, d, [n, 0, 1, n + 256 // G, n], [37, 9, 2000, 60, 1100], pad=3, window=700)


@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("d", (64, 128, 256))
def test_drafts_before_a_row_that_is_not_finite(gpu, d, value):
    """A draft's row that is not finite: the rows before it, in the same narrow tile, stay exact,
    and so do the other sequences."""
    for G, count in ((4, 5), (1, 20), (3, 5)):
        g = gen(4)
        b = rr.Batch(g, "bf16", 2, d, [count, 1, count], [2100, 300, 40])
        q = randn(g, b.T, 2 * G, d)
        t = 2100 + count - 2
        for which in ("K", "V"):
            pool = getattr(b, which).view(b.blocks, 2, 16, d)
            at = (int(b.table[0, t // 16]), slice(None), t % 16, 3)
            was = pool[at].clone()
            pool[at] = value
            O = attend(b, q, 2 * G, 0.1)
            pool[at] = was
            want, tol = b.attend(q, 0.1)
            keep = torch.ones(b.rows, dtype=torch.bool, device="cuda")
            keep[count - 2:count] = False
            close(O[keep], want[keep], tol)
            if which == "V":
                assert not torch.isfinite(O[~keep]).all()


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("d", (34, 320, 512))
def test_split_rows_on_the_vector_alu(gpu, kv, d):
    """Head dims off the matrix cores: long rows split in many units, all masks, slots past the end."""
    d = d if kv != "q8" else (d + 3) // 4 * 4
    run(kv, 8, 2, d, [1, 6, 0, 2], [6000, 700, 3, 1], pad=1)
    run(kv, 8, 2, d, [1, 6, 0, 2], [6000, 700, 3, 1], window=65, softcap=20.0, alibi=True)
    if kv != "q8":
        run(kv, 8, 2, d, [1, 5], [66, 0], fill=math.nan)


def test_one_graph_serves_smaller_ticks(gpu):
    """Captured at its bounds, replayed over lengths that change between the replays: one row,
    drafts and prompt parts by turns, each as the eager call has it."""
    nq, nkv, d = 8, 2, 128
    g = gen(9)
    b = rr.Batch(g, "bf16", nkv, d, [300, 5, 1], [900, 1500, 40])
    q = randn(g, b.T, nq, d)
    O = torch.zeros_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        attend(b, q, nq, 0.1, O=O)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        attend(b, q, nq, 0.1, O=O)
    starts, lens = b.row_start.clone(), b.kv_lens.clone()
    for counts in ([300, 5, 1], [1, 1, 1], [5, 5, 0], [0, 0, 0], [40, 1, 8], [300, 5, 1]):
        now = [0]
        for c in counts:
            now.append(now[-1] + c)
        b.row_start.copy_(torch.tensor(now, dtype=torch.int32))
        b.kv_lens.copy_(lens - torch.tensor([300 - counts[0], 5 - counts[1], 1 - counts[2]],
                                            dtype=torch.int32, device="cuda").clamp(min=0))
        O.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = O.clone()
        want = attend(b, q, nq, 0.1, O=torch.full_like(q, 7.0))
        torch.cuda.synchronize()
        assert (got[now[-1]:] == 7.0).all()
        # (the same kernels over the same lengths: at most another order of a tile's units)
        assert float((got - want).abs().max()) <= 1e-6 * max(1.0, float(want.abs().max()))
    b.row_start.copy_(starts)
    b.kv_lens.copy_(lens)
