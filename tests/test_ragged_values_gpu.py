"""Ragged attention over rows of very different sizes, each output against a bound of its
own terms in 64 bits: small rows beside large ones keep their precision."""
from __future__ import annotations

import math

import pytest
import torch

import ragged_ref as rr
from molot_amd import attn

pytestmark = pytest.mark.gpu

LAYERS = [("f32", 128), ("bf16", 128), ("q8", 128), ("f32", 64), ("bf16", 64), ("q8", 64), ("f32", 256),
          ("bf16", 256), ("q8", 256), ("f32", 512), ("bf16", 512), ("q8", 512)]
EPS = 2.0 ** -24
# prompts, drafts and single tokens at every phase of a run of rows
COUNTS = [200, 1, 5, 1, 1, 70, 5, 1, 1, 1, 1]
CACHED = [10, 300, 77, 40, 42, 500, 9, 1100, 1101, 1106, 1109]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def scaled(b, pool, exps, inside=None):
    """The pool with slot t of sequence s times 2^exps[s][t], and inside[s][t] (d factors)."""
    nkv, d, page = b.nkv, b.d, b.page
    if b.kv == "q8":
        rows = pool[:, nkv * page * d:].view(torch.float32).view(-1, nkv, page, 1)
    else:
        rows = pool.view(-1, nkv, page, d)
    rows = rows.clone()
    for s, e in enumerate(exps):
        t = torch.arange(len(e), device="cuda")
        at, sl = b.table[s].long()[t // page], t % page
        f = torch.exp2(e)[:, None, None]
        if inside is not None:
            f = f * inside[s][:, None]
        rows[at, :, sl] = (rows[at, :, sl].double() * f.double()).to(rows.dtype)
    if b.kv == "q8":
        pool[:, nkv * page * d:] = rows.reshape(pool.shape[0], -1).view(torch.uint8)
    else:
        pool.copy_(rows.view(pool.shape))


def bounds(b, q, K, V, scale, window):
    """For every sequence with rows: o [c][nq][d] in 64 bits and how far an output may be off.

    A product's factors are two 16-bit pieces (2^-22 of an element each), or smaller than
    2^-16 of their row's largest and then off by 2^-39 of that (bf16: below 2^-29 and then off
    by that, one piece): a score is off by 2^-21 of A = sum |q k| scale, the row's floor (F) times
    d |q| |k| at their largest, and by the roundings of its 3 d / 16 sums and the four after it.
    A probability moves by twice that of itself, and exp, a sum over n keys and a merge of 8
    groups and some units round it: n + 40 of 2^-24 in all; P's and V's pieces 2^-21 and their
    floors, n F of V's largest."""
    F = 2.0 ** (-28 if b.kv == "bf16" else -36)
    out = []
    for s, (n0, c) in enumerate(zip(b.cached, b.counts)):
        if not c:
            continue
        n, G, d = n0 + c, q.shape[1] // b.nkv, b.d
        x = q[b.starts[s]:b.starts[s + 1]].double()
        t, slot = torch.arange(n, device="cuda"), torch.arange(n0, n, device="cuda")[:, None]
        seen = (t <= slot) & (t > slot - window) if window else t <= slot
        o, tol = torch.zeros(x.shape, dtype=torch.float64, device="cuda"), torch.zeros_like(x)
        for h in range(x.shape[1]):
            k, v, y = K[s][:, h // G], V[s][:, h // G], x[:, h]
            p = (y @ k.T * scale).masked_fill(~seen, -math.inf).softmax(-1)
            A = (y.abs() @ k.abs().T * scale * seen).amax(-1)
            top = (y.abs().amax(-1)[:, None] * k.abs().amax(-1) * seen).amax(-1) * d * scale
            ds = A * (2.0 ** -21 + (3 * d / 16 + 4) * EPS) + F * top
            vtop = (v.abs().amax(-1) * seen).amax(-1)
            many = seen.sum(-1).double()
            o[:, h] = p @ v
            tol[:, h] = ((2 * ds + 2.0 ** -21 + (many + 40) * EPS)[:, None] * (p @ v.abs())
                         + (many * F * vtop)[:, None])
        out.append((s, o, tol))
    return out


def check(b, O, want, rows=None):
    for s, o, tol in want:
        got = O[b.starts[s]:b.starts[s + 1]].double()
        assert torch.isfinite(got).all()
        bad = (got - o).abs() > tol
        if rows is not None:
            bad = bad[rows[s]]
        worst = float(((got - o).abs() / tol.clamp(min=1e-300))[rows[s] if rows is not None else slice(None)]
                      .max()) if bad.numel() else 0.0
        assert not bad.any(), f"sequence {s}: {int(bad.sum())} of {bad.numel()} outputs, {worst:.3g} of the bound"


def attend(b, q, nq, scale, window):
    O = torch.full((b.T, nq, b.d), math.nan, device="cuda")
    return attn.attn_ragged(q, b.K, b.V, O, *b.args(), nq, b.nkv, b.d, b.page, scale, window)


@pytest.mark.parametrize("kv,d", LAYERS)
@pytest.mark.parametrize("large", ("K", "V", "KV"))
def test_runs_of_small_and_large_rows(gpu, kv, d, large):
    """Runs of 8 slots 2^39 apart, in one tile: the query rows whose window lies in one run."""
    g, nq, nkv, window = gen(d), 8, 2, 5
    b = rr.Batch(g, kv, nkv, d, COUNTS, CACHED)
    q = torch.randn(b.T, nq, d, device="cuda", generator=g)
    exps, pure = [], []
    for s, (n0, c) in enumerate(zip(CACHED, COUNTS)):
        t = torch.arange(n0 + c, device="cuda")
        exps.append(torch.where(t // 8 % 2 == 0, -20.0, 19.0))
        at = t[n0:]
        pure.append((at - window + 1).clamp(min=0) // 8 == at // 8)
        if "K" in large:
            q[b.starts[s]:b.starts[s + 1]] *= torch.exp2(-exps[-1][n0:])[:, None, None]
    assert sum(int(x.sum()) for x in pure) > 100 and any(bool(x) for x in pure if x.numel() == 1)
    for name in large:
        scaled(b, getattr(b, name), exps)
    want = bounds(b, q, b.values(b.K), b.values(b.V), d ** -0.5, window)
    check(b, attend(b, q, nq, d ** -0.5, window), want, pure)


@pytest.mark.parametrize("kv,d", LAYERS)
def test_sequences_of_small_and_large_rows(gpu, kv, d):
    """Whole sequences 2^30 apart, K against V, without a window."""
    g, nq, nkv = gen(d + 1), 8, 2
    b = rr.Batch(g, kv, nkv, d, COUNTS, CACHED)
    q = torch.randn(b.T, nq, d, device="cuda", generator=g)
    ke = [torch.full((n + c,), 15.0 if s % 2 else -15.0, device="cuda")
          for s, (n, c) in enumerate(zip(CACHED, COUNTS))]
    for s in range(b.B):
        q[b.starts[s]:b.starts[s + 1]] *= float(torch.exp2(-ke[s][0]))
    scaled(b, b.K, ke)
    scaled(b, b.V, [-x for x in ke])
    want = bounds(b, q, b.values(b.K), b.values(b.V), d ** -0.5, 0)
    check(b, attend(b, q, nq, d ** -0.5, 0), want)


@pytest.mark.parametrize("kv,d", [x for x in LAYERS if x[0] != "q8"])
def test_elements_of_a_row_far_apart(gpu, kv, d):
    """Elements of a row of K and V up to 2^40 apart: the small ones to the floor of their row."""
    g, nq, nkv = gen(d + 2), 8, 2
    b = rr.Batch(g, kv, nkv, d, COUNTS, CACHED)
    q = torch.randn(b.T, nq, d, device="cuda", generator=g)
    for pool in (b.K, b.V):
        zero = [torch.zeros(n + c, device="cuda") for n, c in zip(CACHED, COUNTS)]
        inside = [torch.exp2(-torch.randint(0, 41, (len(z), d), device="cuda", generator=g).float()) for z in zero]
        scaled(b, pool, zero, inside)
    want = bounds(b, q, b.values(b.K), b.values(b.V), 4 * d ** -0.5, 0)
    check(b, attend(b, q, nq, 4 * d ** -0.5, 0), want)
