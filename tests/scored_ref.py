"""Scored attention and the eviction in 64 bits, plainly: what the GPU tests of
tests/test_scored_gpu.py and tests/test_evict_gpu.py compare with."""
from __future__ import annotations

import math

import torch

PAGE = 16
EPS32 = 2.0 ** -24  # half a step of fp32, relative


def quantize(x):
    """Q8 rows of x[..., d] (quant.h:34-50): codes and fp32 scales."""
    s = x.abs().amax(-1) / 127.0
    s = torch.where(s > 0, s, torch.ones_like(s))
    return torch.clamp(torch.round(x / s[..., None]), -127, 127).to(torch.int8), s


def make_cache(x, kv):
    """A token-major cache of rows x[n][nkv][d] as the library holds them, and the
    values it stands for in 64 bits."""
    n, nkv, d = x.shape
    if kv == "f32":
        return x.reshape(n, nkv * d).contiguous(), x.double()
    if kv == "bf16":
        b = x.to(torch.bfloat16)
        return b.reshape(n, nkv * d).contiguous(), b.double()
    codes, s = quantize(x)
    row = nkv * d + (4 * nkv + 15) // 16 * 16
    out = torch.zeros(n, row, dtype=torch.uint8, device=x.device)
    out[:, :nkv * d] = codes.reshape(n, nkv * d).view(torch.uint8)
    out[:, nkv * d:nkv * d + 4 * nkv] = s.contiguous().view(torch.uint8)
    return out, codes.double() * s.double()[..., None]


def cache_values(c, kv, nkv, d):
    """The values of a token-major cache's rows [n][nkv][d] in 64 bits."""
    n = c.shape[0]
    if kv != "q8":
        return c.reshape(n, nkv, d).double()
    codes = c[:, :nkv * d].contiguous().view(torch.int8).view(n, nkv, d)
    s = c[:, nkv * d:nkv * d + 4 * nkv].contiguous().view(torch.float32)
    return codes.double() * s.double()[..., None]


def make_pages(x, kv, blocks, table, page=PAGE, fill=0.0):
    """Pages [blocks][nkv][page][d] that hold rows x[n][nkv][d] through the block
    ids of `table`; everything else is `fill`."""
    n, nkv, d = x.shape
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}.get(kv)
    if kv == "q8":
        pool = torch.zeros(blocks, nkv * page * (d + 4), dtype=torch.uint8, device=x.device)
    else:
        pool = torch.full((blocks, nkv * page * d), fill, dtype=dt, device=x.device)
    put_pages(pool, x, kv, table, page)
    return pool


def put_pages(pool, x, kv, table, page=PAGE):
    n, nkv, d = x.shape
    codes, s = quantize(x) if kv == "q8" else (None, None)
    for t in range(n):
        blk, sl = int(table[t // page]), t % page
        if kv == "q8":
            cut = nkv * page * d
            pool[blk, :cut].view(torch.int8).view(nkv, page, d)[:, sl] = codes[t]
            pool[blk, cut:].view(torch.float32).view(nkv, page)[:, sl] = s[t]
        else:
            pool[blk].view(nkv, page, d)[:, sl] = x[t].to(pool.dtype)


def scores(q, K, scale, pos, softcap, slopes):
    """[m][nq][n] scores of q[m][nq][d] at pos[m] over K[n][nkv][d], 64 bits."""
    m, nq, d = q.shape
    n, nkv = K.shape[:2]
    s = torch.empty(m, nq, n, dtype=torch.float64, device=q.device)
    for h in range(nq):
        s[:, h] = q[:, h].double() @ K[:, h // (nq // nkv)].T
    s *= scale
    if softcap > 0:
        s = softcap * (s / softcap).tanh()
    if slopes is not None:
        dist = (pos[:, None] - torch.arange(n, device=q.device)).abs().double()
        s -= slopes.double()[None, :, None] * dist[:, None]
    return s


def attend(q, K, V, scale, pos, lo, hi, softcap=0.0, slopes=None):
    """o[m][nq][d] and the weights [m][nq][n]: row i over keys [lo[i], hi[i])."""
    nq, nkv = q.shape[1], K.shape[1]
    t = torch.arange(K.shape[0], device=q.device)
    dead = (t < lo[:, None]) | (t >= hi[:, None])
    Kc = torch.nan_to_num(K) if dead.any() else K  # a masked key counts for nothing
    s = scores(q, Kc, scale, pos, softcap, slopes)
    s.masked_fill_(dead[:, None], -math.inf)
    p = s.softmax(-1)
    p[(lo >= hi)] = 0.0  # nothing to see: o = 0
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    seen = ~dead.all(0)
    for h in range(nq):
        o[:, h] = p[:, h][:, seen] @ torch.nan_to_num(V[:, h // (nq // nkv)][seen])
    return o, p


def tolerance(q, K, V, scale, softcap, slopes, reach):
    """Bound of max |o - exact| from the roundings, for finite inputs.

    A score's products are exact to 2^-21 of each (two 16-bit pieces a factor; fp32
    to 2^-24), their sum and the steps after it to a few 2^-24 of their size:
    |ds| <= A 2^-21 + 4 S 2^-24, A = max sum |q_e k_e| scale, S the largest |score|
    with its bias (`reach` the largest distance).  A probability then moves by 2 |ds|
    of itself (the row's sum moves too), an output by 2 |ds| max|V|, and its own sum
    rounds to 2^-21 of max|V| (pieces again; sums over rows average out: 8 2^-24)."""
    nq, nkv = q.shape[1], K.shape[1]
    G = nq // nkv
    A = 0.0
    for h in range(nq):
        A = max(A, float((q[:, h].double().abs() @ K[:, h // G].abs().T).max()) if K.shape[0] else 0.0)
    A *= abs(scale)
    S = min(A, softcap) if softcap > 0 else A
    if slopes is not None:
        # (far keys of steep heads have no weight left: a bias past 100 is e^-100)
        S += min(float(slopes.max()) * reach, 100.0 + A)
    vmax = float(V.abs().max()) if V.numel() else 0.0
    ds = A * 2.0 ** -21 + 4 * S * EPS32
    return (2 * ds + 2.0 ** -21 + 8 * EPS32) * vmax + 1e-30


def evict(acc, slot_pos, n, keep, recent, pos):
    """Per KV head of acc [nkv][cap]: (to, from) slots of the moves, by the rule of
    molot_hip_kv_evict, slot by slot."""
    moves = []
    for h in range(acc.shape[0]):
        a, p = acc[h, :n].tolist(), slot_pos[h, :n].tolist()

        def rank(i):
            if p[i] > pos - recent:
                return (0, 0.0, i)
            if math.isnan(a[i]):
                return (1, 0.0, i)
            return (2, -a[i] + 0.0, i)

        stay = set(sorted(range(n), key=rank)[:keep]) if n > keep else set(range(n))
        src = [i for i in range(keep, n) if i in stay]
        dst = [i for i in range(min(keep, n)) if i not in stay]
        moves.append(list(zip(dst, src)))
    return moves
