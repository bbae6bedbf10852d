"""Measured cases of the scored attention and of the cache eviction.

Operators (include/molot_amd/attn_hip.h):
  decode   one query row a sequence over its cached rows.  A score is
           s = scale * q.k; with softcap c, s = c * tanh(s / c); with slopes,
           s -= slope_h * |pos - t|; o = softmax(s) V.  `weights`: every row's
           softmax weight, summed over the query heads of its KV head, is added
           to acc.  `append`: the step that stores the new k and v rows first
           (a layer without RoPE).
  prefill  m query rows at positions n0 ..: the same scores, row i over the
           keys [lo_i, hi_i): causal (with a window), `docs` (a packed prompt:
           from its document's first key on), `prefix` (the prompt's first
           rows see each other both ways).
  evict    per KV head, the `keep` of n cached rows that stay: those of the
           `recent` newest positions, then the highest acc, ties to the lowest
           slot.  Kept rows past `keep` move into the evicted slots before it,
           both in order.  A pass marks the newest rows (kv_track), then evicts.

A case is a dict of plain values:
  op, kv ("f32", "bf16", "q8"), nq, nkv, d, softcap (0: none), alibi (slopes)
  decode   n (rows, the newest counted) or batch, lo, hi (pages of 16 rows, lengths
           over [lo, hi]); window, weights, append
  prefill  m, n0, window, mask ("causal", "docs", "prefix"), append
  evict    n, or batch, lo, hi (pages); keep, recent, fresh (rows marked as new)
"""
import ctypes
import math

import torch

own = False

PAGE = 16

# A dense 32q/8kv layer, its 64-query variant, a narrow one, one of an uncommon
# head dim and group, and layers of 256-wide (sliding window) and 512-wide heads.
DENSE = dict(nq=32, nkv=8, d=128)
WIDE_Q = dict(nq=64, nkv=8, d=128)
NARROW = dict(nq=8, nkv=8, d=64)
ODD = dict(nq=12, nkv=4, d=96)
LOCAL = dict(nq=8, nkv=4, d=256)
GLOBAL = dict(nq=8, nkv=2, d=512)


def listed():
    return [
        # The first tokens of a chat on a layer with a distance bias: latency and launches.
        _decode(DENSE, name="step_first", kv="f32", n=301, alibi=True, append=True),
        # One stream at 16k context, capped scores, over the reference's cache type.
        _decode(DENSE, name="decode_16k", kv="f32", n=16385, softcap=50.0),
        # One very long document on a layer with a distance bias, bf16 cache.
        _decode(WIDE_Q, name="step_131k_bf16", kv="bf16", n=131073, alibi=True, append=True),
        # A sliding-window layer with capped scores, late in a long chat.
        _decode(LOCAL, name="decode_window", kv="f32", n=32769, window=1024, softcap=50.0),
        # A step of a stream with a row budget: the weights for the next eviction.
        _decode(DENSE, name="weights_16k_bf16", kv="bf16", n=16001, softcap=50.0, weights=True),
        # A small batch of ragged contexts over the small cache type, with weights.
        _decode(DENSE, name="paged_13_q8", kv="q8", batch=13, lo=1, hi=2999, softcap=30.0,
                weights=True),
        # A fresh 2048-token prompt with capped scores.
        _prefill(DENSE, name="prefill_2k", kv="f32", m=2048, n0=0, softcap=50.0),
        # Several prompts packed into one, 256-wide heads.
        _prefill(LOCAL, name="prefill_docs_bf16", kv="bf16", m=1999, n0=0, softcap=50.0,
                 mask="docs"),
        # A short turn whose first rows see each other both ways, with a distance bias.
        _prefill(NARROW, name="prefill_prefix", kv="bf16", m=77, n0=0, alibi=True, mask="prefix",
                 append=True),
        # One stream cut back to its budget after 256 new tokens.
        _evict(DENSE, name="evict_4k_bf16", kv="bf16", n=4352, keep=4096, recent=512, fresh=256),
        # A batch of ragged streams: those over the budget are cut back to it.
        _evict(DENSE, name="evict_paged_q8", kv="q8", batch=32, lo=700, hi=1399, keep=1024,
               recent=128, fresh=64),
        # A long cache after a chunk of 8192 rows.
        _evict(DENSE, name="evict_131k", kv="bf16", n=131072, keep=122880, recent=8192, fresh=8192),
    ]


def _decode(layer, **kw):
    return dict(dict(layer, op="decode", softcap=0.0, alibi=False, window=0, weights=False,
                     append=False), **kw)


def _prefill(layer, **kw):
    return dict(dict(layer, op="prefill", softcap=0.0, alibi=False, window=0, mask="causal",
                     append=False), **kw)


def _evict(layer, **kw):
    return dict(dict(layer, op="evict", softcap=0.0, alibi=False), **kw)


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges: contexts, prompts, batches and budgets spread
    over their logarithm, every layer kind and cache type."""
    layer = dict(rng.choice([DENSE, WIDE_Q, NARROW, ODD, LOCAL, GLOBAL]))
    kv = rng.choice(["f32", "bf16", "q8"])
    softcap = rng.choice([0.0, 30.0, 50.0])
    alibi = softcap == 0.0 or rng.random() < 0.25
    op = rng.choice(["decode", "decode", "paged", "prefill", "evict", "evict_paged"])
    rows = {"f32": 16384, "bf16": 131072, "q8": 131072}[kv] * 128 // layer["d"]
    if op == "decode":
        append = kv != "q8" and rng.random() < 0.5
        window = 0 if append or rng.random() < 0.7 else _log_int(rng, 1, 4096)
        return _decode(layer, kv=kv, n=_log_int(rng, 1, min(rows, 131072)), softcap=softcap,
                       alibi=alibi, window=window, weights=rng.random() < 0.4, append=append)
    if op == "paged":
        hi = _log_int(rng, 17, 4095 if layer["d"] <= 128 else 2047)
        return _decode(layer, kv=kv, batch=_log_int(rng, 1, 32), lo=max(0, hi // rng.randint(2, 40)),
                       hi=hi, softcap=softcap, alibi=alibi, window=0,
                       weights=rng.random() < 0.5)
    if op == "prefill":
        mask = rng.choice(["causal", "docs", "prefix"])
        wide = layer["nq"] * layer["d"]
        m = _log_int(rng, 1, 1791 if wide <= 4096 else 1023)
        most = max(1, min(16384, 1800000 * 4096 // (wide * m) - m // 2))
        n0 = 0 if mask != "causal" or rng.random() < 0.5 else _log_int(rng, 1, most)
        window = 0 if mask == "prefix" or rng.random() < 0.7 else _log_int(rng, 1, 1024)
        return _prefill(layer, kv=kv, m=m, n0=n0, softcap=softcap, alibi=alibi, window=window,
                        mask=mask, append=kv != "q8" and n0 == 0 and rng.random() < 0.5)
    if op == "evict":
        n = _log_int(rng, 2, min(rows, 131072))
        fresh = _log_int(rng, 1, max(1, n // 8))
        return _evict(layer, kv=kv, n=n, keep=max(1, n - rng.randint(1, fresh)),
                      recent=_log_int(rng, fresh, max(fresh, n // 4)), fresh=fresh)
    hi = _log_int(rng, 33, 4095 if layer["d"] <= 128 else 2047)
    return _evict(layer, kv=kv, batch=_log_int(rng, 1, 32), lo=max(1, hi // 3), hi=hi,
                  keep=max(1, hi * rng.randint(5, 9) // 10), recent=rng.randint(1, max(1, hi // 8)),
                  fresh=rng.randint(1, max(1, hi // 3)))


# --- shapes -----------------------------------------------------------------


def _lengths(case):
    """Rows of every sequence: spread over [lo, hi], dealt in a fixed mixed order."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    at = [lo + (hi - lo) * i // max(1, b - 1) for i in range(b)]
    step = next(s for s in range(max(2, (5 * b) // 8), 10 * b + 2) if math.gcd(s, b) == 1)
    return [at[(i * step) % b] for i in range(b)]


def _row_bytes(case):
    d = case["d"]
    return {"f32": 4 * d, "bf16": 2 * d, "q8": d + 4}[case["kv"]]


def _doc_starts(m):
    """First rows of the documents of a packed prompt of m rows: lengths that
    double from 37 up to 592 and start over."""
    starts, at, k = [], 0, 0
    while at < m:
        starts.append(at)
        at += 37 << (k % 5)
        k += 1
    return starts


def _ranges(case):
    """[lo, hi) of every query row's keys."""
    m, n0, w = case["m"], case["n0"], case["window"]
    lo = [max(0, n0 + i - w + 1) if w > 0 else 0 for i in range(m)]
    hi = [n0 + i + 1 for i in range(m)]
    if case["mask"] == "docs":
        starts = _doc_starts(m)
        at = 0
        for i in range(m):
            while at + 1 < len(starts) and starts[at + 1] <= i:
                at += 1
            lo[i] = max(lo[i], n0 + starts[at])
    elif case["mask"] == "prefix":
        hi = [max(x, min(n0 + m, (m + 1) // 2)) for x in hi]
    return lo, hi


def work(case):
    """Attended cache rows, q, o, new rows and weights read or written once;
    4*d flops per (q head, query, key).  Eviction: the weights and positions
    read, and the rows past the budget read and written once."""
    nq, nkv, d, rb = case["nq"], case["nkv"], case["d"], _row_bytes(case)
    if case["op"] == "decode":
        ns = _lengths(case) if "batch" in case else [case["n"]]
        w = case["window"]
        att = [min(n, w) if w > 0 else n for n in ns]
        new = len(ns) if case["append"] else 0
        return {"bytes": 2 * nkv * rb * (sum(att) - new) + 8 * nq * d * len(ns) +
                2 * nkv * new * (4 * d + rb) + (8 * nkv * sum(att) if case["weights"] else 0),
                "flops": 4 * d * nq * sum(att)}
    if case["op"] == "prefill":
        lo, hi = _ranges(case)
        m = case["m"]
        new = m if case["append"] else 0
        rows = max(hi) - min(lo) - new
        return {"bytes": 2 * nkv * rb * rows + 8 * m * nq * d + 2 * nkv * new * (4 * d + rb),
                "flops": 4 * d * nq * sum(b - a for a, b in zip(lo, hi))}
    ns = _lengths(case) if "batch" in case else [case["n"]]
    cut = [max(0, n - case["keep"]) for n in ns]
    move = sum(min(c, case["fresh"], case["recent"], case["keep"]) for c in cut)
    seen = sum(n for n, c in zip(ns, cut) if c)
    return {"bytes": nkv * (8 * seen + 8 * len(ns) * case["fresh"] + move * 2 * (2 * rb + 8)), "flops": 0}


# --- inputs -----------------------------------------------------------------


def _quantize(x):
    """Q8 rows of x[..., d]: fp32 scale absmax/127 (1 for a zero row), codes."""
    s = x.abs().amax(-1) / 127.0
    s = torch.where(s > 0, s, torch.ones_like(s))
    return torch.clamp(torch.round(x / s[..., None]), -127, 127).to(torch.int8), s


def _q8_row(nkv, d):
    return nkv * d + (4 * nkv + 15) // 16 * 16


def _cache(case, g, rows):
    """A token-major cache of `rows` random rows [rows][nkv][d]."""
    nkv, d = case["nkv"], case["d"]
    if case["kv"] != "q8":
        t = torch.float32 if case["kv"] == "f32" else torch.bfloat16
        x = torch.randn(rows, nkv * d, device="cuda", generator=g)
        return x.to(t)
    codes, s = _quantize(torch.randn(rows, nkv, d, device="cuda", generator=g))
    out = torch.zeros(rows, _q8_row(nkv, d), dtype=torch.uint8, device="cuda")
    out[:, :nkv * d] = codes.view(rows, nkv * d).view(torch.uint8)
    out[:, nkv * d:nkv * d + 4 * nkv] = s.contiguous().view(torch.uint8)
    return out


def _pool(case, g, blocks):
    """A pool of `blocks` random pages [blocks][nkv][PAGE][d]."""
    nkv, d = case["nkv"], case["d"]
    x = torch.randn(blocks, nkv, PAGE, d, device="cuda", generator=g)
    if case["kv"] == "f32":
        return x.view(blocks, -1)
    if case["kv"] == "bf16":
        return x.to(torch.bfloat16).view(blocks, -1)
    codes, s = _quantize(x)
    return torch.cat([codes.view(blocks, -1).view(torch.uint8),
                      s.contiguous().view(blocks, -1).view(torch.uint8)], 1)


def _acc(g, *shape):
    """Accumulated weights as a stream leaves them: most rows little, a few
    much, and rows that never got any."""
    x = torch.exp(2.0 * torch.randn(*shape, device="cuda", generator=g))
    return torch.where(torch.rand(*shape, device="cuda", generator=g) < 0.1, torch.zeros_like(x), x)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    nq, nkv, d, op = case["nq"], case["nkv"], case["d"], case["op"]
    i32 = dict(dtype=torch.int32, device="cuda")
    s = dict(case=case, scale=1.0 / math.sqrt(d))
    paged = "batch" in case
    if paged:
        lens = _lengths(case)
        need = [(n + PAGE - 1) // PAGE for n in lens]
        blocks = sum(need) + 5
        perm = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
        table, at = torch.zeros(len(lens), max(1, max(need)), **i32), 0
        for b, k in enumerate(need):
            table[b, :k] = perm[at:at + k]
            at += k
        s.update(table=table, lens=torch.tensor(lens, **i32), ns=lens)
        s["K"], s["V"] = (_pool(case, g, blocks) for _ in range(2))
        s["acc"] = _acc(g, blocks, nkv, PAGE)
    else:
        n = case["n0"] + case["m"] if op == "prefill" else case["n"]
        s["K"], s["V"] = (_cache(case, g, n) for _ in range(2))
        s["acc"] = _acc(g, nkv, n + 3)
    if op == "evict":
        if paged:
            # the slot's position, where the sequence's pages hold it
            p = torch.zeros(s["acc"].shape, **i32)
            slots = torch.arange(table.shape[1] * PAGE, **i32).view(1, -1, 1, PAGE)
            live = torch.arange(table.shape[1], device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
            p[table[live].long()] = slots.expand(len(lens), -1, nkv, -1)[live]
            s["slot_pos"], s["pos"] = p, s["lens"] - 1 - case["fresh"]
        else:
            s["slot_pos"] = torch.arange(n + 3, **i32).repeat(nkv, 1)
            s["pos"] = n - 1 - case["fresh"]
        return s
    rows = len(lens) if paged else (case["m"] if op == "prefill" else 1)
    if op == "decode":
        s["acc"] *= 1e-4  # a few steps' worth
    # capped layers are those whose raw scores run large
    s["q"] = torch.randn(rows, nq, d, device="cuda", generator=g) * (6.0 if case["softcap"] else 2.0)
    s["o"] = torch.zeros(rows, nq, d, device="cuda")
    s["slopes"] = None
    if case["alibi"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, nq + 1, device="cuda") / nq)
    if case["append"]:
        s["kn"], s["vn"] = torch.randn(2, rows, nkv, d, device="cuda", generator=g).unbind(0)
    if op == "prefill":
        lo, hi = _ranges(case)
        s["lo"], s["hi"] = torch.tensor(lo, **i32), torch.tensor(hi, **i32)
    return s


# --- the plain form ----------------------------------------------------------


def _values(case, x):
    """Cache rows [..., nkv, d] of a token-major cache as fp32."""
    nkv, d, n = case["nkv"], case["d"], x.shape[0]
    if case["kv"] != "q8":
        return x.view(n, nkv, d).float()
    codes = x[:, :nkv * d].contiguous().view(torch.int8).view(n, nkv, d)
    return codes.float() * x[:, nkv * d:nkv * d + 4 * nkv].contiguous().view(torch.float32)[..., None]


def _paged_values(case, x, table):
    """Rows [B][max_blocks * PAGE][nkv][d] of the sequences' pages as fp32."""
    nkv, d = case["nkv"], case["d"]
    x = x[table.long()]
    if case["kv"] == "q8":
        cut = nkv * PAGE * d
        codes = x[..., :cut].contiguous().view(torch.int8).view(*table.shape, nkv, PAGE, d)
        sc = x[..., cut:].contiguous().view(torch.float32).view(*table.shape, nkv, PAGE)
        x = codes.float() * sc[..., None]
    else:
        x = x.view(*table.shape, nkv, PAGE, d).float()
    return x.transpose(2, 3).reshape(table.shape[0], -1, nkv, d)


def _score(s, dot, dist):
    """Scores [..., nq, keys] of raw products; dist [..., 1, keys]."""
    c = s["case"]["softcap"]
    x = dot * s["scale"]
    if c > 0:
        x = c * torch.tanh(x / c)
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None] * dist.float()
    return x


def _softmax(x, seen):
    """exp(x - max) / sum over the seen keys; 0 where a row sees none."""
    x = torch.where(seen, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _plain_decode(s):
    case = s["case"]
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    w = case["window"]
    if "batch" in case:
        K, V = (_paged_values(case, s[x], s["table"]) for x in ("K", "V"))
        B, N = K.shape[:2]
        t = torch.arange(N, device="cuda")
        n = s["lens"].long()[:, None]
    else:
        if case["append"]:
            s["K"][-1] = s["kn"].view(-1).to(s["K"].dtype)
            s["V"][-1] = s["vn"].view(-1).to(s["V"].dtype)
        K, V = (_values(case, s[x])[None] for x in ("K", "V"))
        B, N = 1, K.shape[1]
        t = torch.arange(N, device="cuda")
        n = torch.full((1, 1), N, device="cuda")
    seen = t[None] < n
    if w > 0:
        seen = seen & (t[None] > n - 1 - w)
    dot = s["q"].view(B, nkv, nq // nkv, d) @ K.permute(0, 2, 3, 1)
    dist = (n - 1 - t[None]).abs()[:, None]
    p = _softmax(_score(s, dot.view(B, nq, N), dist), seen[:, None])
    s["o"].copy_((p.view(B, nkv, nq // nkv, N) @ V.permute(0, 2, 1, 3)).view(B, nq, d))
    if case["weights"]:
        got = p.view(B, nkv, nq // nkv, N).sum(2)
        if "batch" in case:
            at = (t // PAGE)[None].expand(B, N)
            blk = s["table"].long().gather(1, at)[seen]
            s["acc"][blk, :, (t % PAGE)[None].expand(B, N)[seen]] += got.transpose(1, 2)[seen]
        else:
            if case["append"]:
                s["acc"][:, N - 1] = 0.0  # the new row starts from nothing
            s["acc"][:, :N] += got[0]
    return _outputs(s)


def _plain_prefill(s):
    case = s["case"]
    nq, nkv, d, m, n0 = case["nq"], case["nkv"], case["d"], case["m"], case["n0"]
    if case["append"]:
        s["K"][n0:] = s["kn"].view(m, -1).to(s["K"].dtype)
        s["V"][n0:] = s["vn"].view(m, -1).to(s["V"].dtype)
    K, V = (_values(case, s[x]) for x in ("K", "V"))
    N = K.shape[0]
    t = torch.arange(N, device="cuda")[None]
    pos = n0 + torch.arange(m, device="cuda")[:, None]
    seen = (t >= s["lo"][:, None]) & (t < s["hi"][:, None])
    q = s["q"].view(m, nkv, nq // nkv, d).permute(1, 2, 0, 3).reshape(nkv, -1, d)
    dot = (q @ K.permute(1, 2, 0)).view(nq, m, N).transpose(0, 1)
    p = _softmax(_score(s, dot, (pos - t).abs()[:, None]), seen[:, None])
    p = p.transpose(0, 1).reshape(nkv, -1, N)
    o = (p @ V.transpose(0, 1)).view(nkv, nq // nkv, m, d)
    s["o"].copy_(o.permute(2, 0, 1, 3).reshape(m, nq, d))
    return _outputs(s)


def _plain_evict(s):
    case = s["case"]
    nkv, d, keep, fresh = case["nkv"], case["d"], case["keep"], case["fresh"]
    acc, sp = s["acc"], s["slot_pos"]
    s["pos"] = s["pos"] + fresh  # the newest token's position
    if "batch" in case:
        B, N = len(s["ns"]), s["table"].shape[1] * PAGE
        t = torch.arange(N, device="cuda")
        n = s["lens"].long()[:, None]
        pos = s["pos"].long()[:, None]
        blk = s["table"].long()[:, t // PAGE]  # [B][N]
        spot = lambda b, h, i: (blk[b, i], h, i % PAGE)  # noqa: E731
        a = acc[blk, :, (t % PAGE)[None]].transpose(1, 2)  # [B][nkv][N]
        p = sp[blk, :, (t % PAGE)[None]].transpose(1, 2)
    else:
        B, N = 1, case["n"]
        t = torch.arange(N, device="cuda")
        n = torch.full((1, 1), N, device="cuda")
        pos = torch.full((1, 1), s["pos"], device="cuda")
        spot = lambda b, h, i: (h, i)  # noqa: E731
        a, p = acc[None, :, :N], sp[None, :, :N]
    live = t[None] < n
    new = live & (t[None] >= n - fresh)  # just appended: no weight yet
    a = torch.where(new[:, None], torch.zeros_like(a), a)
    p = torch.where(new[:, None], (pos - (n - 1 - t[None]))[:, None].to(p.dtype), p)
    key = torch.where(p > (pos - case["recent"])[:, None], torch.full_like(a, math.inf), a)
    key = torch.where(live[:, None], key, torch.full_like(a, -1.0))
    # the rank of every slot: higher keys first, the lowest slot of equals
    order = key.sort(dim=-1, descending=True, stable=True).indices
    stays = torch.zeros_like(live[:, None].expand_as(key))
    stays = stays.scatter(-1, order[..., :keep], True) & live[:, None]
    src = (stays & (t >= keep)).nonzero().unbind(1)  # [sequence, head, slot], in order
    dst = (~stays & live[:, None] & (t < keep) & (n > keep)[:, None]).nonzero().unbind(1)
    mark = new[:, None].expand_as(a).nonzero().unbind(1)
    acc[spot(*mark)] = 0.0
    sp[spot(*mark)] = p[mark].to(sp.dtype)
    acc[spot(*dst)] = acc[spot(*src)]
    sp[spot(*dst)] = sp[spot(*src)]
    for x in (s["K"], s["V"]):
        if "batch" in case:
            cut = nkv * PAGE * d
            rows = x[:, :cut].view(-1, nkv, PAGE, d)
            rows[spot(*dst)] = rows[spot(*src)]
            if case["kv"] == "q8":
                sc = x[:, cut:].view(-1, nkv, PAGE, 4)
                sc[spot(*dst)] = sc[spot(*src)]
        else:
            rows = x[:, :nkv * d].view(-1, nkv, d)
            rows[dst[2], dst[1]] = rows[src[2], src[1]]
            if case["kv"] == "q8":
                sc = x[:, nkv * d:nkv * d + 4 * nkv].view(-1, nkv, 4)
                sc[dst[2], dst[1]] = sc[src[2], src[1]]
    return _outputs(s)


def _outputs(s):
    case = s["case"]
    if case["op"] == "evict":
        return {"k": s["K"], "v": s["V"], "acc": s["acc"], "slot_pos": s["slot_pos"]}
    out = {"o": s["o"]}
    if case["op"] == "decode" and case["weights"]:
        out["acc"] = s["acc"]
    if case["append"]:
        first = case["n0"] if case["op"] == "prefill" else case["n"] - 1
        out["k"], out["v"] = s["K"][first:], s["V"][first:]
    return out


# --- the framework's calls ----------------------------------------------------


def _p(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def _own(s):
    from molot_amd import attn
    from molot_amd import lib

    case, L = s["case"], lib.load()
    nq, nkv, d, cap = case["nq"], case["nkv"], case["d"], case["softcap"]
    kvd = {"f32": attn.KV_F32, "bf16": attn.KV_BF16, "q8": attn.KV_Q8}[case["kv"]]
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    K, V, acc = _p(s["K"]), _p(s["V"]), _p(s["acc"])
    if case["op"] == "evict":
        sp = _p(s["slot_pos"])
        s["pos"] = s["pos"] + case["fresh"]
        if "batch" in case:
            B, width = s["table"].shape
            table, lens, pos, longest = _p(s["table"]), _p(s["lens"]), _p(s["pos"]), max(s["ns"])
            rc = L.molot_hip_kv_track_paged(acc, sp, table, lens, pos, B, width, longest,
                                            case["fresh"], nkv, PAGE, st)
            rc = rc or L.molot_hip_kv_evict_paged(K, V, acc, sp, table, lens, pos, B, width, longest,
                                                  nkv, d, PAGE, case["keep"], case["recent"], kvd, st)
        else:
            width = s["acc"].shape[1]
            rc = L.molot_hip_kv_track(acc, sp, nkv, case["n"], case["fresh"], s["pos"], width, st)
            rc = rc or L.molot_hip_kv_evict(K, V, acc, sp, nkv, case["n"], d, case["keep"],
                                            case["recent"], s["pos"], width, kvd, st)
        lib.check(rc, "kv_evict")
        return _outputs(s)
    q, o, slopes, none = _p(s["q"]), _p(s["o"]), _p(s["slopes"]), _p(None)
    scale, w = s["scale"], case["window"]
    if case["op"] == "prefill":
        m, n0 = case["m"], case["n0"]
        lo, hi = (_p(s["lo"]), _p(s["hi"])) if case["mask"] != "causal" else (none, none)
        if case["append"]:
            rc = L.molot_hip_prefill_step_scored(
                q, _p(s["kn"]), _p(s["vn"]), K, V, o, nq, nkv, d, m, n0, n0, none, none, 0, 0.0,
                none, scale, w, cap, slopes, lo, hi, kvd, st)
        else:
            rc = L.molot_hip_attn_prefill_scored(q, K, V, o, nq, nkv, m, n0 + m, d, scale, n0, w,
                                                 cap, slopes, lo, hi, kvd, st)
        lib.check(rc, "prefill_scored")
        return _outputs(s)
    acc = acc if case["weights"] else none
    if "batch" in case:
        B, width = s["table"].shape
        rc = L.molot_hip_attn_decode_paged_scored(
            q, K, V, o, _p(s["table"]), _p(s["lens"]), none, B, width, max(s["ns"]), nq, nkv, d, PAGE,
            scale, w, cap, slopes, acc, kvd, st)
    elif case["append"]:
        n, width = case["n"], s["acc"].shape[1]
        rc = L.molot_hip_decode_step_scored(
            q, _p(s["kn"]), _p(s["vn"]), K, V, o, nq, nkv, d, n - 1, n - 1, none, none, 0, 0.0, none,
            scale, w, cap, slopes, acc, none, width, kvd, st)
    else:
        n, width = case["n"], s["acc"].shape[1]
        rc = L.molot_hip_attn_decode_scored(q, K, V, o, nq, nkv, n, d, scale, n - 1, w, cap, slopes,
                                            acc, width, kvd, st)
    lib.check(rc, "decode_scored")
    return _outputs(s)


def run(state):
    if own:
        return _own(state)
    return {"decode": _plain_decode, "prefill": _plain_prefill, "evict": _plain_evict}[
        state["case"]["op"]](state)


# --- the same in 64 bits ----------------------------------------------------


def _row64(case, s, name, b, h):
    """Cached rows of sequence b and KV head h as 64-bit numbers [n][d]."""
    nkv, d, x = case["nkv"], case["d"], s[name]
    if "batch" not in case:
        if case["kv"] != "q8":
            return x.view(-1, nkv, d)[:, h].double()
        sc = x[:, nkv * d + 4 * h:nkv * d + 4 * h + 4].contiguous().view(torch.float32)
        return x[:, h * d:(h + 1) * d].contiguous().view(torch.int8).double() * sc.double()
    n = s["ns"][b]
    pages = x[s["table"][b, :(n + PAGE - 1) // PAGE].long()]
    if case["kv"] == "q8":
        at = h * PAGE * d
        codes = pages[:, at:at + PAGE * d].contiguous().view(torch.int8).view(-1, d).double()
        at = nkv * PAGE * d + 4 * h * PAGE
        sc = pages[:, at:at + 4 * PAGE].contiguous().view(torch.float32).view(-1, 1)
        return (codes * sc.double())[:n]
    return pages.view(-1, nkv, PAGE, d)[:, h].reshape(-1, d)[:n].double()


def _attend64(case, q, K, V, pos, lo, hi, slope):
    """o [m][d] and the weights [m][n] of one head's rows, 64 bits."""
    c, t = case["softcap"], torch.arange(K.shape[0], device=K.device)
    x = (q @ K.T) / math.sqrt(case["d"])
    if c > 0:
        x = c * (x / c).tanh()
    if slope is not None:
        x -= slope * (pos[:, None] - t).abs()
    x.masked_fill_((t < lo[:, None]) | (t >= hi[:, None]), -math.inf)
    p = x.softmax(-1).nan_to_num_(0.0)
    return p @ V, p


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(case, s)
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    dev = dict(device="cuda")
    out = {}
    if case["append"]:
        first = case["n0"] if case["op"] == "prefill" else case["n"] - 1
        for name, new in (("K", "kn"), ("V", "vn")):
            s[name][first:] = s[new].reshape(-1, nkv * d).to(s[name].dtype)
            out[name.lower()] = s[name][first:].double()
    o = torch.zeros(s["q"].shape, dtype=torch.float64, **dev)
    acc = s["acc"].double()
    if case["append"] and case["op"] == "decode":
        acc[:, case["n"] - 1] = 0.0
    for b in range(len(s["ns"]) if "batch" in case else 1):
        rows = slice(0, case["m"]) if case["op"] == "prefill" else slice(b, b + 1)
        for h in range(nkv):
            K, V = _row64(case, s, "K", b, h), _row64(case, s, "V", b, h)
            n = K.shape[0]
            if n == 0:
                continue
            if case["op"] == "prefill":
                pos = case["n0"] + torch.arange(case["m"], **dev)
                lo, hi = s["lo"], s["hi"]
            else:
                pos, hi = torch.tensor([n - 1], **dev), torch.tensor([n], **dev)
                lo = (hi - case["window"]).clamp(min=0) if case["window"] > 0 else torch.zeros_like(hi)
            for i in range(h * (nq // nkv), (h + 1) * (nq // nkv)):
                slope = None if s["slopes"] is None else s["slopes"][i].double()
                o[rows, i], p = _attend64(case, s["q"][rows, i].double(), K, V, pos, lo, hi, slope)
                if case["op"] == "decode" and case["weights"]:
                    if "batch" in case:
                        t = torch.arange(n, **dev)
                        acc[s["table"][b].long()[t // PAGE], h, t % PAGE] += p[0]
                    else:
                        acc[h, :n] += p[0]
    out["o"] = o
    if case["op"] == "decode" and case["weights"]:
        out["acc"] = acc
    return out


def _exact_evict(case, s):
    """The definition, slot by slot, on the host."""
    keep, nkv, d = case["keep"], case["nkv"], case["d"]
    paged = "batch" in case
    acc, sp = s["acc"].cpu(), s["slot_pos"].cpu()
    moved = []  # (page or slot, head, row of the page) pairs: to, from
    for b in range(len(s["ns"]) if paged else 1):
        n = s["ns"][b] if paged else case["n"]
        newest = (int(s["pos"][b]) if paged else s["pos"]) + case["fresh"]
        table = s["table"][b].tolist() if paged else None
        for h in range(nkv):
            spot = (lambda i: (table[i // PAGE], h, i % PAGE)) if paged else (lambda i: (h, i))
            for i in range(max(0, n - case["fresh"]), n):
                acc[spot(i)], sp[spot(i)] = 0.0, newest - (n - 1 - i)
            if n <= keep:
                continue
            if paged:
                idx = [spot(i) for i in range(n)]
                pages, rows = torch.tensor([x[0] for x in idx]), torch.tensor([x[2] for x in idx])
                a, p = acc[pages, h, rows].tolist(), sp[pages, h, rows].tolist()
            else:
                a, p = acc[h, :n].tolist(), sp[h, :n].tolist()
            ranked = sorted(range(n), key=lambda i: (p[i] <= newest - case["recent"],
                                                     0.0 if p[i] > newest - case["recent"] else -a[i], i))
            stay = set(ranked[:keep])
            src = [i for i in range(keep, n) if i in stay]
            dst = [i for i in range(keep) if i not in stay]
            for to, at in zip(dst, src):
                acc[spot(to)], sp[spot(to)] = a[at], p[at]
                moved.append((spot(to), spot(at)) if paged else ((to, h), (at, h)))
    if moved:
        ints = dict(dtype=torch.long, device="cuda")
        to, at = (torch.tensor([m[k] for m in moved], **ints).unbind(1) for k in (0, 1))
        per = (nkv, PAGE) if paged else (nkv,)
        cut = d * math.prod(per)
        for x in (s["K"], s["V"]):
            views = [x[:, :cut].view(-1, *per, d)]
            if case["kv"] == "q8":  # the rows' scales after the codes
                views.append(x[:, cut:cut + 4 * math.prod(per)].view(-1, *per, 4))
            for view in views:
                view[to] = view[at]
    k, v = (x.double() if x.is_floating_point() else x for x in (s["K"], s["V"]))
    return {"k": k, "v": v, "acc": acc.double().cuda(), "slot_pos": sp.cuda()}
