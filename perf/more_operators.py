"""Measured cases of ragged batches: packed rows of sequences of different lengths
over a paged cache.

Operators (include/molot_amd/attn_hip.h):
  plan    from how many rows every sequence brings and how many it has cached:
          the blocks of finished sequences go back to the free list (a stack:
          pushed sequence by sequence, block by block), the blocks that the new
          rows need come off its top in the same order, into the block tables;
          the lengths with the new rows; where each sequence's rows start in the
          packed batch; and for each row its sequence, its position and its slot
          in the pool (block * PAGE + row of the block).
  append  every packed row's q and k normed (`norm`) and rotated at its position,
          k and v stored at its slot.
  attend  every row of a sequence over the slots up to its own: s = scale * q.k,
          with softcap c, s = c * tanh(s / c); with slopes, s -= slope_h * distance;
          o = softmax(s) V; a window leaves out the slots further back.
  step    one layer of one tick: plan, append and attend.

A case is a dict of plain values:
  op, kv ("f32", "bf16", "q8"), nq, nkv, d, softcap (0: none), alibi, window, norm
  seqs, few      sequences, and the rows that each brings (1: one new token)
  prompts, lo, hi  the first `prompts` of them bring prompts (or parts) of lo .. hi rows
  clo, chi       rows cached before
  done           (plan) of the others, this many are finished
"""
import ctypes
import math

import torch

own = False

PAGE = 16
SHORT = 32  # rows up to which a sequence counts as a short one in the plain form

# A dense 32q/8kv layer, its 64-query variant, a narrow one, one of an uncommon
# head dim and group, and a layer of 256-wide (sliding window) heads.
DENSE = dict(nq=32, nkv=8, d=128)
WIDE_Q = dict(nq=64, nkv=8, d=128)
NARROW = dict(nq=8, nkv=8, d=64)
ODD = dict(nq=12, nkv=4, d=96)
LOCAL = dict(nq=8, nkv=4, d=256)


def listed():
    return [
        # A tick of a chat server: every sequence one token, two chats just ended.
        _case(DENSE, "plan", name="plan_tick", seqs=64, clo=40, chi=4000, done=2),
        # An offline job's batch: thousands of prompts taken in at once.
        _case(DENSE, "plan", name="plan_prompts", seqs=4099, prompts=4050, lo=1, hi=31, clo=0, chi=500,
              done=40),
        # A small tick's new rows on a layer with norms, the reference's cache type.
        _case(DENSE, "append", name="append_tick_f32", kv="f32", seqs=40, clo=3, chi=3000, norm=True),
        # Parts of three prompts beside the tokens of running chats.
        _case(DENSE, "append", name="append_chunks_bf16", kv="bf16", seqs=32, prompts=3, lo=300, hi=1200,
              clo=0, chi=2000, norm=True),
        # The first turns of a few chats on a small layer: latency and launches.
        _case(NARROW, "attend", name="attend_few_f32", kv="f32", seqs=7, prompts=5, lo=2, hi=20, clo=0,
              chi=300),
        # Chats decoding beside one part of a long prompt.
        _case(DENSE, "attend", name="attend_tick_bf16", kv="bf16", seqs=64, prompts=1, lo=512, hi=512,
              clo=100, chi=4000),
        # Drafts of four tokens checked in one go, over the small cache type.
        _case(DENSE, "attend", name="attend_drafts_q8", kv="q8", seqs=32, few=5, clo=500, chi=9000),
        # Fresh prompts of very different lengths, the reference's cache type.
        _case(DENSE, "attend", name="attend_prompts_f32", kv="f32", seqs=9, prompts=9, lo=37, hi=1200,
              clo=0, chi=0),
        # A sliding-window layer with capped scores: parts of prompts and running chats.
        _case(LOCAL, "attend", name="attend_window_bf16", kv="bf16", seqs=16, prompts=4, lo=200, hi=900,
              clo=0, chi=4000, window=1024, softcap=50.0),
        # A question of 17 tokens about a very long document, beside fresh prompts.
        _case(WIDE_Q, "attend", name="attend_long_bf16", kv="bf16", seqs=3, prompts=2, lo=700, hi=2000,
              few=17, clo=0, chi=131072),
        # A whole tick of a layer for a few chats.
        _case(DENSE, "step", name="step_tick_f32", kv="f32", seqs=17, clo=50, chi=2000),
        # A whole tick with parts of two prompts, on a layer with norms and a distance bias.
        _case(DENSE, "step", name="step_chunks_f32", kv="f32", seqs=50, prompts=2, lo=256, hi=500,
              clo=20, chi=3000, norm=True, alibi=True),
    ]


def _case(layer, op, **kw):
    return dict(dict(layer, op=op, kv="bf16", softcap=0.0, alibi=False, window=0, norm=False, few=1,
                     prompts=0, lo=1, hi=1, clo=0, chi=0, done=0), **kw)


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges: batches, prompts and contexts spread over their
    logarithm, every layer kind and cache type."""
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "step"])
    if op == "plan":
        seqs = _log_int(rng, 1, 4000)
        hi = _log_int(rng, 1, max(1, 60000 // seqs))
        prompts = rng.choice([0, seqs // 5, seqs // 2])
        return _case(DENSE, op, seqs=seqs, prompts=prompts, lo=max(1, hi // rng.randint(1, 30)), hi=hi,
                     clo=0, chi=_log_int(rng, 1, 4095), done=rng.randint(0, max(0, seqs - prompts) // 4))
    layer = dict(rng.choice([DENSE, WIDE_Q, NARROW, ODD, LOCAL]))
    # (a step's k, rounded to fewer bits on either side of a tie, would be another key to its rows)
    kv = rng.choice({"attend": ["f32", "bf16", "q8"], "append": ["f32", "bf16"], "step": ["f32"]}[op])
    softcap = rng.choice([0.0, 0.0, 30.0, 50.0]) if op != "append" else 0.0
    alibi = op != "append" and rng.random() < 0.3
    norm = op != "attend" and rng.random() < 0.5
    window = 0 if op == "append" or rng.random() < 0.7 else _log_int(rng, 1, 4096)
    wide = layer["nq"] * layer["d"] / 4096.0
    if rng.random() < 0.35:  # no prompts: running chats, or drafts of a few tokens
        few = rng.choice([1, 1, rng.randint(2, 20)])
        seqs = _log_int(rng, 1, max(2, 200 // few))
        chi = _log_int(rng, 17, int(min(60000, 200000 // seqs)))
        return _case(layer, op, kv=kv, softcap=softcap, alibi=alibi, window=window, norm=norm, seqs=seqs,
                     few=few, clo=max(0, chi // rng.randint(2, 40) - 1), chi=chi)
    prompts = _log_int(rng, 1, 9)
    hi = _log_int(rng, 1, int(min(1100, 2600 / prompts / wide)))
    chi = rng.choice([0, _log_int(rng, 1, int(max(2, min(9000, 2.5e6 / wide / prompts / hi - hi))))])
    return _case(layer, op, kv=kv, softcap=softcap, alibi=alibi, window=window, norm=norm,
                 seqs=prompts + rng.choice([0, _log_int(rng, 1, 50)]), prompts=prompts,
                 lo=max(1, hi // rng.randint(1, 30)), hi=hi, clo=chi // rng.randint(2, 40), chi=chi)


# --- shapes -----------------------------------------------------------------


def _spread(n, lo, hi):
    """n whole numbers spread over [lo, hi], dealt in a fixed mixed order."""
    at = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]
    step = next(s for s in range(max(2, (5 * n) // 8), 10 * n + 2) if math.gcd(s, max(1, n)) == 1)
    return [at[(i * step) % n] for i in range(n)]


def _batch(case):
    """Rows cached before, rows brought, and the finished of every sequence."""
    n, p = case["seqs"], case["prompts"]
    cached = _spread(n, case["clo"], case["chi"])
    if p and case["chi"] > 10000:  # a very long context is the last one's, beside fresh prompts
        cached = [0] * (n - 1) + [case["chi"]]
    counts = (_spread(p, case["lo"], case["hi"]) if p else []) + [case["few"]] * (n - p)
    done = [0] * n
    for i in range(case["done"]):
        done[n - 1 - 2 * i if n - 1 - 2 * i >= p else n - 1] = 1
    return cached, [0 if x else c for c, x in zip(counts, done)], done


def _row_bytes(case):
    d = case["d"]
    return {"f32": 4 * d, "bf16": 2 * d, "q8": d + 4}[case["kv"]]


def _blocks(n):
    return (n + PAGE - 1) // PAGE


def work(case):
    """plan: the batch's counts and lengths, the blocks given back and taken, the
    rows' maps.  append: q read and written, k and v read and stored.  attend: q, o
    and the attended slots of every sequence once; 4*d flops a (q head, row, slot)."""
    nq, nkv, d, rb = case["nq"], case["nkv"], case["d"], _row_bytes(case)
    cached, counts, done = _batch(case)
    rows = sum(counts)
    bytes_, flops = 0, 0
    if case["op"] in ("plan", "step"):
        back = sum(_blocks(c) for c, x in zip(cached, done) if x)
        taken = sum(_blocks(c + m) - _blocks(c) for c, m, x in zip(cached, counts, done) if not x)
        held = sum(_blocks(c + m) - c // PAGE for c, m in zip(cached, counts) if m)
        bytes_ += 4 * (5 * len(counts) + 2 * back + 2 * taken + held + 3 * rows)
    if case["op"] in ("append", "step"):
        bytes_ += 8 * rows * nq * d + 2 * rows * nkv * (4 * d + rb)
    if case["op"] in ("attend", "step"):
        w, seen, slots = case["window"], 0, 0
        for c, m in zip(cached, counts):
            if m:
                slots += c + m - (max(0, c - w + 1) if w > 0 else 0)
            if w > 0 and c + m > w:
                full = min(m, max(0, c + m - w))  # rows whose window is full
                k = m - full
                seen += full * w + k * c + k * (k + 1) // 2
            else:
                seen += m * c + m * (m + 1) // 2
        if case["op"] == "step":
            slots -= rows  # the new ones are at hand
        bytes_ += 8 * rows * nq * d + 2 * nkv * rb * slots
        flops = 4 * d * nq * seen
    return {"bytes": bytes_, "flops": flops}


# --- inputs -----------------------------------------------------------------


def _pool(case, g, blocks):
    """A pool of `blocks` random pages [blocks][nkv][PAGE][d]."""
    nkv, d = case["nkv"], case["d"]
    x = torch.randn(blocks, nkv, PAGE, d, device="cuda", generator=g)
    if case["kv"] == "f32":
        return x.view(blocks, -1)
    if case["kv"] == "bf16":
        return x.to(torch.bfloat16).view(blocks, -1)
    s = x.abs().amax(-1) / 127.0
    s = torch.where(s > 0, s, torch.ones_like(s))
    codes = torch.clamp(torch.round(x / s[..., None]), -127, 127).to(torch.int8)
    return torch.cat([codes.view(blocks, -1).view(torch.uint8),
                      s.contiguous().view(blocks, -1).view(torch.uint8)], 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    nq, nkv, d, op = case["nq"], case["nkv"], case["d"], case["op"]
    i32 = dict(dtype=torch.int32, device="cuda")
    cached, counts, done = _batch(case)
    B, rows = len(counts), sum(counts)
    after = [m if x else c + m for c, m, x in zip(cached, counts, done)]
    planned = op in ("plan", "step")  # the tables are of the rows cached before
    have = [_blocks(n) for n in (cached if planned else after)]
    taken = sum(_blocks(n) for n, x in zip(after, done) if not x) if planned else 0
    blocks = max(sum(have), taken) + 5 + sum(_blocks(m) for m in counts if planned)
    width = max(1, max(_blocks(max(a, c)) for a, c in zip(after, cached)))
    perm = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    hold = torch.tensor(have, device="cuda")
    live = torch.arange(width, device="cuda")[None] < hold[:, None]
    table = torch.zeros(B, width, **i32)
    table[live] = perm[:sum(have)]
    free = torch.zeros(blocks, **i32)
    free[:blocks - sum(have)] = perm[sum(have):]
    s = dict(case=case, scale=1.0 / math.sqrt(d), rows=rows, blocks=blocks, longest=max(after + [1]),
             table=table, lens=torch.tensor(cached, **i32), counts=torch.tensor(counts, **i32),
             done=torch.tensor(done, **i32), free=free,
             left=torch.tensor([blocks - sum(have)], **i32), cached=cached, ns=counts, after=after)
    # the plan's outputs (of the other operators: a plan made before)
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), s["counts"].long())
    start = torch.cat([torch.zeros(1, **i32), s["counts"].cumsum(0).to(torch.int32)])
    slot = s["lens"].long()[seq] + torch.arange(rows, device="cuda") - start.long()[seq]
    s.update(after_lens=torch.tensor(after, **i32), start=start, left_after=torch.zeros(1, **i32),
             seq=seq.to(torch.int32), row_pos=slot.to(torch.int32), status=torch.zeros(1, **i32),
             row_slot=(table[seq, slot // PAGE] * PAGE + slot % PAGE).to(torch.int32))
    if op == "plan":
        return s
    s["K"], s["V"] = (_pool(case, g, blocks) for _ in range(2))
    # capped layers are those whose raw scores run large
    s["q"] = torch.randn(rows, nq, d, device="cuda", generator=g) * (6.0 if case["softcap"] else 2.0)
    s["o"] = torch.zeros(rows, nq, d, device="cuda")
    s["slopes"] = s["q_norm"] = s["k_norm"] = None
    if case["alibi"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, nq + 1, device="cuda") / nq)
    if op != "attend":
        s["kn"], s["vn"] = torch.randn(2, rows, nkv, d, device="cuda", generator=g).unbind(0)
        s["freq"] = (1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)).float()
    if case["norm"]:
        s["q_norm"], s["k_norm"] = (1 + 0.1 * torch.randn(2, d, device="cuda", generator=g)).unbind(0)
    # the sequences with rows, short ones and prompts apart: which, most rows, most slots
    apart = [[b for b in range(B) if 0 < counts[b] <= SHORT], [b for b in range(B) if counts[b] > SHORT]]
    s["groups"] = [(torch.tensor(b, device="cuda"), max(counts[i] for i in b), max(after[i] for i in b))
                   for b in apart if b]
    return s


# --- the plain form ----------------------------------------------------------


def _plain_plan(s):
    table, free, left = s["table"], s["free"], s["left"].long()
    cols = torch.arange(table.shape[1], device="cuda")[None]
    off = s["done"] != 0
    lens, counts = s["lens"].long(), s["counts"].long()
    back = off[:, None] & (cols < ((lens + PAGE - 1) // PAGE)[:, None])
    lens = torch.where(off, torch.zeros_like(lens), lens)
    given = table[back]
    free[left + torch.arange(given.numel(), device="cuda")] = given
    top = left + given.numel()
    after = lens + counts
    take = (cols >= ((lens + PAGE - 1) // PAGE)[:, None]) & (cols < ((after + PAGE - 1) // PAGE)[:, None])
    number = take.view(-1).long().cumsum(0).view_as(take)
    table[take] = free[top - number[take]]
    s["status"].copy_(torch.where(number[-1, -1] > top, -28, 0))
    s["after_lens"].copy_(after)
    s["left_after"].copy_(top - number[-1, -1])
    s["start"][1:] = counts.cumsum(0)
    r = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["start"][1:].long(), r, right=True)
    slot = lens[seq] + r - s["start"].long()[seq]
    s["seq"].copy_(seq)
    s["row_pos"].copy_(slot)
    s["row_slot"].copy_(table[seq, slot // PAGE] * PAGE + slot % PAGE)


def _rotated(s, x, weight):
    """Rows [rows][heads][d] normed with weight (None: not) and rotated, in 32 bits;
    the angle is the product of position and frequency in 32 bits."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
    ang = (s["row_pos"].float()[:, None] * s["freq"]).double()[:, None]
    c, n = ang.cos().float(), ang.sin().float()
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * n, a * n + b * c], -1)


def _plain_append(s):
    case = s["case"]
    nkv, d = case["nkv"], case["d"]
    at, sl = s["row_slot"].long() // PAGE, s["row_slot"].long() % PAGE
    s["q"].copy_(_rotated(s, s["q"], s["q_norm"]))
    for pool, x in ((s["K"], _rotated(s, s["kn"], s["k_norm"])), (s["V"], s["vn"])):
        pool.view(-1, nkv, PAGE, d)[at, :, sl] = x.to(pool.dtype)


def _values(case, pool, table):
    """Rows [sequences][slots][nkv][d] of the sequences' pages in 32 bits."""
    nkv, d = case["nkv"], case["d"]
    x = pool[table.long()]
    if case["kv"] == "q8":
        cut = nkv * PAGE * d
        codes = x[..., :cut].contiguous().view(torch.int8).view(*table.shape, nkv, PAGE, d)
        x = codes.float() * x[..., cut:].contiguous().view(torch.float32).view(*table.shape, nkv, PAGE, 1)
    else:
        x = x.view(*table.shape, nkv, PAGE, d).float()
    return x.transpose(2, 3).reshape(table.shape[0], -1, nkv, d)


def _plain_group(s, which, M, N):
    """The rows of some sequences, padded to M rows and N slots."""
    case = s["case"]
    nq, nkv, d, w, c = case["nq"], case["nkv"], case["d"], case["window"], case["softcap"]
    counts, n = s["counts"].long()[which], s["after_lens"].long()[which]
    K, V = (_values(case, s[x], s["table"][which][:, :_blocks(N)])[:, :N] for x in ("K", "V"))
    i = torch.arange(M, device="cuda")[None]
    real = i < counts[:, None]
    row = torch.where(real, s["start"].long()[which][:, None] + i, torch.zeros_like(i))
    own_slot = (n - counts)[:, None] + i
    q = s["q"][row].view(-1, M, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4).reshape(-1, nkv, nq // nkv * M, d)
    x = (q @ K.permute(0, 2, 3, 1)).view(-1, nq, M, N) * s["scale"]
    if c > 0:
        x = c * torch.tanh(x / c)
    t = torch.arange(N, device="cuda")
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * (own_slot[..., None] - t).abs().float()[:, None]
    seen = t <= own_slot[..., None]
    if w > 0:
        seen = seen & (t > own_slot[..., None] - w)
    x = torch.where(seen[:, None], x, torch.full_like(x, -math.inf))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = p.view(-1, nkv, nq // nkv * M, N) @ V.transpose(1, 2)
    o = o.view(-1, nkv, nq // nkv, M, d).permute(0, 3, 1, 2, 4).reshape(-1, M, nq, d)
    s["o"][row[real]] = o[real]


def _plain(s):
    op = s["case"]["op"]
    if op in ("plan", "step"):
        _plain_plan(s)
    if op in ("append", "step"):
        _plain_append(s)
    if op in ("attend", "step"):
        for group in s["groups"]:
            _plain_group(s, *group)
    return _outputs(s)


def _outputs(s):
    op, out = s["case"]["op"], {}
    if op in ("plan", "step"):
        out.update(table=s["table"], lens=s["after_lens"], free=s["free"], left=s["left_after"],
                   start=s["start"], seq=s["seq"], pos=s["row_pos"], slot=s["row_slot"], status=s["status"])
    if op in ("append", "step"):
        out.update(q=s["q"], k=s["K"], v=s["V"])
    if op in ("attend", "step"):
        out["o"] = s["o"]
    return out


# --- the framework's calls ----------------------------------------------------


def _p(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def _own(s):
    from molot_amd import attn
    from molot_amd import lib

    case, L, op = s["case"], lib.load(), s["case"]["op"]
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    kvd = {"f32": attn.KV_F32, "bf16": attn.KV_BF16, "q8": attn.KV_Q8}[case["kv"]]
    st, none = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), _p(None)
    B, width = s["table"].shape
    table, after, start = _p(s["table"]), _p(s["after_lens"]), _p(s["start"])
    pos, slot = _p(s["row_pos"]), _p(s["row_slot"])
    if op in ("plan", "step"):
        lib.check(L.molot_hip_ragged_plan(
            _p(s["counts"]), _p(s["done"]), none, _p(s["lens"]), after, table, _p(s["free"]),
            _p(s["left"]), _p(s["left_after"]), B, width, PAGE, s["blocks"], s["rows"], start,
            _p(s["seq"]), pos, slot, _p(s["status"]), st), "ragged_plan")
    if op == "append":
        lib.check(L.molot_hip_rope_append_ragged(
            _p(s["q"]), _p(s["kn"]), _p(s["vn"]), _p(s["K"]), _p(s["V"]), pos, slot, s["rows"],
            s["blocks"], nq, nkv, d, PAGE, _p(s["q_norm"]), _p(s["k_norm"]), 0, 1e-6, _p(s["freq"]),
            kvd, st), "rope_append_ragged")
    if op == "attend":
        lib.check(L.molot_hip_attn_ragged(
            _p(s["q"]), _p(s["K"]), _p(s["V"]), _p(s["o"]), table, after, start, s["rows"], B, width,
            s["blocks"], s["longest"], nq, nkv, d, PAGE, s["scale"], case["window"], case["softcap"],
            _p(s["slopes"]), kvd, st), "attn_ragged")
    if op == "step":
        lib.check(L.molot_hip_step_ragged(
            _p(s["q"]), _p(s["kn"]), _p(s["vn"]), _p(s["K"]), _p(s["V"]), _p(s["o"]), table, after,
            start, pos, slot, s["rows"], B, width, s["blocks"], s["longest"], nq, nkv, d, PAGE,
            _p(s["q_norm"]), _p(s["k_norm"]), 0, 1e-6, _p(s["freq"]), s["scale"], case["window"],
            case["softcap"], _p(s["slopes"]), kvd, st), "step_ragged")
    return _outputs(s)


def run(state):
    return _own(state) if own else _plain(state)


# --- the same in 64 bits ----------------------------------------------------


def _stored64(case, pool, ids, h, n):
    """The n cached rows of KV head h in the blocks ids as 64-bit numbers [n][d]."""
    nkv, d = case["nkv"], case["d"]
    pages = pool[ids]
    if case["kv"] != "q8":
        return pages.view(-1, nkv, PAGE, d)[:, h].reshape(-1, d)[:n].double()
    at = h * PAGE * d
    codes = pages[:, at:at + PAGE * d].contiguous().view(torch.int8).view(-1, d).double()
    at = nkv * PAGE * d + 4 * h * PAGE
    sc = pages[:, at:at + 4 * PAGE].contiguous().view(torch.float32).view(-1, 1)
    return (codes * sc.double())[:n]


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    nq, nkv, d, w, c = case["nq"], case["nkv"], case["d"], case["window"], case["softcap"]
    tables = [t[:_blocks(n)].tolist() for t, n in zip(s["table"].cpu(), s["after"])]
    out = {}
    if case["op"] == "step":  # the blocks off the stack, one by one
        free = s["free"].cpu().tolist()[:int(s["left"])]
        for b, n in enumerate(s["cached"]):
            tables[b] = tables[b][:_blocks(n)]
            while len(tables[b]) < _blocks(s["after"][b]):
                tables[b].append(free.pop())
        out.update({x: None for x in ("table", "lens", "free", "left", "start", "seq", "pos", "slot",
                                      "status")})
    q = s["q"].double()
    if case["op"] != "attend":
        place = [(tables[b][i // PAGE], i % PAGE, i) for b in range(len(s["ns"]))
                 for i in range(s["cached"][b], s["after"][b])]
        blk, sl, at = torch.tensor(place, device="cuda").view(-1, 3).unbind(1)
        ang = (at.float()[:, None, None] * s["freq"]).double()  # the definition's angle
        turn = torch.complex(ang.cos(), ang.sin())

        def spun(x, weight):
            x = x.double()
            if weight is not None:
                x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
            z = torch.complex(x[..., :d // 2], x[..., d // 2:]) * turn
            return torch.cat([z.real, z.imag], -1)

        q = spun(q, s["q_norm"])
        for name, new in (("K", spun(s["kn"], s["k_norm"])), ("V", s["vn"].double())):
            s[name].view(-1, nkv, PAGE, d)[blk, :, sl] = new.to(s[name].dtype)
            out[name.lower()] = s[name].double()
        out["q"] = q
    if case["op"] == "append":
        return out
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, m in enumerate(s["ns"]):
        n, ids = s["after"][b], torch.tensor(tables[b], dtype=torch.long, device="cuda")
        for h in range(nkv if m else 0):
            K, V = _stored64(case, s["K"], ids, h, n), _stored64(case, s["V"], ids, h, n)
            t, slot = torch.arange(n, device="cuda"), torch.arange(n - m, n, device="cuda")[:, None]
            hide = (t > slot) | (t <= slot - w) if w > 0 else t > slot
            for i in range(h * (nq // nkv), (h + 1) * (nq // nkv)):
                x = (q[first:first + m, i] @ K.T) / math.sqrt(d)
                if c > 0:
                    x = c * (x / c).tanh()
                if s["slopes"] is not None:
                    x -= s["slopes"][i].double() * (slot - t)
                o[first:first + m, i] = x.masked_fill_(hide, -math.inf).softmax(-1) @ V
        first += m
    out["o"] = o
    return out
