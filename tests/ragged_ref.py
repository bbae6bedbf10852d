"""Ragged batches plainly: what tests/test_ragged_gpu.py and test_ragged_plan_gpu.py
compare with."""
from __future__ import annotations

import torch

import scored_ref as ref

ENOSPC, EINVAL, E2BIG = -28, -22, -7


def plan(counts, seq_lens, table, page, num_blocks, max_rows, free=None, done=None, pos=None):
    """The rule of molot_hip_ragged_plan, block by block: a dict of lists (free: the stack
    left, lowest first; status)."""
    B, width = len(counts), len(table[0]) if table else 1
    done = done or [0] * B
    table = [list(t) for t in table]

    def failed(st):
        return dict(status=st, kv_lens=list(seq_lens), table=table, free=free, row_start=[0] * (B + 1),
                    row_seq=[-1] * max_rows, row_pos=[0] * max_rows, row_slot=[-1] * max_rows)

    lens = [0 if x else n for n, x in zip(seq_lens, done)]
    for n, m, c in zip(seq_lens, lens, counts):
        if n < 0 or c < 0 or n > width * page or m + c > width * page:
            return failed(EINVAL)
    if sum(counts) > max_rows:
        return failed(E2BIG)
    blocks = lambda n: (n + page - 1) // page  # noqa: E731
    stack = None
    if free is not None:
        stack = list(free)
        for b in range(B):
            if done[b]:
                stack += table[b][:blocks(seq_lens[b])]
        if len(stack) > num_blocks:
            return failed(EINVAL)
        if sum(blocks(n + c) - blocks(n) for n, c in zip(lens, counts)) > len(stack):
            return failed(ENOSPC)
        if any(not 0 <= x < num_blocks for x in stack[len(free):]):
            return failed(EINVAL)
    out = dict(status=0, kv_lens=[n + c for n, c in zip(lens, counts)], table=table, free=stack,
               row_start=[0], row_seq=[], row_pos=[], row_slot=[])
    for b in range(B):
        if stack is not None:
            for j in range(blocks(lens[b]), blocks(lens[b] + counts[b])):
                table[b][j] = stack.pop()
        for i in range(counts[b]):
            s = lens[b] + i
            out["row_seq"].append(b)
            out["row_pos"].append(pos[b] + i if pos else s)
            blk = table[b][s // page]
            out["row_slot"].append(blk * page + s % page if 0 <= blk < num_blocks else -1)
        out["row_start"].append(out["row_start"][-1] + counts[b])
    more = max_rows - len(out["row_seq"])
    out["row_seq"] += [-1] * more
    out["row_pos"] += [0] * more
    out["row_slot"] += [-1] * more
    return out


class Batch:
    """A batch on the GPU whose sequences have `cached` rows and bring `counts`: shuffled
    pages, the index arrays, `pad` rows behind the last, and the cached values [n][nkv][d]
    of every sequence in 64 bits.  fill: what unused rows of the pool hold."""

    def __init__(self, g, kv, nkv, d, counts, cached, page=16, pad=0, spare=3, fill=None, sigma=1.0):
        self.kv, self.nkv, self.d, self.page = kv, nkv, d, page
        self.counts, self.cached, self.B = list(counts), list(cached), len(counts)
        after = [a + c for a, c in zip(counts, cached)]
        need = [(n + page - 1) // page for n in after]
        self.blocks = sum(need) + spare
        self.width = max([1] + need) + 1
        self.max_len = max([1] + after)
        self.rows, self.T = sum(counts), sum(counts) + pad
        i32 = dict(dtype=torch.int32, device="cuda")
        perm = torch.randperm(self.blocks, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((self.B, self.width), -7, **i32)  # past a sequence's blocks: none
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = perm[at:at + k]
            at += k
        self.kv_lens = torch.tensor(after, **i32)
        start = [0]
        for c in counts:
            start.append(start[-1] + c)
        self.starts, self.row_start = start, torch.tensor(start, **i32)
        self.K, self.kval = self._pool(g, after, fill, sigma)
        self.V, self.vval = self._pool(g, after, fill, sigma)

    def _pool(self, g, after, fill, sigma):
        nkv, d, page = self.nkv, self.d, self.page
        x = torch.randn(self.blocks, nkv, page, d, device="cuda", generator=g) * sigma
        if fill is not None and self.kv != "q8":  # slots that hold no row
            used = torch.zeros(self.blocks, page, dtype=torch.bool, device="cuda")
            for b, n in enumerate(after):
                t = torch.arange(n, device="cuda")
                used[self.table[b].long()[t // page], t % page] = True
            x = torch.where(used[:, None, :, None], x, torch.full_like(x, fill))
        if self.kv == "q8":
            codes, s = ref.quantize(x)
            vals = codes.double() * s.double()[..., None]
            pool = torch.cat([codes.reshape(self.blocks, -1).view(torch.uint8),
                              s.contiguous().view(self.blocks, -1).view(torch.uint8)], 1).contiguous()
        else:
            pool = x.to(torch.float32 if self.kv == "f32" else torch.bfloat16).view(self.blocks, -1)
            vals = pool.view(self.blocks, nkv, page, d).double()
        return pool, [self.rows_of(vals, b, n) for b, n in enumerate(after)]

    def rows_of(self, vals, b, n):
        ids = self.table[b, :(n + self.page - 1) // self.page].long()
        return vals[ids].transpose(1, 2).reshape(-1, self.nkv, self.d)[:n]

    def values(self, pool):
        """The rows that the sequences hold in a pool, in 64 bits."""
        nkv, d, page = self.nkv, self.d, self.page
        if self.kv == "q8":
            cut = nkv * page * d
            codes = pool[:, :cut].contiguous().view(torch.int8).view(-1, nkv, page, d)
            sc = pool[:, cut:].contiguous().view(torch.float32).view(-1, nkv, page, 1)
            vals = codes.double() * sc.double()
        else:
            vals = pool.view(-1, nkv, page, d).double()
        return [self.rows_of(vals, b, n + c) for b, (n, c) in enumerate(zip(self.cached, self.counts))]

    def args(self):
        """The arguments between O and nq of attn_ragged."""
        return (self.table, self.kv_lens, self.row_start, self.T, self.B, self.width, self.blocks,
                self.max_len)

    def attend(self, q, scale, window=0, softcap=0.0, slopes=None, K=None, V=None):
        """o [rows][nq][d] in 64 bits and the largest error that roundings may leave."""
        out, tol = [], 0.0
        for b, (n, c) in enumerate(zip(self.cached, self.counts)):
            if c == 0:
                continue
            kb, vb = (K or self.kval)[b], (V or self.vval)[b]
            pos = torch.arange(n, n + c, device="cuda")
            lo = (pos - window + 1).clamp(min=0) if window > 0 else torch.zeros_like(pos)
            x = q[self.starts[b]:self.starts[b + 1]]
            out.append(ref.attend(x, kb, vb, scale, pos, lo, pos + 1, softcap, slopes)[0])
            tol = max(tol, ref.tolerance(x, torch.nan_to_num(kb, 0, 0, 0), torch.nan_to_num(vb, 0, 0, 0),
                                         scale, softcap, slopes, n + c))
        return torch.cat(out) if out else torch.zeros(0, *q.shape[1:], device="cuda").double(), tol
