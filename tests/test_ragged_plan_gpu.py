"""The plan of a ragged batch on the GPU against the rule of tests/ragged_ref.py."""
from __future__ import annotations

import random

import pytest
import torch

import ragged_ref as rr
from molot_amd import attn

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


def ints(x):
    return torch.tensor(x, **I32)


def problem(seed, B, page, top, longest, done=0.2, spare=5, none=0.3):
    """Counts, lengths, a table, a free list with room for them, and the finished."""
    rng = random.Random(seed)
    width = (top + longest + page - 1) // page + 1
    lens = [rng.randint(0, top) for _ in range(B)]
    off = [int(rng.random() < done) for _ in range(B)]
    counts = [0 if rng.random() < none else rng.choice([1, 1, rng.randint(0, longest)]) for _ in range(B)]
    have = [(n + page - 1) // page for n in lens]
    need = sum((n * (1 - x) + c + page - 1) // page for n, c, x in zip(lens, counts, off))
    num = max(sum(have), need) + sum(have) + spare
    ids = list(range(num))
    rng.shuffle(ids)
    table = [[-1] * width for _ in range(B)]
    for b in range(B):
        for j in range(have[b]):
            table[b][j] = ids.pop()
    return dict(counts=counts, lens=lens, table=table, free=ids, done=off, num=num, width=width, page=page)


class Plan:
    def __init__(self, p, max_rows, pos=None, pool=True, done=True, in_place=False):
        B = len(p["counts"])
        self.counts, self.lens = ints(p["counts"]), ints(p["lens"])
        self.kv = self.lens if in_place else torch.full((B,), 99, **I32)
        self.table = ints(p["table"]).view(B, p["width"])
        self.free = ints(p["free"] + [-5] * (p["num"] - len(p["free"]))) if pool else None
        self.count = ints([len(p["free"])]) if pool else None
        self.left = self.count if in_place else ints([77]) if pool else None
        self.done = ints(p["done"]) if done and pool else None
        self.pos = ints(pos) if pos else None
        self.start, self.status = torch.full((B + 1,), 55, **I32), ints([9])
        self.seq, self.rpos, self.slot = (torch.full((max_rows,), 44, **I32) for _ in range(3))
        self.args = (B, p["width"], p["page"], p["num"], max_rows)

    def run(self):
        attn.ragged_plan(self.counts, self.lens, self.kv, self.table, *self.args, self.start, self.seq,
                         self.rpos, self.slot, self.status, self.free, self.count, self.left, self.done,
                         self.pos)

    def check(self, want, width):
        assert int(self.status) == want["status"]
        assert self.kv.tolist() == want["kv_lens"]
        assert self.start.tolist() == want["row_start"]
        assert self.seq.tolist() == want["row_seq"]
        assert self.rpos.tolist() == want["row_pos"]
        assert self.slot.tolist() == want["row_slot"]
        assert self.table.tolist() == want["table"]
        if self.free is not None:
            n = len(want["free"])
            assert int(self.left) == n and self.free.tolist()[:n] == want["free"]


def both(p, max_rows, pool=True, done=True, pos=None, in_place=False):
    want = rr.plan(p["counts"], p["lens"], p["table"], p["page"], p["num"], max_rows,
                   p["free"] if pool else None, p["done"] if done and pool else None, pos)
    g = Plan(p, max_rows, pos, pool, done, in_place)
    g.run()
    g.check(want, p["width"])
    return want, g


# (sequences, page, longest cache, most new rows): the batch's rows in one launch, a long
# search, more sequences than LDS holds, more rows than one launch takes
SIZES = [(1, 16, 0, 1), (1, 1, 5, 9), (2, 16, 40, 16), (7, 16, 100, 33), (64, 16, 300, 2), (65, 4, 50, 7),
         (300, 16, 64, 20), (1024, 32, 70, 3), (1025, 16, 40, 2), (4096, 16, 20, 1), (4097, 16, 20, 1),
         (5000, 8, 30, 3), (3, 16, 20, 5000), (40, 64, 3000, 900), (2500, 16, 9, 12)]


@pytest.mark.parametrize("B,page,top,longest", SIZES)
def test_plan(gpu, B, page, top, longest):
    for seed in range(3):
        p = problem(seed, B, page, top, longest)
        rows = sum(p["counts"])
        want, _ = both(p, rows + seed * 5)
        assert want["status"] == 0
        both(p, rows, done=False)
        both(p, rows + 1, in_place=True)


@pytest.mark.parametrize("B,page,top,longest", [(5, 16, 60, 20), (3, 8, 900, 5000)])
def test_plan_with_positions_and_without_a_pool(gpu, B, page, top, longest):
    p = problem(3, B, page, top, longest, done=0.0)
    both(p, sum(p["counts"]) + 2, pos=[1000 + 7 * b for b in range(B)])
    for b in range(B):  # tables that hold the new rows' blocks
        k = (p["lens"][b] + p["counts"][b] + page - 1) // page
        have = (p["lens"][b] + page - 1) // page
        p["table"][b][have:k] = [p["free"].pop() for _ in range(k - have)]
    both(p, sum(p["counts"]), pool=False)
    p["table"][0][0] = p["num"]  # no block of the pool: its rows have no slot
    p["table"][B - 1][0] = -3
    both(p, sum(p["counts"]) + 1, pool=False)


def test_no_sequences_and_no_rows(gpu):
    p = dict(counts=[], lens=[], table=[], free=[2, 0, 1], done=[], num=3, width=1, page=16)
    both(p, 5)
    p = problem(1, 9, 16, 50, 4)
    p["counts"] = [0] * 9
    both(p, 0)
    both(p, 3)


def test_a_plan_that_fails_changes_nothing(gpu):
    for rows in (40, 6000):  # in one launch and in two
        p = problem(5, 30, 16, 90, 8)
        fits, _ = both(p, rows)
        assert fits["status"] == 0
        q = dict(p, free=p["free"][:0], done=[0] * 30, counts=[20] + p["counts"][1:])
        assert both(q, 6000)[0]["status"] == rr.ENOSPC
        assert both(dict(p, counts=[rows + 1 if rows == 40 else 41] + p["counts"][1:],
                         lens=[0] + p["lens"][1:]), 40 if rows == 40 else 41)[0]["status"] == rr.E2BIG
        for name, value in (("counts", -1), ("lens", -2), ("lens", p["width"] * 16 + 1)):
            bad = list(p[name])
            bad[7] = value
            assert both(dict(p, **{name: bad}, done=[0] * 30), rows)[0]["status"] == rr.EINVAL
        at = next(b for b in range(30) if p["lens"][b])  # a finished one's table names no block
        table = [list(t) for t in p["table"]]
        table[at][0] = p["num"]
        off = [0] * 30
        off[at] = 1
        assert both(dict(p, table=table, done=off), rows)[0]["status"] == rr.EINVAL
        # a sequence given back that would fill the list past the pool
        assert both(dict(p, free=list(range(p["num"])), done=off), rows)[0]["status"] == rr.EINVAL


def test_free_count_that_is_none(gpu):
    p = problem(2, 4, 16, 30, 4)
    for n in (-1, p["num"] + 1):
        g = Plan(p, 20)
        g.count.fill_(n)
        g.run()
        assert int(g.status) == rr.EINVAL and g.kv.tolist() == p["lens"] and int(g.left) == n
        assert g.seq.tolist() == [-1] * 20 and g.start.tolist() == [0] * 5


@pytest.mark.parametrize("B,longest,max_rows", [(6, 3, 300), (3, 1500, 4500)])
def test_a_serving_loop_in_a_graph(gpu, B, longest, max_rows):
    """Ticks replayed from one graph, lengths and pool in place, against the rule."""
    page, width, num = 4, 700, 2000
    rng = random.Random(B)
    g = Plan(dict(counts=[0] * B, lens=[0] * B, table=[[-1] * width] * B, free=list(range(num)),
                  done=[0] * B, num=num, width=width, page=page), max_rows, in_place=True)
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        g.run()  # sizes the workspace
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        g.run()
    state = dict(lens=[0] * B, table=[[-1] * width] * B, free=list(range(num)))
    for tick in range(12):
        counts = [rng.choice([0, 1, rng.randint(0, longest)]) for _ in range(B)]
        done = [int(rng.random() < 0.3) for _ in range(B)]
        g.counts.copy_(ints(counts))
        g.done.copy_(ints(done))
        graph.replay()
        torch.cuda.synchronize()
        want = rr.plan(counts, state["lens"], state["table"], page, num, max_rows, state["free"], done)
        g.check(want, width)
        if want["status"] == 0:
            state = dict(lens=want["kv_lens"], table=want["table"], free=want["free"])
