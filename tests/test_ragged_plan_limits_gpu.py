"""Plans of ragged batches that fail, on the GPU, against the rule of tests/ragged_ref.py."""
from __future__ import annotations

import pytest
import torch

import ragged_ref as rr
from molot_amd import attn

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


def plan(counts, lens, table, page, num, max_rows, free, count=None, done=None):
    """The arrays after a plan on the GPU: a dict as ragged_ref.plan's, and the free list whole."""
    B, width = len(counts), len(table[0])
    counts, lens, table = (torch.tensor(x, **I32) for x in (counts, lens, table))
    stack = torch.tensor(free + [-5] * (num - len(free)), **I32)
    count = torch.tensor([len(free) if count is None else count], **I32)
    left, status, kv = torch.full((1,), 77, **I32), torch.full((1,), 9, **I32), torch.full((B,), 99, **I32)
    start = torch.full((B + 1,), 55, **I32)
    seq, pos, slot = (torch.full((max_rows,), 44, **I32) for _ in range(3))
    attn.ragged_plan(counts, lens, kv, table, B, width, page, num, max_rows, start, seq, pos, slot, status,
                     stack, count, left, None if done is None else torch.tensor(done, **I32))
    n = int(left)
    return dict(status=int(status), kv_lens=kv.tolist(), table=table.tolist(), free=stack.tolist()[:max(0, n)],
                row_start=start.tolist(), row_seq=seq.tolist(), row_pos=pos.tolist(), row_slot=slot.tolist())


@pytest.mark.parametrize("B,apart", [(1030, 1024), (5200, 1024), (5200, 4096), (5200, 5), (40, 3)])
@pytest.mark.parametrize("first", ("length", "count"))
def test_the_status_of_several_errors(gpu, B, apart, first):
    """A batch with a sequence that has a bad length and one of too many rows has one status,
    wherever the two stand."""
    page, width, num, max_rows = 16, 4, 9, 50
    counts, lens, table = [0] * B, [0] * B, [[0] * width] * B
    a, b = 2, 2 + apart
    bad, many = (a, b) if first == "length" else (b, a)
    lens[bad] = -1
    counts[many] = 51  # more than max_rows, of a table's 64
    want = rr.plan(counts, lens, table, page, num, max_rows, list(range(num)))
    assert want["status"] == rr.EINVAL
    same = plan(counts, lens, table, page, num, max_rows, list(range(num))) == want
    assert same
    lens[bad] = 0
    want = rr.plan(counts, lens, table, page, num, max_rows, list(range(num)))
    assert want["status"] == rr.E2BIG
    same = plan(counts, lens, table, page, num, max_rows, list(range(num))) == want
    assert same


@pytest.mark.parametrize("B,each,max_rows", [(4, 20, 300), (300, 9, 2700), (5000, 1, 5000), (3, 2000, 6000)])
def test_new_blocks_that_are_none(gpu, B, each, max_rows):
    """Ids out of the pool among those that the new blocks come off: nothing is planned.  Below
    them, and beneath what finished sequences give back, the list is not asked."""
    page, width = 16, 130
    need = B * -(-each // page)
    num = need + 2 * page + 9
    ids = list(range(num))[::-1]
    counts, lens, table = [each] * B, [0] * B, [[-1] * width] * B
    fits = rr.plan(counts, lens, table, page, num, max_rows, ids)
    same = plan(counts, lens, table, page, num, max_rows, ids) == fits
    assert fits["status"] == 0 and same
    for at in {num - 1, num - 1 - need // 2, num - need}:  # the first, one between, the last taken
        for value in (num, -1, 2 ** 31 - 1, -2 ** 31):
            free = list(ids)
            free[at] = value
            got = plan(counts, lens, table, page, num, max_rows, free)
            same = got == dict(status=rr.EINVAL, kv_lens=lens, table=table, free=free, row_start=[0] * (B + 1),
                               row_seq=[-1] * max_rows, row_pos=[0] * max_rows, row_slot=[-1] * max_rows)
            assert same, (at, value, got["status"])
    free = list(ids)
    free[num - need - 1] = num  # not taken
    got = plan(counts, lens, table, page, num, max_rows, free)
    same = got == dict(fits, free=free[:num - need])
    assert same
    # a finished sequence's blocks come off first: the list's own top is one further down
    have = min(3, need)
    lens, done = [have * page] + lens[1:], [1] + [0] * (B - 1)
    table = [ids[num - have:] + [-1] * (width - have)] + table[1:]
    free = ids[:num - have]
    fits = rr.plan(counts, lens, table, page, num, max_rows, free, done)
    same = plan(counts, lens, table, page, num, max_rows, free, done=done) == fits
    assert fits["status"] == 0 and same
    for at, st in ((len(free) - (need - have), rr.EINVAL), (len(free) - (need - have) - 1, 0)):
        if at == len(free):  # nothing of the list is taken
            continue
        bad = list(free)
        bad[at] = num
        got = plan(counts, lens, table, page, num, max_rows, bad, done=done)
        if st:
            same = got["kv_lens"] == lens and got["table"] == table and got["free"] == bad
            assert got["status"] == st and same and set(got["row_slot"]) == {-1}
        else:
            same = got == dict(fits, free=bad[:len(fits["free"])])
            assert same
