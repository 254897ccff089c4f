"""lw_pages_advance against the same step taken request by request with lists: growing, ending and cutting sequences, pages handed on,
pools that run out, tables and rows that are too small, many sequences, calls in place, on streams and captured."""
import random

import pytest

pytestmark = pytest.mark.gpu


class Plain:
    """The sequences and their pages, with lists."""

    def __init__(self, count, page, seqs, width):
        self.page, self.width, self.pool = page, width, count
        self.stack = list(range(count - 1, -1, -1))
        self.length, self.table = [0] * seqs, [[-1] * width for _ in range(seqs)]

    def pages(self, n):
        return -(-n // self.page)

    def advance(self, new, keep=None, rows=1 << 30):
        """(lack, q_start, position, slot)"""
        kept = [n if keep is None else min(max(keep[s], 0), n) for s, n in enumerate(self.length)]
        new = [max(n, 0) for n in new]
        had, need = [self.pages(n) for n in self.length], [self.pages(k + n) for k, n in zip(kept, new)]
        take, give = sum(max(b - a, 0) for a, b in zip(had, need)), sum(max(a - b, 0) for a, b in zip(had, need))
        lack = ((1 if take - give > len(self.stack) else 0) + (2 if any(k + n > self.width * self.page for k, n in zip(kept, new)) else 0) +
                (4 if sum(new) > rows else 0))
        if lack:
            return lack, [0] * (len(new) + 1), [], []
        back = [p for t, a, b in zip(self.table, had, need) for p in t[b:a]]
        starts, position, slot = [0], [], []
        for s, (a, b) in enumerate(zip(had, need)):
            for i in range(a, b):
                self.table[s][i] = back.pop(0) if back else self.stack.pop()
            self.length[s] = kept[s] + new[s]
            starts.append(starts[-1] + new[s])
            for i in range(kept[s], self.length[s]):
                position.append(i)
                slot.append(self.table[s][i // self.page] * self.page + i % self.page)
        self.stack += back
        return 0, starts, position, slot


def agree(torch, pages, plain, got, want):
    lack, starts, position, slot = want
    assert pages.left.tolist() == [len(plain.stack), lack]
    assert pages.kv_len.tolist() == plain.length
    assert got[0].tolist() == starts
    n = len(position)
    assert got[1][:n].tolist() == position and got[2][:n].tolist() == slot
    table = pages.table.tolist()
    for s, length in enumerate(plain.length):
        held = plain.pages(length)
        assert table[s][:held] == plain.table[s][:held], s
    assert pages.free[:len(plain.stack)].tolist() == plain.stack
    assert not pages.workspace.any()


@pytest.mark.parametrize("count, page, seqs, width", [(40, 16, 1, 12), (300, 1, 5, 60), (200, 32, 64, 5), (2000, 16, 511, 9), (2000, 8, 513, 9),
                                                      (30000, 64, 8192, 3), (500, 128, 3, 400)], ids=str)
def test_many_steps(gpu, lib, count, page, seqs, width):
    """Steps of all kinds one after the other, in place; now and then one that lacks something, which changes nothing."""
    import torch
    from lazyweights_amd import Pages
    rng = random.Random(count + seqs)
    pages, plain = Pages.empty(count, page, seqs, width), Plain(count, page, seqs, width)
    most = width * page
    lacked = 0
    for step in range(8 if seqs > 1000 else 30):
        big = max(1, min(most, count * page // max(seqs, 1)) // rng.choice((1, 2, 4, 40)))
        keep = None if step % 3 == 0 else [rng.choice((0, n, n, n, max(0, n - rng.randrange(20)), -3, n + 5)) for n in plain.length]
        new = [rng.choice((0, 1, 1, rng.randrange(big + 1), -2)) for _ in range(seqs)]
        if step % 7 == 6:
            new[rng.randrange(seqs)] = most + 1
        rows = sum(max(n, 0) for n in new) + rng.choice((0, 3, 0, -1 if step % 5 == 4 else 0))
        rows = max(rows, 0)
        dev = [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (new, keep)]
        got = pages.advance(dev[0], keep=dev[1], rows=rows)
        want = plain.advance(new, keep, rows)
        lacked += want[0] > 0
        agree(torch, pages, plain, got, want)
    assert lacked and max(plain.length) > 0


def test_large_prompts_over_many_blocks(gpu, lib):
    """Rows enough for all blocks of a launch, half of the sequences ended in the same step."""
    import torch
    from lazyweights_amd import Pages
    rng = random.Random(5)
    seqs, page, width = 700, 16, 200
    pages, plain = Pages.empty(90000, page, seqs, width), Plain(90000, page, seqs, width)
    for step in range(3):
        new = [rng.randrange(1, 1600) for _ in range(seqs)]
        keep = [0 if rng.random() < 0.5 else n // 2 for n in plain.length]
        got = pages.advance(torch.tensor(new, dtype=torch.int32, device="cuda"), keep=torch.tensor(keep, dtype=torch.int32, device="cuda"),
                            rows=sum(new))
        agree(torch, pages, plain, got, plain.advance(new, keep))


def test_given_outputs_and_rows_behind_the_last(gpu, lib):
    """With outputs of one's own the pages' state stays, so that the step can be taken again; rows past the sum are left alone."""
    import torch
    from lazyweights_amd import Pages
    pages, plain = Pages.empty(20, 16, 2, 8), Plain(20, 16, 2, 8)
    first = torch.tensor([30, 5], dtype=torch.int32, device="cuda")
    pages.advance(first, rows=35)
    plain.advance([30, 5])
    new, keep = torch.tensor([3, 40], dtype=torch.int32, device="cuda"), torch.tensor([10, 5], dtype=torch.int32, device="cuda")
    kv, left = pages.kv_len.clone(), pages.left.clone()
    out = [torch.full((n,), -9, dtype=t, device="cuda") for n, t in ((2, torch.int32), (2, torch.int32), (3, torch.int32), (50, torch.int32),
                                                                    (50, torch.int64))]
    free = pages.free.clone()
    for _ in range(3):
        pages.advance(new, keep=keep, kv_len_out=out[0], left_out=out[1], q_start=out[2], position=out[3], slot=out[4])
        assert torch.equal(pages.kv_len, kv) and torch.equal(pages.left, left) and torch.equal(pages.free, free)
        want = plain.__class__.advance(_copy(plain), [3, 40], [10, 5])
        assert out[2].tolist() == want[1] and out[3][:43].tolist() == want[2] and out[4][:43].tolist() == want[3]
        assert out[0].tolist() == [13, 45] and (out[3][43:] == -9).all() and (out[4][43:] == -9).all()
    q_start, position, slot = pages.advance(new, rows=43, places=False)
    assert position is None and slot is None and q_start.tolist() == [0, 3, 43]


def _copy(plain):
    import copy
    return copy.deepcopy(plain)


def test_arrays_that_hold_anything(gpu, lib):
    """Lengths, counts and page numbers out of range are kept in range: nothing outside the arrays is read or written, slots of
    pages that are not there are -1."""
    import torch
    from lazyweights_amd import Pages

    def whole(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    big = 2 ** 31 - 1
    guard = whole([77] * 64)
    table = guard[8:20].view(3, 4)
    table.copy_(whole([[-5, big, 1 << 20, 3]] * 3))
    free, left = whole([9, -1, 1 << 29]), whole([1 << 30, 5])
    pages = Pages(16, whole([-7, big, 40]), table, free, left)
    for new, keep in (([big, big, big], None), ([1, 2, 3], [big, -big, 39]), ([-big] * 3, [0, 0, 0]), ([20, 0, 0], [0, 0, -1])):
        outs = whole([0] * 3), whole([0] * 2)
        q_start, position, slot = pages.advance(whole(new), keep=None if keep is None else whole(keep), rows=70, kv_len_out=outs[0],
                                                left_out=outs[1])
        torch.cuda.synchronize()
        assert (outs[0] >= 0).all() and 0 <= int(outs[1][0]) <= 3
        assert (guard[:8] == 77).all() and (guard[20:] == 77).all()
        n = int(q_start[-1])
        assert ((slot[:n] == -1) | ((slot[:n] >= 0) & (slot[:n] < 3 * 16))).all()


def test_no_sequences_and_no_pages(gpu, lib):
    import torch
    from lazyweights_amd import Pages
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    pages = Pages.empty(4, 16, 0, 3)
    q_start, position, slot = pages.advance(none, rows=0)
    assert q_start.tolist() == [0] and pages.left.tolist() == [4, 0]
    pages = Pages.empty(0, 16, 2, 3)
    pages.advance(torch.tensor([1, 0], dtype=torch.int32, device="cuda"), rows=1)
    assert pages.left.tolist() == [0, 1] and pages.kv_len.tolist() == [0, 0]


def test_streams_and_captured_steps(gpu, lib):
    """A captured step replayed with other counts each time, the program's own work between, gives the lists' steps."""
    import torch
    from lazyweights_amd import Pages
    rng = random.Random(9)
    seqs = 600
    pages, plain = Pages.empty(3000, 16, seqs, 40), Plain(3000, 16, seqs, 40)
    new, keep = (torch.zeros(seqs, dtype=torch.int32, device="cuda") for _ in range(2))
    q_start, rows = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda"), 9000
    position, slot = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int64, device="cuda")

    def step():
        return pages.advance(new, keep=keep, q_start=q_start, position=position, slot=slot)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    pages.advance(new, keep=keep, q_start=q_start, position=position, slot=slot, stream=side.cuda_stream)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(8):
        counts = [rng.randrange(15) for _ in range(seqs)]
        keeps = [n if rng.random() < 0.8 else n // 2 for n in plain.length]
        new.copy_(torch.tensor(counts))
        keep.copy_(torch.tensor(keeps))
        graph.replay()
        torch.cuda.synchronize()
        agree(torch, pages, plain, (q_start, position, slot), plain.advance(counts, keeps, rows))


def test_python_refusals(gpu, lib):
    import torch
    from lazyweights_amd import Pages
    pages = Pages.empty(4, 16, 2, 3)
    kv, table, free, left = pages.kv_len, pages.table, pages.free, pages.left
    for args in ((24, kv, table, free, left), (0, kv, table, free, left), (16, kv[:1], table, free, left), (16, kv, table, free, left[:1]),
                 (16, kv.long(), table, free, left), (16, kv.cpu(), table, free, left), (16, kv, table.T, free, left),
                 (16, kv, table, free[::2], left), (1 << 17, kv, table, free, left),
                 (16, torch.zeros(8193, dtype=torch.int32, device="cuda"), torch.zeros((8193, 1), dtype=torch.int32, device="cuda"), free, left)):
        with pytest.raises(ValueError):
            Pages(*args)
    new = torch.ones(2, dtype=torch.int32, device="cuda")
    for kw in (dict(), dict(rows=-1), dict(rows=1 << 30), dict(rows=2, q_start=new), dict(rows=2, keep=new[:1]), dict(rows=2, keep=new.long()),
               dict(rows=2, position=new.long()), dict(rows=2, slot=new), dict(rows=2, kv_len_out=new.cpu()), dict(rows=2, left_out=new[:1])):
        with pytest.raises(ValueError):
            pages.advance(new, **kw)
    with pytest.raises(ValueError):
        pages.advance(new.float(), rows=2)
    assert pages.kv_len.tolist() == [0, 0]
