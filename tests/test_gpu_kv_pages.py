"""MI355X: pages handed out and taken back (kv_ops.reserve, trim), against
tests/blocks_reference.py, exactly."""

import numpy as np
import pytest
import torch

from drinkme_amd import kv_ops
from tests import blocks_reference as B

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


class Pool:
    """Sequences of `lengths` in shuffled pages and what is left of `pages`, on the
    GPU and as lists."""

    def __init__(self, rng, lengths, cols, page, pages):
        self.page, self.lengths = page, list(lengths)
        order = rng.permutation(pages).tolist()
        self.table = [[-1] * cols for _ in lengths]
        for row, length in zip(self.table, lengths):
            for c in range(min(cols, -(-max(length, 0) // page))):
                row[c] = order.pop() if order else -1
        self.free, self.count = order + [int(x) for x in rng.integers(-5, pages, pages - len(order))], len(order)
        self.lacking = 0
        self.pool = {"free": i32(self.free), "count": i32([self.count]), "lacking": i32([0])}
        self.gpu_table, self.gpu_lengths = i32(self.table), i32(self.lengths)

    def reserve(self, new, total):
        got = kv_ops.reserve(self.pool, self.gpu_table, self.gpu_lengths, self.page, total, new=None if new is None else i32(new))
        new = [total // len(self.lengths)] * len(self.lengths) if new is None else new
        cu, positions, slots, self.count, self.lacking = B.reserve(self.free, self.count, self.table, self.lengths, new,
                                                                   self.page, total, len(self.free))
        for mine, want, dtype in zip(got, (cu, positions, slots), (torch.int32, torch.int32, torch.int64)):
            assert mine.dtype == dtype and mine.tolist() == want
        self.same()

    def trim(self, keep):
        assert kv_ops.trim(self.pool, self.gpu_table, self.gpu_lengths, self.page, i32(keep)) is None
        self.count = B.trim(self.free, self.count, self.table, self.lengths, keep, self.page)
        self.same()

    def same(self):
        assert self.gpu_table.tolist() == self.table and self.gpu_lengths.tolist() == self.lengths
        assert self.pool["free"].tolist() == self.free
        assert self.pool["count"].item() == self.count and self.pool["lacking"].item() == self.lacking


@pytest.mark.parametrize("page", [8, 16, 64, 1024])
@pytest.mark.parametrize("batch", [1, 2, 63, 65, 300])
@pytest.mark.parametrize("short", [False, True])
def test_steps_of_a_batch(batch, page, short):
    """Even steps, uneven ones with empty sequences, padded rows, more tokens than
    rows, requests that end, drafts that are dropped; with enough pages and without."""
    rng = np.random.default_rng(batch * page + short)
    lengths = rng.integers(0, 6 * page, batch).tolist()
    pages = sum(-(-n // page) for n in lengths) + (batch if short else 12 * batch) + 1
    p = Pool(rng, lengths, 14, page, pages)
    p.reserve(None, batch)
    p.reserve(None, 3 * batch)
    new = rng.integers(-2, 2 * page, batch) * (rng.random(batch) < 0.8)
    total = int(np.maximum(new, 0).sum())
    p.reserve(new.tolist(), total + 7)
    p.trim((np.asarray(p.lengths) - rng.integers(-3, 2 * page, batch)).tolist())
    p.reserve(new.tolist(), max(0, total - 2 * page))
    p.trim([0 if x else 2 ** 31 - 1 for x in rng.random(batch) < 0.3])
    p.reserve(rng.integers(0, 4, batch).tolist(), 4 * batch)
    p.trim([0] * batch)
    p.reserve(None, batch)


@pytest.mark.parametrize("batch", [1024, 1025, 5000])
def test_more_sequences_than_a_turn(batch):
    rng = np.random.default_rng(batch)
    p = Pool(rng, rng.integers(0, 40, batch).tolist(), 8, 8, 5 * batch)
    p.reserve(rng.integers(0, 3, batch).tolist(), 3 * batch)
    p.trim(rng.integers(-1, 40, batch).tolist())
    p.reserve(None, batch)


@pytest.mark.parametrize("total", [4095, 4096, 4097, 30000])
def test_many_tokens(total):
    """Both sides of the number of tokens that a launch of its own places."""
    rng = np.random.default_rng(total)
    p = Pool(rng, [0, 17, 4000, 0, 5], 1200, 16, 3000)
    new = [total // 2, 0, 33, total // 3, 1]
    p.reserve(new, total)
    p.trim([0, 17, 4000, 100, 5])
    p.reserve(new, sum(new))


@pytest.mark.parametrize("columns", [1023, 1024, 1025, 4096, 4097, 12001])
@pytest.mark.parametrize("batch", [1, 37])
@pytest.mark.parametrize("pages", [1.0, 0.8])
def test_many_pages(columns, batch, pages):
    """Pages of a call that one pass of the lanes does not hand out or take back, some of them none; with
    enough in the pool and without."""
    rng = np.random.default_rng(columns + batch)
    cuts = np.sort(rng.integers(0, columns + 1, batch - 1))
    counts = np.diff(np.concatenate([[0], cuts, [columns]])) * 8  # (whole pages: `columns` in all)
    p = Pool(rng, [0] * batch, int(counts.max()) // 8 + 1, 8, int(columns * pages))
    p.reserve(counts.tolist(), int(counts.sum()))
    holes = torch.rand(p.gpu_table.shape, device="cuda") < 0.05
    p.gpu_table[holes & (p.gpu_table >= 0)] = -3
    p.table = p.gpu_table.tolist()
    p.trim([0] * batch)
    p.reserve(counts.tolist(), int(counts.sum()) - 5)


def test_prompts_longer_than_the_table():
    rng = np.random.default_rng(3)
    p = Pool(rng, [10, 30, 0], 4, 8, 40)
    p.reserve([100, 1, 31], 132)  # (position 32 and on have no column)
    p.reserve([1, 5, 1], 7)
    p.trim([33, 20, 0])
    p.reserve([0, 0, 9], 9)


def test_lengths_and_numbers_that_are_none():
    """Negative lengths count as 0; numbers in the table that are no page's are not returned, and slots
    have none of them."""
    rng = np.random.default_rng(4)
    p = Pool(rng, [-5, 24, 16], 4, 8, 12)
    p.reserve([3, 1, 1], 5)
    for value in (-7, 12, 2 ** 31 - 1):
        p.table[1][1] = value
        p.gpu_table[1, 1] = value
        p.reserve([1, 1, 1], 3)
        p.trim([p.lengths[0], 8, p.lengths[2]])
        p.reserve([0, 20, 0], 20)


def test_a_count_that_is_none_s():
    """A count below 0 is an empty pool, one past its pages a full one."""
    for count in (-3, 99):
        p = Pool(np.random.default_rng(5), [8, 8], 4, 8, 6)
        p.pool["count"].fill_(count)
        p.free = list(range(6))
        p.pool["free"].copy_(i32(p.free))
        p.count = min(max(count, 0), 6)
        p.reserve([8, 1], 9)
        p.trim([0, 0])  # (what a full stack does not hold is dropped)


def test_sums_past_32_bits():
    """Numbers of tokens that 32 bits do not sum: the first sequences get the rows."""
    p = Pool(np.random.default_rng(6), [0, 0, 0], 4, 8, 12)
    p.reserve([20, 2 ** 31 - 1, 2 ** 31 - 1], 30)
    q = Pool(np.random.default_rng(6), [0] * 70, 4, 8, 12)
    q.reserve([2 ** 31 - 1] * 70, 9)


def test_reserve_then_trim_is_where_it_began():
    rng = np.random.default_rng(7)
    p = Pool(rng, rng.integers(0, 200, 40).tolist(), 60, 8, 3000)
    before = [t.clone() for t in (*p.pool.values(), p.gpu_table, p.gpu_lengths)]
    keep = list(p.lengths)
    for _ in range(3):
        p.reserve(rng.integers(0, 90, 40).tolist(), 4000)
        p.trim(keep)
        assert all(torch.equal(a, b) for a, b in zip(before, (*p.pool.values(), p.gpu_table, p.gpu_lengths)))


def test_no_tokens():
    p = Pool(np.random.default_rng(8), [5, 9], 4, 8, 12)
    p.reserve([0, 0], 0)
    p.reserve([3, 4], 0)
    p.reserve(None, 0)


def test_a_captured_step_replays():
    """A step's reserve and trim in a graph: every replay goes on from the state that
    the last one left, with new numbers."""
    rng = np.random.default_rng(9)
    p = Pool(rng, rng.integers(0, 60, 20).tolist(), 40, 8, 500)
    new, keep = i32([0] * 20), i32(p.lengths)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        kv_ops.reserve(p.pool, p.gpu_table, p.gpu_lengths, 8, 64, new=new)
        kv_ops.trim(p.pool, p.gpu_table, p.gpu_lengths, 8, keep)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_ops.reserve(p.pool, p.gpu_table, p.gpu_lengths, 8, 64, new=new)
        kv_ops.trim(p.pool, p.gpu_table, p.gpu_lengths, 8, keep)
    for _ in range(5):
        numbers, kept = rng.integers(0, 4, 20).tolist(), rng.integers(0, 80, 20).tolist()
        new.copy_(i32(numbers))
        keep.copy_(i32(kept))
        graph.replay()
        torch.cuda.synchronize()
        cu, positions, slots, p.count, p.lacking = B.reserve(p.free, p.count, p.table, p.lengths, numbers, 8, 64, 500)
        p.count = B.trim(p.free, p.count, p.table, p.lengths, kept, 8)
        assert [t.tolist() for t in out] == [cu, positions, slots]
        p.same()
        torch.empty(1 << 20, device="cuda").fill_(1).sum().item()


def test_on_another_stream():
    p = Pool(np.random.default_rng(10), [5, 9], 400, 8, 900)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        p.gpu_lengths.add_(1)
        p.lengths = [6, 10]
        p.reserve([1500, 1400], 2900)
        p.trim([0, 11])
    torch.cuda.current_stream().wait_stream(stream)


def test_refusals():
    p = Pool(np.random.default_rng(11), [5, 9], 4, 8, 12)
    args = [p.pool, p.gpu_table, p.gpu_lengths, 8]

    def reserve(**kw):
        a = dict(zip(("pool", "block_table", "lengths", "page_size"), args), total=2, new=None)
        a.update(kw)
        return lambda: kv_ops.reserve(**a)

    def trim(**kw):
        a = dict(zip(("pool", "block_table", "lengths", "page_size"), args), keep=i32([1, 1]))
        a.update(kw)
        return lambda: kv_ops.trim(**a)

    for call, match in ((reserve(total=3), "3 tokens"), (reserve(total=-2), "-2 tokens"), (reserve(total=2 ** 30), "tokens"),
                        (reserve(new=i32([1])), "new"), (reserve(new=torch.ones(2, device="cuda")), "new"),
                        (reserve(page_size=12), "power of two"), (trim(page_size=4), "power of two"),
                        (reserve(block_table=p.gpu_table.t()), "block_table"), (trim(lengths=p.gpu_lengths.long()), "lengths"),
                        (trim(lengths=i32([1])), "rows"), (trim(keep=i32([1])), "keep"), (trim(keep=torch.ones(2)), "keep"),
                        (reserve(block_table=p.gpu_table.cpu()), "GPU"), (reserve(pool={**p.pool, "count": i32([1, 2])}), "counts"),
                        (reserve(pool={**p.pool, "free": p.pool["free"].long()}), "free"),
                        (trim(block_table=torch.empty((2, 0), dtype=torch.int32, device="cuda")), "columns")):
        with pytest.raises(ValueError, match=match):
            call()
    p.same()
    with pytest.raises(RuntimeError, match="2\\^30 positions"):
        kv_ops.trim(p.pool, torch.empty((1, 1 << 20), dtype=torch.int32, device="cuda"), i32([0]), 1024, i32([0]))
