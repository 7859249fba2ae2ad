"""The pages of a cache on the GPU against pages_oracle.py, to the bit: the tables, lengths, counts and
results, and every byte of the pools."""
import numpy as np
import pytest
import torch

import dashmag_amd as dm
from pages_oracle import Cache

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


class Both:
    """A cache on the GPU and its oracle, changed together."""

    def __init__(self, rows, cols, pages, page, shapes=((2, 8),), seed=0, dtype=np.int16, views=False):
        rng = np.random.default_rng(seed)
        self.rng, self.page = rng, page
        host = [rng.integers(-30000, 30000, (pages, page, *s)).astype(dtype) for s in shapes]
        self.cache = Cache([[-1] * cols for _ in range(rows)], [0] * rows, [0] * pages, page, host)
        if views:  # one tensor of keys and values by page
            both = torch.from_numpy(np.stack(host, 1)).cuda()
            self.pools = list(both.unbind(1))
        else:
            self.pools = [torch.from_numpy(h).cuda() for h in host]
        self.table = torch.full((rows, cols), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.counts = torch.zeros(pages, dtype=torch.int32, device="cuda")

    def put(self):
        """The oracle's state to the GPU."""
        self.table.copy_(_i32(self.cache.table).view(self.table.shape))
        self.lengths.copy_(_i32(self.cache.lengths))
        self.counts.copy_(_i32(self.cache.counts))
        return self

    def same(self):
        assert self.table.tolist() == self.cache.table
        assert self.lengths.tolist() == self.cache.lengths
        assert self.counts.tolist() == self.cache.counts
        for a, b in zip(self.pools, self.cache.pools):
            assert np.array_equal(a.cpu().numpy(), b)

    def reserve(self, new):
        got = dm.cache_reserve(self.table, self.lengths, self.counts, _i32(new), self.page)
        assert got.dtype == torch.bool and got.tolist() == self.cache.reserve(new)
        self.same()
        return got.tolist()

    def fork(self, parents, children):
        got = dm.cache_fork(self.pools, self.table, self.lengths, self.counts, _i32(parents), _i32(children))
        assert got.tolist() == self.cache.fork(parents, children)
        self.same()
        return got.tolist()

    def free(self, rows):
        dm.cache_free(self.table, self.lengths, self.counts, _i32(rows), self.page)
        self.cache.free(rows)
        self.same()

    def compact(self):
        got = dm.cache_compact(self.pools, self.table, self.lengths, self.counts)
        assert got.tolist() == self.cache.compact()
        self.same()


@pytest.mark.parametrize("seed", range(8))
def test_many_rounds(seed):
    """Rows that come, fork, grow, end and are closed up, with calls that are too much among them."""
    rng = np.random.default_rng(seed)
    rows, page = int(rng.choice([5, 40, 130])), int(rng.choice([1, 7, 16, 64]))
    pages = int(rng.choice([30, 700, 5000, 9000]))
    cols = int(rng.choice([4, 50, 300]))
    shapes = [((2, 8), (2, 8)), ((3,), (5, 1), (2, 8)), ((),)][seed % 3]
    c = Both(rows, cols, pages, page, shapes, seed)
    print(f"rows={rows} cols={cols} pages={pages} page={page}", flush=True)
    for _ in range(12):
        what = rng.integers(0, 5)
        if what <= 1:
            grow = rng.integers(-3, 3 * page * max(1, pages // rows), rows) * (rng.random(rows) < 0.4)
            c.reserve([int(x) for x in np.asarray(c.cache.lengths) + grow])
        elif what == 2:
            n = int(rng.integers(1, rows + 3))
            c.fork([int(x) for x in rng.integers(-1, rows + 1, n)], [int(x) for x in rng.integers(-1, rows + 1, n)])
        elif what == 3:
            c.free([int(x) for x in rng.integers(-1, rows + 1, int(rng.integers(1, rows)))])
        else:
            c.compact()


def test_lengths_around_a_page():
    c = Both(8, 6, 60, 16, seed=3)
    c.reserve([0, 1, 15, 16, 17, 32, 33, 96])
    c.free([7])
    c.fork([1, 2, 3], [0, 7, 7])
    c.free([0, 7])
    c.fork([6, 5], [7, 0])
    c.reserve([x + 1 for x in c.cache.lengths])


def test_free_pages_that_fall_short():
    c = Both(6, 10, 12, 4, seed=4)
    assert c.reserve([20, 21, 16, 1, 0, 3]) == [True, True, False, False, True, False]  # 5 + 6 of 12 pages
    assert c.fork([1, 1, 0], [2, 3, 4]) == [11, -2, -1]
    c.reserve([20, 24, 24, 0, 20, 4])
    c.free([0, 4])
    assert c.counts.tolist()[:5] == [0] * 5


def test_forks_that_are_not_made():
    c = Both(6, 4, 30, 4, seed=5)
    c.reserve([7, 4, 0, 0, 0, 0])
    # a child that holds keys, one named twice, itself, rows outside, an empty parent, a parent that is a child
    c.fork([0, 0, 0, 2, 9, 0, 3, 2], [1, 2, 2, 3, 4, -1, 5, 2])
    c.fork([0], [0])


def test_a_row_named_twice_is_freed_once():
    c = Both(4, 4, 20, 4, seed=6)
    c.reserve([9, 0, 0, 0])
    c.fork([0, 0], [1, 2])
    c.free([1, 1, 1, 0, 0])


def test_many_rows_and_forks():
    """More rows than a planning workgroup has threads, more pages than a chunk of the counts."""
    c = Both(3000, 6, 20000, 4, shapes=((4,),), seed=7)
    rng = np.random.default_rng(7)
    c.reserve([int(x) for x in rng.integers(0, 20, 1500)] + [0] * 1500)
    c.fork([int(x) for x in rng.integers(0, 1500, 1400)], [int(x) for x in rng.permutation(1500)[:1400] + 1500])
    c.free([int(x) for x in rng.permutation(3000)[:1700]])
    c.compact()
    c.compact()


@pytest.mark.parametrize("in_use", ["none", "all", "low", "high", "one"])
@pytest.mark.parametrize("pages", [9000, 1, 100, 4095, 4096, 4097, 8192])
def test_compaction_of(in_use, pages):
    """Pools around the pages that a planning workgroup takes at a time (4096)."""
    c = Both(4, 4096, pages, 2, shapes=((8,),), seed=8)
    n = {"none": 0, "all": pages, "low": pages // 3, "high": pages // 3, "one": 1}[in_use]
    start = pages - n if in_use in ("high", "one") else 0
    ids = list(range(start, start + n))
    for r in range(4):
        mine = ids[r * 3000:r * 3000 + 3000]
        c.cache.table[r][:len(mine)] = mine
        c.cache.lengths[r] = 2 * len(mine)
        for p in mine:
            c.cache.counts[p] += r + 1
    c.put().compact()


@pytest.mark.parametrize("dtype,shapes,views", [(np.int16, ((8, 128), (8, 128)), True), (np.int16, ((3, 5),), False),
                                                (np.uint8, ((1,),) * 33, False), (np.float32, ((8, 64),) * 40, False),
                                                (np.int8, ((3,), (3,)), True)])
def test_pools(dtype, shapes, views):
    """Pools of one tensor, of odd bytes, and more of them than a launch takes; pages of several pieces."""
    c = Both(20, 9, 150, 16, shapes, seed=9, dtype=dtype, views=views)
    c.reserve([33, 100, 16] + [0] * 17)
    c.fork([0, 1, 2, 1, 1], [5, 6, 7, 8, 9])
    c.free([0, 1, 8])
    c.compact()


def test_pools_past_four_gigabytes():
    """Pages whose bytes lie past 32 bits are copied and moved: 5 GB, the last pages in use."""
    pages, page, width = 5 * 2 ** 30 // 65536, 16, 4096
    pool = torch.empty(pages, page, width, dtype=torch.int8, device="cuda")
    table = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    table[0, :2] = _i32([pages - 1, pages - 3])
    lengths, counts = _i32([21, 0, 0]), torch.zeros(pages, dtype=torch.int32, device="cuda")
    counts[pages - 1] = counts[pages - 3] = 1
    counts[1] = 1  # (nobody's here, in use all the same)
    keys = torch.randint(-128, 128, (2, page, width), dtype=torch.int8, device="cuda")
    pool[pages - 1], pool[pages - 3] = keys[0], keys[1]
    assert dm.cache_fork([pool], table, lengths, counts, _i32([0]), _i32([2])).tolist() == [0]
    assert table[2].tolist() == [pages - 1, 0, -1, -1] and torch.equal(pool[0, :5], keys[1, :5])
    moved = dm.cache_compact([pool], table, lengths, counts)
    assert counts.nonzero()[:, 0].tolist() == [0, 1, 2, 3]
    assert table.tolist() == [[3, 2, -1, -1], [-1] * 4, [3, 0, -1, -1]]
    assert torch.equal(pool[3], keys[0]) and torch.equal(pool[2], keys[1]) and torch.equal(pool[0, :5], keys[1, :5])
    assert moved[pages - 1] == 3 and moved[pages - 3] == 2 and moved[[0, 1, 2]].tolist() == [0, 1, -1]


def test_entries_outside_the_pages_are_passed_over():
    c = Both(4, 5, 20, 4, seed=10)
    c.reserve([15, 9, 0, 0])
    c.cache.table[0][1], c.cache.table[0][3], c.cache.table[1][0] = 1 << 20, -5, -1
    c.cache.lengths[3] = -7
    c.put()
    c.fork([0, 1], [2, 3])
    c.compact()
    c.free([0, 1, 2, 3])
    c.cache.lengths[0] = 1 << 30  # more than the table has room for
    c.put()
    c.reserve([0, 21, 20, 0])
    c.fork([0], [3])
    c.free([0])


def test_nothing_to_do():
    c = Both(3, 4, 10, 4)
    c.fork([], [])
    c.free([])
    empty = Both(0, 4, 10, 4)
    assert dm.cache_reserve(empty.table, empty.lengths, empty.counts, _i32([]), 4).shape == (0,)
    none = Both(3, 4, 0, 4)
    none.reserve([0, 4, 0])
    none.compact()


def test_captured():
    """A captured round of fork, reserve and free: every replay gives what the eager calls give."""
    c, e = (Both(12, 8, 60, 4, shapes=((8,), (8,)), seed=11) for _ in range(2))
    for x in (c, e):
        x.reserve([14, 7] + [0] * 10)
    par, ch, want = _i32([0, 0, 1]), _i32([5, 6, 7]), _i32([15, 8, 0, 0, 0, 17, 18, 9, 0, 0, 0, 0])

    def step(x):
        a = dm.cache_fork(x.pools, x.table, x.lengths, x.counts, par, ch)
        b = dm.cache_reserve(x.table, x.lengths, x.counts, want, 4)
        dm.cache_free(x.table, x.lengths, x.counts, ch[:2], 4)
        return a, b, dm.cache_compact(x.pools, x.table, x.lengths, x.counts)
    step(e)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(c)
    graph.replay()
    for r in range(3):
        torch.cuda.synchronize()
        for x, y in zip((c.table, c.lengths, c.counts, *c.pools), (e.table, e.lengths, e.counts, *e.pools)):
            assert torch.equal(x, y), r
        junk = torch.randn(1 << 20, device="cuda").sum()
        graph.replay()
        for x, y in zip(outs, step(e)):
            assert torch.equal(x, y), r
        del junk
