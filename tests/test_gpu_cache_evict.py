"""Eviction on the GPU against evict_oracle.py, to the bit: tables, lengths, counts, weights, the kept keys and
every byte of the pools."""
import ctypes

import numpy as np
import pytest
import torch

import dashmag_amd as dm
from dashmag_amd import _lib, ops
from evict_oracle import Evicting

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


class Both:
    def __init__(self, lengths, page, cols, shapes=((2, 8),), dtype=np.int16, seed=0, shared=0, spare=3, weights=None,
                 views=False):
        rng = np.random.default_rng(seed)
        each = [-(-x // page) for x in lengths]
        n = sum(each) + spare
        order = rng.permutation(n).tolist()
        table, counts = [], [0] * n
        for r, x in enumerate(each):
            row = [order.pop() for _ in range(x)]
            if r and r % 2 and shared:  # odd rows begin with pages of the row in front
                m = min(shared, each[r], each[r - 1])
                order += row[:m]
                row[:m] = table[r - 1][:m]
            table.append(row + [-1] * (cols - x))
            for p in row:
                counts[p] += 1
        host = [rng.integers(-100, 100, (n, page, *s)).astype(dtype) for s in shapes]
        if weights is None:
            weights = np.exp(2 * rng.standard_normal((len(lengths), cols * page))).astype(np.float32)
        self.cache = Evicting(table, lengths, counts, page, host, weights=[[float(y) for y in w] for w in weights])
        if views:
            both = torch.from_numpy(np.stack(host, 1)).cuda()
            self.pools = list(both.unbind(1))
        else:
            self.pools = [torch.from_numpy(h).cuda() for h in host]
        self.table, self.lengths, self.counts = _i32(table).view(len(lengths), cols), _i32(list(lengths)), _i32(counts)
        self.weights = torch.tensor(np.asarray(weights, dtype=np.float32)).cuda()

    def evict(self, budgets, recent=0):
        kept = dm.cache_evict(self.pools, self.weights, self.table, self.lengths, self.counts, _i32(budgets), recent)
        want = self.cache.evict(budgets, recent)
        assert kept.dtype == torch.int32 and kept.tolist() == want
        self.same()
        return kept

    def same(self):
        assert self.table.tolist() == self.cache.table
        assert self.lengths.tolist() == self.cache.lengths
        assert self.counts.tolist() == self.cache.counts
        w = np.array(self.cache.weights, dtype=np.float32).reshape(self.weights.shape)
        assert np.array_equal(self.weights.cpu().numpy(), w, equal_nan=True)
        for a, b in zip(self.pools, self.cache.pools):
            assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("seed", range(12))
def test_many(seed):
    rng = np.random.default_rng(seed)
    page, rows = int(rng.choice([1, 7, 16, 64])), int(rng.choice([1, 3, 20]))
    most = int(rng.choice([5, 90, 1500, 5000]))
    lengths = [int(x) for x in rng.integers(0, most, rows)]
    shapes, dtype = [(((2, 8), (2, 8)), np.int16), (((3,), (5, 1), (2, 8)), np.int8), (((),), np.int32),
                     (((8, 128), (4,)), np.int16)][seed % 4]
    b = Both(lengths, page, -(-most // page) + 1, shapes, dtype, seed, shared=int(rng.choice([0, 2])), views=seed % 3 == 0
             and len(set(shapes)) == 1)
    print(f"rows={rows} most={most} page={page} {shapes}", flush=True)
    for _ in range(3):
        b.evict([int(x) for x in rng.integers(-1, most, rows)], int(rng.choice([0, 1, 30, 10 ** 9])))


def test_lengths_budgets_and_recents_around_edges():
    for page in (1, 2, 16):
        lengths = [0, 1, 2, 15, 16, 17, 33, 64]
        for budget in (0, 1, 2, 15, 16, 17, 32):
            for recent in (0, 1, 16, 40):
                Both(lengths, page, 64 // page + 1, seed=budget).evict([budget] * 8, recent)


def test_ties_zeros_and_what_is_not_finite():
    """Equal weights go to the first; -0 is 0; NaN, of either sign, is above all; infinities and negative weights are
    in their order."""
    n = 5000
    rng = np.random.default_rng(1)
    some = np.array([0.0, -0.0, 1.0, 1.0, -1.0, np.inf, -np.inf, np.nan, -np.nan, 1e-45, -1e-45, 3.4e38], np.float32)
    for weights in (np.zeros((2, n + 40), np.float32), rng.choice(some, (2, n + 40)).astype(np.float32),
                    rng.choice(some[:4], (2, n + 40)).astype(np.float32),
                    (1 + rng.integers(0, 3, (2, n + 40)) * 2.0 ** -23).astype(np.float32)):
        for budget in (1, 100, 2500, n - 1):
            Both([n, 4097], 40, (n + 40) // 40, weights=weights, seed=budget).evict([budget, budget // 2], 7)


def test_a_long_row():
    Both([70001, 8193], 16, 4400, ((4,),), seed=5).evict([20000, 8000], 512)
    Both([70001], 16, 4400, ((4,),), seed=6).evict([69999], 0)


def test_shared_prefixes_and_repeats():
    b = Both([300, 310, 200, 250], 16, 24, ((8, 16),), seed=2, shared=9)
    b.evict([200, 150, 10, 0], 20)
    b.evict([150, 150, 150, 150], 0)  # (what is shared is more)
    b.evict([0, 0, 0, 0], 3)


def test_pages_outside_are_passed_over():
    b = Both([100, 80], 16, 9, ((2, 8),), seed=3)
    for r, c, x in ((0, 2, -1), (0, 5, len(b.cache.counts)), (1, 0, 2 ** 31 - 1), (1, 3, -7)):
        b.cache.table[r][c] = x
        b.table[r, c] = x
    b.evict([50, 30], 4)


def test_a_pool_without_pages():
    """Rows whose pages are all outside: nothing is read or moved, the rows get shorter all the same."""
    table, lengths = _i32([[0, 3, -1, 1]]), _i32([60])
    weights, kept = torch.arange(64.0, device="cuda")[None], torch.empty(1, 64, dtype=torch.int32, device="cuda")
    counts, budget, ws = _i32([0]), _i32([20]), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    t = _lib.CacheTable(rows=1, max_pages=4, num_pages=0, page_size=16, block_table=table.data_ptr(),
                        lengths=lengths.data_ptr(), refcounts=counts.data_ptr())
    pool = (_lib.CachePool * 1)(_lib.CachePool(None, 512, 512))
    assert _lib.lib().dm_cache_evict_workspace(ctypes.byref(t)) <= ws.numel()
    rc = _lib.lib().dm_cache_evict(ctypes.byref(t), pool, 1, weights.data_ptr(), 64, budget.data_ptr(), 5, kept.data_ptr(),
                                   ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.DM_OK
    torch.cuda.synchronize()
    assert lengths.tolist() == [20] and kept[0, :21].tolist() == [*range(40, 60), -1]
    assert weights[0, :21].tolist() == [float(x) for x in range(40, 60)] + [0.0] and table.tolist() == [[0, 3, -1, -1]]


def test_lengths_past_the_table_and_below_zero():
    b = Both([64, 64, 30], 16, 4, seed=4)
    b.cache.lengths[0] = 1000
    b.cache.lengths[2] = -3
    b.lengths[0], b.lengths[2] = 1000, -3
    b.evict([20, 64, 0], 5)


def test_many_pools_and_wide_pages():
    """More pools than one launch takes; rows of 2, 4, 6, 8, 24 and 4096 bytes."""
    Both([90, 40], 16, 7, ((2,),) * 35, seed=1).evict([30, 30], 4)
    for shape, dtype in (((1,), np.int16), ((2,), np.int16), ((3,), np.int16), ((4,), np.int16), ((12,), np.int16),
                         ((4096,), np.int8), ((1,), np.int8), ((5, 7), np.int8), ((100,), np.int64)):
        Both([300, 280], 8, 40, (shape,), dtype, seed=7).evict([100, 131], 9)


def test_strided_weights_and_a_stream():
    b = Both([90, 80], 16, 7, seed=9)
    wide = torch.full((2, 120), -1.0, device="cuda")
    wide[:, 4:116] = b.weights
    b.weights = wide[:, 4:116]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b.evict([40, 50], 6)
    assert (wide[:, :4] == -1).all() and (wide[:, 116:] == -1).all()


def test_pools_past_32_bits():
    """Pages 3 GB apart: the places of the third on lie past 2^32 bytes."""
    b = Both([50, 40], 16, 6, ((2, 8),) * 2, seed=3, spare=0)
    n, each = len(b.cache.counts), 16 * 2 * 8
    buf = torch.empty((n - 1) * (3 << 29) + 2 * each, dtype=torch.int16, device="cuda")
    for i, p in enumerate(b.pools):
        b.pools[i] = buf.as_strided(p.shape, (3 << 29, 16, 8, 1), i * each).copy_(p)
    b.evict([20, 33], 4)


def test_what_the_workspace_holds(monkeypatch):
    """Nothing of a call's workspace is read before the call has written it."""
    for fill in (0, 255):
        monkeypatch.setattr(ops, "_workspace", lambda n, dev: torch.full((max(int(n), 1),), fill, dtype=torch.uint8, device=dev))
        Both([9000, 40, 4097, 700], 16, 570, ((2, 8),), seed=fill, shared=2).evict([1000, 20, 4096, 700], 9)


def test_two_streams_at_once():
    """Calls of two caches in flight together."""
    two = [Both([6000, 900], 16, 380, ((8, 16),), seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in two]
    budgets = [_i32([2000, 300]), _i32([100, 899])]
    kept = []
    torch.cuda.synchronize()
    for s, b, n in zip(streams, two, budgets):
        with torch.cuda.stream(s):
            kept.append(dm.cache_evict(b.pools, b.weights, b.table, b.lengths, b.counts, n, 64))
    torch.cuda.synchronize()
    for b, n, k in zip(two, budgets, kept):
        assert k.tolist() == b.cache.evict(n.tolist(), 64)
        b.same()


def test_graph():
    """A captured eviction, replayed on rows that have changed."""
    state = [Both([500, 300, 77], 16, 40, ((8, 16),) * 2, seed=s) for s in (1, 2, 3)]
    at, caches = state[0], [s.cache for s in state]
    live = [at.weights, at.table, at.lengths, at.counts, *at.pools]
    first = [[x.clone() for x in (s.weights, s.table, s.lengths, s.counts, *s.pools)] for s in state]
    budgets = _i32([200, 100, 90])
    run = lambda: dm.cache_evict(at.pools, at.weights, at.table, at.lengths, at.counts, budgets, 16)  # noqa: E731
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        kept = run()
    for i, new in ((1, [200, 100, 90]), (2, [40, 299, 0]), (0, [500, 1, 50])):
        for x, y in zip(live, first[i]):
            x.copy_(y)
        budgets.copy_(_i32(new))
        g.replay()
        torch.cuda.synchronize()
        at.cache = caches[i]
        assert kept.tolist() == at.cache.evict(new, 16)
        at.same()
