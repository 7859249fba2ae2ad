"""The sequential pages of pages_oracle.py by hand, and what the device operations refuse, without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

import dashmag_amd as dm
from dashmag_amd import _lib, ops
from dashmag_amd.contract import Unsupported
from pages_oracle import Cache


def test_a_round_by_hand():
    pool = np.arange(6 * 2).reshape(6, 2)
    c = Cache([[-1] * 4 for _ in range(4)], [0] * 4, [0] * 6, 2, [pool])
    assert c.reserve([3, 0, 9, 2]) == [True, True, False, True]  # nine keys are past the table
    assert c.table[0] == [0, 1, -1, -1] and c.table[3] == [2, -1, -1, -1]
    assert c.fork([0, 0, 3], [1, 1, 2]) == [3, -2, -1]
    assert c.table[1] == [0, 3, -1, -1] and c.table[2] == [2, -1, -1, -1]
    assert c.counts == [2, 1, 2, 1, 0, 0] and c.pools[0][3].tolist() == [2, 7]
    assert c.reserve([3, 3, 8, 0]) == [True, True, False, True] and c.lengths == [3, 3, 2, 2]
    c.free([0, 0, 9, 3])
    assert c.counts == [1, 0, 1, 1, 0, 0] and c.table[0] == [-1] * 4
    assert c.compact() == [0, -1, 2, 1, -1, -1] and c.table[1] == [0, 1, -1, -1]


def _arrays(rows=3, cols=4, pages=10):
    return (torch.full((rows, cols), -1, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32),
            torch.zeros(pages, dtype=torch.int32))


def test_the_mirror_refuses():
    t, n, c = _arrays()
    ops._cache_desc("cache_free", t, n, c, 16)
    for args, what in [((t.long(), n, c, 16), "the block table"), ((t.t(), n, c, 16), "the block table"),
                       ((t, n[:, None], c, 16), "the cache lengths"), ((t, n[:2], c, 16), "the cache lengths"),
                       ((t, n, c.float(), 16), "the page counts"), ((t, n, c, 0), "at least one key")]:
        with pytest.raises(Unsupported, match="^cache_free: .*" + what):
            ops._cache_desc("cache_free", *args)
    cpu = torch.device("cpu")
    pool = torch.zeros(10, 16, 2, 8)
    arr, page = ops._cache_pools("cache_fork", [pool, torch.zeros(10, 2, 16, 4)[:, 1]], 10, cpu)
    assert page == 16 and arr[0].page_bytes == 1024 and arr[1].page_stride == 512 and arr[1].page_bytes == 256
    for pools, what in [([], "list of at least one"), (pool, "list of at least one"),
                        ([pool, torch.zeros(9, 16, 2)], "one page_size"), ([pool, torch.zeros(10, 8, 2)], "one page_size"),
                        ([pool.transpose(2, 3)], "contiguous"), ([pool[:1].expand(10, 16, 2, 8)], "contiguous"),
                        ([torch.zeros(10)], "page_size"), ([torch.zeros(10, 0, 4)], "at least one key")]:
        with pytest.raises(Unsupported, match="^cache_fork: .*" + what):
            ops._cache_pools("cache_fork", pools, 10, cpu)
    with pytest.raises(Unsupported, match="on the GPU"):
        dm.cache_free(t, n, c, [0], 16)


def _table(**kw):
    x = dict(rows=3, max_pages=4, num_pages=10, page_size=16, block_table=256, lengths=256, refcounts=256)
    x.update(kw)
    return _lib.CacheTable(**x)


@pytest.mark.parametrize("kw,what", [(dict(rows=-1), "not negative"), (dict(page_size=0), "not negative"),
                                     (dict(num_pages=1 << 31), "not negative"), (dict(max_pages=-4), "not negative"),
                                     (dict(block_table=None), "missing"), (dict(lengths=None), "missing"),
                                     (dict(refcounts=None), "missing")])
def test_the_library_refuses_tables(kw, what):
    lb, t = _lib.lib(), ctypes.byref(_table(**kw))
    pool = _lib.CachePool(pages=256, page_bytes=64, page_stride=64)
    for op, rc in [("cache_reserve", lb.dm_cache_reserve(t, 256, 256, None, 1 << 50, None)),
                   ("cache_fork", lb.dm_cache_fork(t, ctypes.byref(pool), 1, 256, 256, 1, 256, None, 1 << 50, None)),
                   ("cache_free", lb.dm_cache_free(t, 256, 1, None)),
                   ("cache_compact", lb.dm_cache_compact(t, ctypes.byref(pool), 1, 256, None, 1 << 50, None))]:
        assert rc == _lib.DM_ERR_REFUSED
    for op, call in [("cache_reserve", lambda: lb.dm_cache_reserve(t, 256, 256, None, 1 << 50, None)),
                     ("cache_free", lambda: lb.dm_cache_free(t, 256, 1, None))]:
        call()
        assert _lib.last_error().startswith(op + ": ") and what in _lib.last_error()
    if what == "not negative":
        assert lb.dm_cache_reserve_workspace(t) == lb.dm_cache_fork_workspace(t, 1) == 0
        assert lb.dm_cache_compact_workspace(t) == 0


def test_the_library_refuses_the_rest():
    lb, t = _lib.lib(), ctypes.byref(_table())
    big, pool = 1 << 50, _lib.CachePool(pages=256, page_bytes=64, page_stride=64)

    def said(rc, op, what):
        assert rc == _lib.DM_ERR_REFUSED and _lib.last_error().startswith(op + ": ") and what in _lib.last_error()
    said(lb.dm_cache_reserve(t, None, 256, None, big, None), "cache_reserve", "missing")
    said(lb.dm_cache_reserve(t, 256, 256, None, 0, None), "cache_reserve", "workspace")
    said(lb.dm_cache_free(t, None, 1, None), "cache_free", "missing")
    said(lb.dm_cache_free(t, 256, -1, None), "cache_free", "rows are [N]")
    said(lb.dm_cache_free(t, 256, 1 << 40, None), "cache_free", "rows are [N]")
    p = ctypes.byref(pool)
    said(lb.dm_cache_fork(t, p, 1, None, 256, 1, 256, None, big, None), "cache_fork", "missing")
    said(lb.dm_cache_fork(t, p, 1, 256, 256, -1, 256, None, big, None), "cache_fork", "[N]")
    said(lb.dm_cache_fork(t, None, 1, 256, 256, 1, 256, None, big, None), "cache_fork", "pools are missing")
    said(lb.dm_cache_fork(t, p, 1, 256, 256, 1, 256, None, 0, None), "cache_fork", "workspace")
    said(lb.dm_cache_compact(t, p, 1, None, None, big, None), "cache_compact", "missing")
    said(lb.dm_cache_compact(t, p, 1, 256, None, 0, None), "cache_compact", "workspace")
    for kw in (dict(page_bytes=63), dict(page_stride=32), dict(page_bytes=-16), dict(page_stride=1 << 60)):
        bad = _lib.CachePool(**{**dict(pages=256, page_bytes=64, page_stride=64), **kw})
        said(lb.dm_cache_compact(t, ctypes.byref(bad), 1, 256, None, big, None), "cache_compact", "a pool's pages")
    assert lb.dm_cache_free(t, None, 0, None) == _lib.DM_OK
    assert lb.dm_cache_fork(t, p, 1, None, None, 0, None, None, big, None) == _lib.DM_OK
