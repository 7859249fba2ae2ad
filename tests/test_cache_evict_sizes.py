"""What the eviction of keys refuses by its size and its arrays, without a GPU."""
import ctypes

import pytest

from dashmag_amd import _lib


def _evict(rows, pools, **kw):
    x = dict(rows=rows, max_pages=4, num_pages=9, page_size=16, block_table=256, lengths=256, refcounts=256)
    x.update(kw)
    arr = (_lib.CachePool * len(pools))(*pools)
    rc = _lib.lib().dm_cache_evict(ctypes.byref(_lib.CacheTable(**x)), arr, len(pools), 256, 64, 256, 0, 256, None,
                                   1 << 40, None)
    return rc, _lib.last_error()


def _pools(widths):
    """Pools of 16 keys of so many bytes a page, behind one another."""
    at, out = 1 << 20, []
    for w in widths:
        out.append(_lib.CachePool(at, 16 * w, 16 * w))
        at += 9 * 16 * w
    return out


@pytest.mark.parametrize("rows,widths", [(16384, [1 << 16] + [2] * 31), (16384, [2] * 31 + [1 << 16]), (1 << 17, [2, 2, 16384, 2, 2, 2]),
                                         (1 << 20, [2] * 8), (16384, [2] * 40 + [1 << 16] + [2] * 23)])
def test_more_workgroups_than_a_launch_has(rows, widths):
    """A launch has as many columns for each of its pools as the widest one needs."""
    rc, msg = _evict(rows, _pools(widths))
    assert rc == _lib.DM_ERR_REFUSED and msg.startswith("cache_evict: ") and "more rows and bytes" in msg
