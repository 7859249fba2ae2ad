"""Evictions of as many rows as a call takes."""
import ctypes

import pytest
import torch

from dashmag_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [65534, 65536, 131071, 1 << 22])
def test_rows_of_more_than_one_launch(rows):
    """Rows of up to two keys, cut to their budgets, with no pools to move: each row's lengths, kept keys, weights,
    entries and counts."""
    gen = torch.Generator().manual_seed(rows)
    lengths, budgets = (torch.randint(0, 3, (rows,), generator=gen, dtype=torch.int32) for _ in range(2))
    w = torch.randint(0, 5, (rows, 2), generator=gen).float()
    n = torch.minimum(lengths, budgets)
    first = torch.where((lengths == 2) & (n == 1) & (w[:, 1] > w[:, 0]), 1, 0)  # (ties to the first)
    kept = torch.full((rows, 2), -1, dtype=torch.int32)
    kept[:, 0] = torch.where(n > 0, first.int(), -1)
    kept[:, 1] = torch.where(n == 2, 1, -1)
    after = w.clone()
    cut = n < lengths
    after[:, 0] = torch.where(cut, torch.where(n > 0, w.gather(1, first[:, None].long())[:, 0], 0.0), w[:, 0])
    after[:, 1] = torch.where(cut & (lengths == 2), 0.0, w[:, 1])
    pages = 1 << 20
    table = torch.randint(0, pages, (rows, 2), generator=gen, dtype=torch.int32)
    held = torch.arange(2) < lengths[:, None]
    table = torch.where(held, table, -1)
    # (no page counts as another row's)
    counts = torch.zeros(pages, dtype=torch.int32)
    gone = held & (torch.arange(2) >= n[:, None])
    want_counts = counts - torch.bincount(table[gone].long(), minlength=pages).int()
    dev = [x.cuda() for x in (table, lengths, counts, w, budgets)]
    t = _lib.CacheTable(rows=rows, max_pages=2, num_pages=pages, page_size=1, block_table=dev[0].data_ptr(),
                        lengths=dev[1].data_ptr(), refcounts=dev[2].data_ptr())
    out = torch.empty(rows, 2, dtype=torch.int32, device="cuda")
    ws = torch.empty(_lib.lib().dm_cache_evict_workspace(ctypes.byref(t)), dtype=torch.uint8, device="cuda")
    print(f"{rows} rows", flush=True)
    rc = _lib.lib().dm_cache_evict(ctypes.byref(t), (_lib.CachePool * 1)(), 0, dev[3].data_ptr(), 2, dev[4].data_ptr(), 0,
                                   out.data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.DM_OK, _lib.last_error()
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), kept) and torch.equal(dev[1].cpu(), n) and torch.equal(dev[3].cpu(), after)
    assert torch.equal(dev[0].cpu(), torch.where(gone, -1, table)) and torch.equal(dev[2].cpu(), want_counts)
