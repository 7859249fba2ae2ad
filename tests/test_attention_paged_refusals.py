"""What the attention of new tokens over a paged cache and the eviction refuse, without a GPU."""
import ctypes

import pytest
import torch

import dashmag_amd as dm
from dashmag_amd import _lib, ops
from dashmag_amd.contract import Unsupported

CPU = torch.device("cpu")


def test_the_mirror_refuses():
    op = "attention_paged"
    ok = lambda **kw: ops._paged_arrays(op, **{**dict(block_table=torch.zeros(2, 3, dtype=torch.int32),  # noqa: E731
                                                      lengths=[3, 4], cu_seqlens=[0, 2, 5], n=5, device=CPU), **kw})
    ok()
    ok(cu_seqlens=None, n=2)
    ok(cu_seqlens=[1, 1, 4])
    for kw, what in [(dict(lengths=[1]), "the block table is"), (dict(lengths=[[1, 2]]), "the cache lengths are"),
                     (dict(lengths=[0.5, 1.0]), "whole numbers"), (dict(cu_seqlens=None), "one token a sequence"),
                     (dict(cu_seqlens=[0, 5]), r"cu_seqlens is \[S \+ 1\]"), (dict(cu_seqlens=[0, 3, 2]), "must go from"),
                     (dict(cu_seqlens=[-1, 3, 5]), "must go from"), (dict(cu_seqlens=[0, 3, 6]), "must go from"),
                     (dict(block_table=torch.zeros(6, dtype=torch.int32)), "the block table is")]:
        with pytest.raises(Unsupported, match="^attention_paged: .*" + what):
            ok(**kw)
    for f, n in ((dm.attention_paged, 5), (dm.attention_paged_with_lse, 5), (dm.attention_paged_with_weights, 6)):
        with pytest.raises(Unsupported, match="on the GPU"):
            f(*[torch.zeros(1)] * n)
    with pytest.raises(Unsupported, match="^cache_evict: .*on the GPU"):
        dm.cache_evict([torch.zeros(2, 2)], *[torch.zeros(2, 2, dtype=torch.int32)] * 4, [1, 1])


@pytest.mark.parametrize("w,what", [(torch.zeros(2, 5), "one a key"), (torch.zeros(3, 6), "one a key"),
                                    (torch.zeros(2, 6, dtype=torch.float64), "one a key"),
                                    (torch.zeros(6, 2).t(), "each contiguous and apart"),
                                    (torch.zeros(6).expand(2, 6), "each contiguous and apart"),
                                    (torch.zeros(10).as_strided((2, 6), (4, 1)), "each contiguous and apart")])
def test_weights(w, what):
    with pytest.raises(Unsupported, match="^op: .*" + what):
        ops._paged_weights("op", w, 2, 6)
    assert ops._paged_weights("op", torch.zeros(2, 9)[:, :6], 2, 6) == 9
    assert ops._paged_weights("op", None, 2, 6) == 0


def _call(ws=1 << 40, ps=16, mp=4, bt=256, ln=256, np=4, w=None, stride=64, **kw):
    x = dict(b=2, tq=2, tk=64, hq=4, hkv=2, d=64, dtype=_lib.DM_BF16)
    x.update(kw)
    d = _lib.AttentionDesc(**x)
    rc = _lib.lib().dm_attention_paged(ctypes.byref(d), None, None, None, np, ps, bt, mp, ln, None, None, w, stride,
                                       None, ws, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("kw,what", [
    (dict(hq=3), "multiple of the key-value heads"), (dict(d=300), "above 256"), (dict(dtype=9), "dtype"),
    (dict(b=-1), "bad dimensions"), (dict(tq=-1), "bad dimensions"), (dict(ps=0), "page_size"), (dict(mp=-1), "page_size"),
    (dict(np=-1), "page_size"), (dict(mp=3), "desc->tk (64)"), (dict(bt=None), "block table"),
    (dict(ln=None), "block table"), (dict(ws=0), "workspace"), (dict(cu_seqlens_k=256), "cu_seqlens_q alone"),
    (dict(mask_kind=1), "cu_seqlens_q alone"), (dict(tq=3), "one token a sequence"), (dict(b=1 << 40), "more tokens"),
    (dict(tq=1 << 40), "more tokens"), (dict(tq=1 << 25), "more tokens"), (dict(np=1 << 32), "more tokens"),
    (dict(tk=(1 << 30) + 16, mp=(1 << 26) + 1), "more tokens"), (dict(w=256, stride=63), "their rows apart"),
    (dict(strided=1, sk=_lib.Strides(0, -1, 0)), "strides"), (dict(strided=1, sq=_lib.Strides(0, -1, 0)), "strides")])
def test_the_library_refuses(kw, what):
    rc, msg = _call(**kw)
    assert rc == _lib.DM_ERR_REFUSED and msg.startswith("attention_paged: ") and what in msg


@pytest.mark.parametrize("kw", [dict(b=-1), dict(b=1 << 40), dict(hkv=0), dict(d=1 << 40), dict(tk=1 << 40),
                                dict(hq=1 << 40), dict(tq=1 << 40), dict(hq=3), dict(tq=-2)])
def test_workspace_of_refused_sizes(kw):
    x = dict(b=2, tq=2, tk=64, hq=4, hkv=2, d=64, dtype=_lib.DM_BF16)
    x.update(kw)
    assert _lib.lib().dm_attention_paged_workspace(ctypes.byref(_lib.AttentionDesc(**x)), 16, 1) == 0
    assert _lib.lib().dm_attention_paged_workspace(None, 16, 1) == 0
    assert _lib.lib().dm_attention_paged_workspace(ctypes.byref(_lib.AttentionDesc(**dict(x, b=2, tq=2, tk=64, hq=4,
                                                                                         hkv=2, d=64))), 0, 0) == 0


def test_nothing_to_do_launches_nothing():
    assert _call(tq=0, b=0)[0] == _lib.DM_OK
    assert _call(hq=0)[0] == _lib.DM_OK
    assert _evict(rows=0)[0] == _lib.DM_OK
    assert _evict(max_pages=0)[0] == _lib.DM_OK


def _evict(ws=1 << 40, pools=(), w=256, stride=64, b=256, kept=256, recent=0, **kw):
    x = dict(rows=2, max_pages=4, num_pages=9, page_size=16, block_table=256, lengths=256, refcounts=256)
    x.update(kw)
    t = _lib.CacheTable(**x)
    arr = (_lib.CachePool * max(1, len(pools)))(*pools)
    rc = _lib.lib().dm_cache_evict(ctypes.byref(t), arr, len(pools), w, stride, b, recent, kept, None, ws, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("kw,what", [
    (dict(page_size=0), "page_size"), (dict(rows=-1), "page_size"), (dict(num_pages=1 << 22), "page_size"),
    (dict(lengths=None), "missing"), (dict(refcounts=None), "missing"), (dict(block_table=None), "missing"),
    (dict(w=None), "missing"), (dict(b=None), "missing"), (dict(kept=None), "missing"), (dict(ws=0), "workspace"),
    (dict(recent=-1), "recent"), (dict(stride=63), "their rows apart"), (dict(rows=(1 << 22) + 1), "at most 2^22"),
    (dict(max_pages=(1 << 26) + 1), "at most 2^30"), (dict(rows=1 << 22, max_pages=1 << 13, page_size=1), "less than 2^35"),
    (dict(rows=1 << 22, pools=[_lib.CachePool(256, 32, 32)]), "more rows and bytes"),
    (dict(rows=1 << 20, pools=[_lib.CachePool(256, 1 << 16, 1 << 16)]), "more rows and bytes"),
    (dict(pools=[_lib.CachePool(256, 24, 24)]), "a pool's pages"), (dict(pools=[_lib.CachePool(256, 32, 32)] * 2), "two of them"),
    (dict(pools=[_lib.CachePool(256, 64, 128), _lib.CachePool(4096, 64, 128), _lib.CachePool(304, 32, 128)]), "two of them"),
    (dict(pools=[_lib.CachePool(256, 64, 128), _lib.CachePool(368, 32, 128)]), "two of them"),
    (dict(pools=[_lib.CachePool(256, 32, 64), _lib.CachePool(320, 16, 128)]), "two of them"), (dict(pools=[_lib.CachePool(None, 32, 32)]), "missing")])
def test_the_eviction_refuses(kw, what):
    rc, msg = _evict(**kw)
    assert rc == _lib.DM_ERR_REFUSED and msg.startswith("cache_evict: ") and what in msg


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(page_size=0), dict(rows=1 << 30), dict(max_pages=1 << 30)])
def test_evicts_workspace_of_refused_sizes(kw):
    x = dict(rows=2, max_pages=4, num_pages=9, page_size=16)
    x.update(kw)
    assert _lib.lib().dm_cache_evict_workspace(ctypes.byref(_lib.CacheTable(**x))) == 0
    assert _lib.lib().dm_cache_evict_workspace(None) == 0
