"""What the norms and the rotation of queries and keys refuse, without a GPU: the host mirror's
descriptor checks on CPU tensors, and the C entry points before any launch."""
import ctypes

import pytest
import torch

import dashmag_amd as dm
from dashmag_amd import _lib, ops
from dashmag_amd.contract import Unsupported


def _desc(q, k, wq=None, wk=None, freq=None, paged=False):
    return ops._qk_norm_rope_desc("qk_norm_rope", q, k, wq, wk, torch.zeros(4) if freq is None else freq,
                                  dm.QkNormRopeOptions(), paged)


def test_the_mirror_refuses():
    z = torch.zeros
    q, k = z(2, 3, 4, 16), z(2, 3, 2, 16)
    assert _desc(q, k, z(16), z(16)).n == 4
    for args, what in [((q[0], k[0]), r"query and key are \[B, T, H, D\]"),
                       ((q, z(2, 4, 2, 16)), "the same tokens"), ((q, z(2, 3, 2, 8)), "one head dimension"),
                       ((q, k.half()), "one dtype"), ((q, k, z(15)), r"q_weight is \[D\]"),
                       ((q, k, None, z(16).half()), "k_weight must be f32"),
                       ((q.half(), k.half(), z(16), z(16).half()), "share one dtype"),
                       ((q, k, None, None, z(9)), "2 n at most"), ((q, k, None, None, z(4).half()), "f32"),
                       ((q, k, None, None, z(2, 2)), "inv_freq"), ((q.double(), k.double()), "dtype")]:
        with pytest.raises(Unsupported, match="^qk_norm_rope: .*" + what):
            _desc(*args)
    with pytest.raises(Unsupported, match=r"\[N, H, D\]"):
        _desc(q, k, paged=True)
    with pytest.raises(Unsupported, match="on the GPU"):
        dm.qk_norm_rope(q, k, None, None, z(4))


def test_positions():
    desc = _desc(torch.zeros(2, 3, 4, 16), torch.zeros(2, 3, 2, 16))
    cpu = torch.device("cpu")
    assert ops._positions("qk_norm_rope", desc, None, cpu) is None and not desc.positions
    p = torch.arange(6).view(2, 3)
    assert ops._positions("qk_norm_rope", desc, p, cpu) is not None
    assert desc.positions_i64 == 1 and desc.positions_b == 3
    ops._positions("qk_norm_rope", desc, torch.arange(3, dtype=torch.int32), cpu)
    assert desc.positions_i64 == 0 and desc.positions_b == 0
    for bad in (torch.zeros(2, 3), torch.arange(6), torch.zeros(3, 2, dtype=torch.int64)):
        with pytest.raises(Unsupported, match="^qk_norm_rope: the positions"):
            ops._positions("qk_norm_rope", desc, bad, cpu)


def test_pages_that_cannot_be_written_in_place():
    ok = torch.zeros(4, 16, 2, 8)
    ops._in_pages("qk_norm_rope_paged", ok, "key_pages")
    for bad in (ok.transpose(2, 3), torch.zeros(1, 16, 2, 8).expand(4, 16, 2, 8)):
        with pytest.raises(Unsupported, match="^qk_norm_rope_paged: key_pages"):
            ops._in_pages("qk_norm_rope_paged", bad, "key_pages")


def test_arrays_of_whole_numbers():
    cpu = torch.device("cpu")
    a = torch.tensor([1, 2], dtype=torch.int32)
    assert ops._device_i32("cache_free", a, cpu, "rows").data_ptr() == a.data_ptr()
    assert ops._device_i32("cache_free", [3, 4], cpu, "rows").tolist() == [3, 4]
    for bad, what in (([1.5], "whole numbers"), ([1 << 31], "fit in int32")):
        with pytest.raises(Unsupported, match="^cache_free: rows must .*" + what):
            ops._device_i32("cache_free", bad, cpu, "rows")


def _c(**kw):
    x = dict(b=1, t=4, hq=2, hkv=1, d=64, n=32, dtype=_lib.DM_BF16, weight_dtype=_lib.DM_BF16, eps=1e-6)
    x.update(kw)
    return _lib.QkNormRopeDesc(**x)


@pytest.mark.parametrize("kw,what", [
    (dict(t=-1), "bad dimensions"), (dict(b=1 << 40, t=1 << 40), "bad dimensions"),
    (dict(b=1 << 30, t=1 << 30), "bad dimensions"),
    (dict(hq=-1), "bad dimensions"), (dict(d=257), "above 256"), (dict(n=33), "2 n at most"),
    (dict(n=-1), "2 n at most"), (dict(dtype=7), "dtype"), (dict(weight_dtype=_lib.DM_F16), "weights"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(positions_b=-1), "strides"),
    (dict(strided=1, sq=_lib.Strides(0, -1, 0)), "strides")])
def test_the_library_refuses(kw, what):
    lb, d = _lib.lib(), _c(**kw)
    assert lb.dm_qk_norm_rope(ctypes.byref(d), *[None] * 8) == _lib.DM_ERR_REFUSED
    assert _lib.last_error().startswith("qk_norm_rope: ") and what in _lib.last_error()
    nbytes = lb.dm_qk_norm_rope_bwd_workspace(ctypes.byref(d))
    assert nbytes <= 1024 * 2 * 256 * 4
    assert lb.dm_qk_norm_rope_bwd(ctypes.byref(d), *[None] * 12, nbytes, None) == _lib.DM_ERR_REFUSED
    assert _lib.last_error().startswith("qk_norm_rope_backward: ") and what in _lib.last_error()


def test_the_library_refuses_a_small_workspace_and_no_descriptor():
    lb, d = _lib.lib(), _c()
    need = lb.dm_qk_norm_rope_bwd_workspace(ctypes.byref(d))
    assert need > 0
    assert lb.dm_qk_norm_rope_bwd(ctypes.byref(d), *[None] * 12, need - 1, None) == _lib.DM_ERR_REFUSED
    assert "workspace" in _lib.last_error()
    assert lb.dm_qk_norm_rope(None, *[None] * 8) == _lib.DM_ERR_REFUSED
    assert lb.dm_qk_norm_rope_bwd_workspace(None) == 0


@pytest.mark.parametrize("kw,pkw,what", [
    (dict(b=2), {}, "B = 1"), ({}, dict(page_size=0), "page_size"), ({}, dict(num_pages=-1), "page_size"),
    ({}, dict(nseq=3), "one token a sequence"), ({}, dict(lengths=None), "block table"),
    ({}, dict(block_table=None), "block table"), ({}, dict(sk=_lib.Strides(-1, 0, 0)), "strides")])
def test_the_library_refuses_pages(kw, pkw, what):
    lb, d = _lib.lib(), _c(**kw)
    x = dict(num_pages=4, page_size=16, max_pages=2, nseq=4, block_table=256, lengths=256)
    x.update(pkw)
    p = _lib.KvPages(**x)
    assert lb.dm_qk_norm_rope_paged(ctypes.byref(d), ctypes.byref(p), *[None] * 10) == _lib.DM_ERR_REFUSED
    assert _lib.last_error().startswith("qk_norm_rope_paged: ") and what in _lib.last_error()
    assert lb.dm_qk_norm_rope_paged(ctypes.byref(d), None, *[None] * 10) == _lib.DM_ERR_REFUSED
