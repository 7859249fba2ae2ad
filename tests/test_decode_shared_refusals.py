"""What the shared-prefix decode refuses, without a GPU."""
import ctypes

import pytest
import torch

import dashmag_amd as dm
from dashmag_amd import _lib, ops
from dashmag_amd.contract import Unsupported


def test_the_mirror_refuses():
    cpu, op = torch.device("cpu"), "attention_decode_shared"
    ok = lambda **kw: ops._shared_arrays(op, **{**dict(lengths=[3, 4], groups=[0, 2], prefix_lengths=[2],  # noqa: E731
                                                       b=2, device=cpu), **kw})
    ok()
    ok(lengths=None, groups=[0], prefix_lengths=torch.zeros(0, dtype=torch.int32))
    for kw, what in [(dict(lengths=[1]), "the cache lengths are"), (dict(groups=[0, 3]), "groups must go"),
                     (dict(groups=[2, 0]), "groups must go"), (dict(groups=[-1, 2]), "groups must go"),
                     (dict(prefix_lengths=[1, 2]), "the prefix lengths are"),
                     (dict(groups=[[0, 2]]), r"groups is \[G \+ 1\]"),
                     (dict(groups=[]), r"groups is \[G \+ 1\]"),
                     (dict(prefix_lengths=[0.5]), "whole numbers")]:
        with pytest.raises(Unsupported, match="^attention_decode_shared: .*" + what):
            ok(**kw)
    with pytest.raises(Unsupported, match="on the GPU"):
        dm.attention_decode_shared(*[torch.zeros(1)] * 7)


def _call(ws=1 << 40, ps=16, mp=4, bt=256, g=256, ng=1, pl=256, **kw):
    x = dict(b=2, tq=1, tk=64, hq=4, hkv=2, d=64, dtype=_lib.DM_BF16)
    x.update(kw)
    d = _lib.AttentionDesc(**x)
    rc = _lib.lib().dm_attention_decode_shared(ctypes.byref(d), None, None, None, 4, ps, bt, mp, None, g, ng, pl,
                                               None, None, ws, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("kw,what", [
    (dict(hq=3), "multiple of the key-value heads"), (dict(d=300), "above 256"), (dict(dtype=9), "dtype"),
    (dict(b=-1), "bad dimensions"), (dict(ps=0), "page_size"), (dict(mp=-1), "page_size"), (dict(ng=-1), "ngroups"),
    (dict(mp=3), "desc->tk (64)"), (dict(bt=None), "block table"), (dict(g=None), "groups is [G + 1]"),
    (dict(pl=None), "groups is [G + 1]"), (dict(ws=0), "workspace"), (dict(cu_seqlens_k=256), "not cu_seqlens_k"),
    (dict(b=1 << 40), "more rows"), (dict(b=1 << 30, hq=64), "more rows"), (dict(ng=1 << 40), "more rows"),
    (dict(tk=(1 << 30) + 16, mp=(1 << 26) + 1), "more rows"),
    (dict(strided=1, sk=_lib.Strides(0, -1, 0)), "strides")])
def test_the_library_refuses(kw, what):
    rc, msg = _call(**kw)
    assert rc == _lib.DM_ERR_REFUSED and msg.startswith("attention_decode_shared: ") and what in msg


@pytest.mark.parametrize("kw", [dict(b=-1), dict(b=1 << 40), dict(hkv=0), dict(d=1 << 40), dict(tk=1 << 40),
                                dict(hq=1 << 40)])
def test_workspace_of_refused_sizes(kw):
    x = dict(b=2, tq=1, tk=64, hq=4, hkv=2, d=64, dtype=_lib.DM_BF16)
    x.update(kw)
    assert _lib.lib().dm_attention_decode_shared_workspace(ctypes.byref(_lib.AttentionDesc(**x)), 16, 1) == 0
    assert _lib.lib().dm_attention_decode_shared_workspace(None, 16, 1) == 0


def test_nothing_to_do_launches_nothing():
    assert _call(b=0)[0] == _lib.DM_OK
    assert _call(hq=0)[0] == _lib.DM_OK
