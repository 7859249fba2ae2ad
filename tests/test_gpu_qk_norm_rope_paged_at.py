"""The library's two entry points of the norms and rotation into a paged cache: one goes by the places alone, whatever
positions its descriptor holds, the other by those positions."""
import ctypes

import pytest
import torch

import dashmag_amd as dm
from dashmag_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,code,d,n", [(torch.bfloat16, _lib.DM_BF16, 128, 64), (torch.float32, _lib.DM_F32, 50, 11)])
def test_positions_of_the_descriptor(dtype, code, d, n):
    gen = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn(9, h, d, generator=gen).to(dtype).cuda() for h in (4, 2, 2))
    freq = (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float().cuda()
    table = torch.arange(6, dtype=torch.int32).view(2, 3).cuda()
    ln, cu = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([20, 40], [0, 3, 9]))
    at = torch.arange(700, 709).cuda()
    pages = [torch.zeros(6, 16, 2, d, dtype=dtype, device="cuda") for _ in range(2)]

    def call(f, positions):
        out = torch.empty_like(q)
        for x in pages:
            x.zero_()
        desc = _lib.QkNormRopeDesc(b=1, t=9, hq=4, hkv=2, d=d, n=n, dtype=code, weight_dtype=_lib.DM_F32, eps=1e-6,
                                   positions=positions, positions_i64=1)
        each = _lib.Strides(16 * 2 * d, 2 * d, d)
        pg = _lib.KvPages(num_pages=6, page_size=16, max_pages=3, nseq=2, block_table=table.data_ptr(),
                          lengths=ln.data_ptr(), cu_seqlens=cu.data_ptr(), sk=each, sv=each)
        rc = f(ctypes.byref(desc), ctypes.byref(pg), q.data_ptr(), k.data_ptr(), v.data_ptr(), None, None, freq.data_ptr(),
               out.data_ptr(), pages[0].data_ptr(), pages[1].data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == _lib.DM_OK, _lib.last_error()
        return out, *(x.clone() for x in pages)

    def mirror(positions):
        mine = [torch.zeros_like(x) for x in pages]
        out = dm.qk_norm_rope_paged(q, k, v, None, None, freq, *mine, table, ln, cu, dm.QkNormRopeOptions(eps=1e-6), positions)
        return out, *mine

    lib = _lib.lib()
    places, turned = mirror(None), mirror(at)
    assert not torch.equal(places[0], turned[0])
    for f, positions, want in ((lib.dm_qk_norm_rope_paged, None, places), (lib.dm_qk_norm_rope_paged, at.data_ptr(), places),
                               (lib.dm_qk_norm_rope_paged_at, None, places),
                               (lib.dm_qk_norm_rope_paged_at, at.data_ptr(), turned)):
        assert all(torch.equal(x, y) for x, y in zip(call(f, positions), want))
