"""The norms and rotation into a paged cache at positions of the caller's: the queries and keys that the same
call without pages gives, in the places that the lengths say."""
import pytest
import torch

import dashmag_amd as dm
from dashmag_amd.contract import Unsupported

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d,n,page", [(torch.bfloat16, 128, 64, 16), (torch.float16, 96, 24, 7),
                                            (torch.float32, 64, 32, 16), (torch.bfloat16, 50, 11, 4)], ids=str)
@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
def test_positions(dtype, d, n, page, ints):
    gen = torch.Generator().manual_seed(d)
    new, lengths = [5, 0, 40, 1], [30, 17, 40, 0]
    total, cols = sum(new), -(-40 // page)
    q, k, v = (torch.randn(total, h, d, generator=gen).to(dtype).cuda() for h in (6, 2, 2))
    w = [(1 + 0.1 * torch.randn(d, generator=gen)).cuda() for _ in range(2)]
    freq = (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float().cuda()
    at = torch.randint(0, 1 << 20, (total,), generator=gen).to(ints).cuda()
    kp, vp = (torch.zeros(4 * cols, page, 2, d, dtype=dtype, device="cuda") for _ in range(2))
    table = torch.randperm(4 * cols, generator=gen).view(4, cols).to(torch.int32).cuda()
    cu = torch.tensor([0, 5, 5, 45, 46], dtype=torch.int32).cuda()
    ln = torch.tensor(lengths, dtype=torch.int32).cuda()
    out = dm.qk_norm_rope_paged(q, k, v, *w, freq, kp, vp, table, ln, cu, None, at)
    qw, kw = (x[0] for x in dm.qk_norm_rope(q[None], k[None], *w, freq, at))
    assert torch.equal(out[:45], qw[:45]) and not out[45].any()  # (a length of 0: no token)
    token = 0
    for r, (m, x) in enumerate(zip(new, lengths)):
        for i in range(m if x else 0):
            j = x - m + i
            pg = int(table[r, j // page])
            assert torch.equal(kp[pg, j % page], kw[token + i]) and torch.equal(vp[pg, j % page], v[token + i])
        token += m
    assert int((vp.flatten(2) != 0).any(-1).sum()) == 45
    # places alone: the same as before
    kp2, vp2 = torch.zeros_like(kp), torch.zeros_like(vp)
    own = torch.tensor([x - m + i for m, x in zip(new, lengths) for i in range(m)], dtype=ints).clamp(min=0).cuda()
    a = dm.qk_norm_rope_paged(q, k, v, *w, freq, kp, vp, table, ln, cu)
    b = dm.qk_norm_rope_paged(q, k, v, *w, freq, kp2, vp2, table, ln, cu, None, own)
    assert torch.equal(a, b) and torch.equal(kp, kp2) and torch.equal(vp, vp2)
    for bad, what in ((at[:-1], "the positions are"), (at.float(), "whole numbers")):
        with pytest.raises(Unsupported, match="^qk_norm_rope_paged: .*" + what):
            dm.qk_norm_rope_paged(q, k, v, *w, freq, kp, vp, table, ln, cu, None, bad)
