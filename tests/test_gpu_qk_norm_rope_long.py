"""The norms and rotation of more tokens than the kernels' workgroups take a tile of: those then go through
further tiles, whose angles, places and first heads are fetched while they work on the one in front. Against
the 64-bit forms of rope_cases.py.

A forward has 4096 workgroups at most, of tiles of up to 16 tokens (fewer where a token's heads fill the
workgroup): more than 4096 tiles are two and more a workgroup, and the last tile is ragged here."""
import pytest
import torch

import dashmag_amd as dm
import rope_cases as rc

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(dtype, t, hq, hkv, d, n, seed):
    gen = torch.Generator().manual_seed(seed)
    q, k, v, gq, gk = (torch.randn(t, h, d, generator=gen).to(dtype) for h in (hq, hkv, hkv, hq, hkv))
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=gen)).to(dtype) for _ in range(2))
    freq = (10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float()
    return gen, q, k, v, gq, gk, wq, wk, freq


# tokens, heads: tiles of 16 tokens (4376 tiles), of 2 (4151), of 8 (4126)
CASES = [
    (BF, 70003, 1, 1, 64, 32, False),
    (BF, 70003, 1, 1, 64, 16, True),
    (F16, 70003, 2, 0, 80, 40, False),
    (BF, 70003, 0, 2, 64, 32, False),     # keys alone
    (F32, 8301, 12, 4, 256, 64, True),
    (F32, 33003, 6, 2, 128, 64, False),
    (BF, 70003, 1, 1, 56, 28, False),     # the simple kernels: a token at a time
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_forward_and_backward_of_many_tiles(case):
    dtype, t, hq, hkv, d, n, inter = case
    gen, q, k, _, gq, gk, wq, wk, freq = _inputs(dtype, t, hq, hkv, d, n, t + d)
    p = torch.randint(0, 1 << 20, (t,), generator=gen)
    opts = dm.QkNormRopeOptions(interleaved=inter)
    cuda = [x[None].cuda() for x in (q, k, gq, gk)]
    w = [x.cuda() for x in (wq, wk, freq)]
    outs = dm.qk_norm_rope(*cuda[:2], *w, p.cuda(), opts)
    grads = dm.qk_norm_rope_backward(*cuda[:2], *w, *cuda[2:], p.cuda(), opts)
    turn = rc.turns(freq, p.numpy(), n, d, inter)
    for name, x, wt, z, out, dx, dw in (("q", q, wq, gq, outs[0], grads[0], grads[2]),
                                        ("k", k, wk, gk, outs[1], grads[1], grads[3])):
        if not x.numel():
            assert not out.numel() and not dx.numel() and not dw.any()
            continue
        rc.held(name, out[0], *rc.forward(x, wt, False, opts.eps, turn))
        want, bound, wantw, boundw = rc.backward(x, wt, False, opts.eps, turn, z)
        rc.held("d" + name, dx[0], want, bound)
        # A weight's gradient: a lane's own heads of the 768 workgroups' tokens, the lanes' and then the
        # workgroups' sums, 12 of these a thread and 64 threads; terms off by 48 u as in rope_cases.
        bound = boundw / (48 + 96 + x.shape[1] * -(-t // 1024)) * (48 + x.shape[1] * -(-t // 768) + 64 + 12 + 64)
        rc.held("dw" + name, dw, wantw, bound)


# dtype, page, hq, hkv, D, n, interleaved
PAGED = [
    (BF, 16, 1, 1, 64, 32, False),
    (BF, 7, 2, 1, 64, 8, True),
    (F32, 32, 1, 2, 128, 64, False),
    (BF, 16, 0, 1, 64, 32, False),
    (BF, 16, 1, 1, 56, 28, False),
]


@pytest.mark.parametrize("case", PAGED, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_many_tiles_into_pages(case):
    """Four prompts of 70003 tokens in all, one of them the padding of a batch (length 0), one whose first
    tokens lie in front of its sequence's start, and rows behind the last one."""
    dtype, page, hq, hkv, d, n, inter = case
    new, lengths = [30001, 9, 4002, 35987], [30040, 9, 0, 35980]
    t = sum(new) + 4
    gen, q, k, v, _, _, wq, wk, freq = _inputs(dtype, t, hq, hkv, d, n, page + d)
    each = [-(-x // page) for x in lengths]
    perm = torch.randperm(sum(each) + 3, generator=gen)
    table = torch.full((4, max(each) + 1), -1, dtype=torch.int32)
    at, seq, pos = 0, [], []
    for s, x in enumerate(each):
        table[s, :x] = perm[at:at + x]
        at += x
        seq += [s] * new[s]
        pos += range(lengths[s] - new[s], lengths[s])
    seq, pos = torch.tensor(seq + [0] * 4), torch.tensor(pos + [-1] * 4)
    cut = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    opts = dm.QkNormRopeOptions(interleaved=inter)
    kp, vp = (torch.full((len(perm), page, hkv, d), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    qo = dm.qk_norm_rope_paged(*(x.cuda() for x in (q, k, v, wq, wk, freq)), kp, vp, table.cuda(),
                               torch.tensor(lengths, dtype=torch.int32).cuda(), cut.cuda(), opts).cpu()
    has = pos >= 0
    turn = rc.turns(freq, pos[has].numpy(), n, d, inter)
    if hq:
        rc.held("q", qo[has], *rc.forward(q[has], wq, False, opts.eps, turn))
        assert not qo[~has].any()
    slots = table[seq[has], pos[has] // page].long() * page + pos[has] % page
    kp, vp = (x.cpu().flatten(0, 1) for x in (kp, vp))
    rc.held("k", kp[slots], *rc.forward(k[has], wk, False, opts.eps, turn))
    assert torch.equal(vp[slots], v[has])
    rest = torch.ones(len(kp), dtype=torch.bool)
    rest[slots] = False
    assert torch.isnan(kp[rest]).all() and torch.isnan(vp[rest]).all()
