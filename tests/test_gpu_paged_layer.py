"""The operators around a paged cache run together, as a serving program runs an attention layer: pages
reserved, a prompt's keys and values appended, the prompt forked, a token of every sequence appended and
attended for several steps, some sequences ended, the pool closed up, and on. Each step's output is the
64-bit causal attention over what each sequence holds, of queries and keys as the layer rounds them."""
import numpy as np
import pytest
import torch

import dashmag_amd as dm
import rope_cases as rc
from shared_cases import U

pytestmark = pytest.mark.gpu


def _want(q, keys, values):
    """(output, bound) of one row, as shared_cases derives it."""
    k, v = (torch.stack(x).double().transpose(0, 1) for x in (keys, values))  # [Hkv, n, D]
    n, d = k.shape[1:]
    x = q.double().unflatten(0, (k.shape[0], -1))
    p = torch.softmax(x @ k.transpose(1, 2) * d ** -0.5, -1)
    s = (x.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * d ** -0.5
    bound = (torch.finfo(q.dtype).eps / 2 + 2 * (d + 16) * U * s + 2 * (n / 16 + 64) * U) * (p @ v.abs())
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -25 * v.abs().sum(1, keepdim=True)
    return (p @ v).flatten(0, 1), bound.flatten(0, 1)


@pytest.mark.parametrize("dtype,hq,hkv,d,n,page", [(torch.bfloat16, 8, 2, 128, 64, 16),
                                                   (torch.float16, 4, 4, 64, 16, 32),
                                                   (torch.bfloat16, 8, 1, 256, 32, 16)])
def test_serving(dtype, hq, hkv, d, n, page):
    gen = torch.Generator().manual_seed(d)
    rows, cols, pages = 7, 20, 90
    kp, vp = (torch.full((pages, page, hkv, d), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    table = torch.full((rows, cols), -1, dtype=torch.int32, device="cuda")
    lengths, counts = (torch.zeros(x, dtype=torch.int32, device="cuda") for x in (rows, pages))
    wq, wk = (0.1 * torch.randn(d, generator=gen) for _ in range(2))
    freq = (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float()
    opts = dm.QkNormRopeOptions(unit_offset=True)
    weights = [x.cuda() for x in (wq, wk, freq)]
    held_k, held_v = [[] for _ in range(rows)], [[] for _ in range(rows)]  # what each row holds, on the host

    def append(new):
        """new[r] tokens to each row: reserved, normalised, rotated, written; returns the last ones' queries."""
        want = [len(x) + m for x, m in zip(held_k, new)]
        granted = dm.cache_reserve(table, lengths, counts, torch.tensor(want, dtype=torch.int32), page)
        assert granted.all()
        cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
        total = int(cu[-1])
        q, k, v = (torch.randn(total, h, d, generator=gen).to(dtype) for h in (hq, hkv, hkv))
        # (rows without new tokens are of length 0 here: they take none)
        ln = torch.where(torch.tensor(new) > 0, lengths.cpu(), 0).to(torch.int32).cuda()
        qo = dm.qk_norm_rope_paged(q.cuda(), k.cuda(), v.cuda(), *weights, kp, vp, table, ln, cu.cuda(), opts)
        at = [len(held_k[r]) + i for r, m in enumerate(new) for i in range(m)]
        turn = rc.turns(freq, at, n, d, False)
        rc.held("q", qo, *rc.forward(q, wq, True, 1e-6, turn))
        ko, _ = dm.qk_norm_rope(k[None].cuda(), k[None, :, :0].cuda(), weights[1], None, weights[2],
                                torch.tensor(at), opts)
        x = 0
        for r, m in enumerate(new):
            for i in range(m):
                held_k[r].append(ko[0, x].cpu()), held_v[r].append(v[x])
                x += 1
        return qo

    def attend(q, groups, prefix):
        out = dm.attention_decode_shared(q, kp, vp, table, lengths, groups, prefix)
        assert torch.equal(torch.isnan(out), torch.zeros_like(out, dtype=torch.bool))
        for r in range(rows):
            if not held_k[r]:
                assert not out[r].any()
            else:
                rc.held(f"row {r}", out[r], *_want(q[r].cpu(), held_k[r], held_v[r]))
        paged = dm.attention_decode_paged(q, kp, vp, table, lengths)
        assert (out.double() - paged.double()).abs().max() <= 0.05

    append([0, 93, 0, 0, 0, 40, 0])
    fresh = dm.cache_fork([kp, vp], table, lengths, counts, [1, 1, 1, 5], [0, 2, 3, 6])
    assert (fresh >= 0).all()
    for r, p in ((0, 1), (2, 1), (3, 1), (6, 5)):
        held_k[r], held_v[r] = list(held_k[p]), list(held_v[p])
    groups, prefix = torch.tensor([0, 4, 5, 7]), torch.tensor([93, 0, 40])
    for step in range(4):
        q = append([1, 1, 1, 1, 0, 1, 1])
        q = torch.cat([q[:4], torch.randn(1, hq, d, generator=gen).to(dtype).cuda(), q[4:]])
        attend(q, groups, prefix)
        if step == 1:  # two sequences end, a prompt arrives, the pool is closed up
            dm.cache_free(table, lengths, counts, [0, 5], page)
            for r in (0, 5):
                held_k[r], held_v[r] = [], []
            append([0, 0, 0, 0, 70, 3, 0])
            moved = dm.cache_compact([kp, vp], table, lengths, counts)
            used = int((counts > 0).sum())
            assert int(moved.max()) == used - 1 and int(table.max()) == used - 1
            groups, prefix = torch.tensor([1, 4]), torch.tensor([93])
            q = torch.randn(rows, hq, d, generator=gen).to(dtype).cuda()
            attend(q, groups, prefix)
            append([2, 0, 0, 0, 0, 0, 0])
    dm.cache_free(table, lengths, counts, list(range(rows)), page)
    assert not counts.any() and (table == -1).all() and not lengths.any()


def test_a_training_layer():
    """Norms and rotation, attention and its backward, the norms' backward: against the same in 64 bits
    under autograd. Roundings to bf16 in between: queries, keys, the output, the gradients of each (six
    half steps of 2^-9 of the value's scale, against the largest value of each result: 6 of 2^-8 at most)."""
    gen = torch.Generator().manual_seed(1)
    t, hq, hkv, d, n = 200, 4, 2, 64, 32
    q, k, v, do = (torch.randn(1, t, h, d, generator=gen).bfloat16() for h in (hq, hkv, hkv, hq))
    wq, wk = (1 + 0.1 * torch.randn(d, generator=gen) for _ in range(2))
    freq = (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float()
    opts = dm.AttentionOptions(causal=True)
    c = [x.cuda() for x in (q, k, v, do, wq, wk, freq)]
    qr, kr = dm.qk_norm_rope(c[0], c[1], *c[4:])
    o, lse = dm.attention_with_lse(qr, kr, c[2], None, opts)
    gq, gk, gv = dm.attention_backward(qr, kr, c[2], o, lse, c[3], None, opts)
    got = [o, *dm.qk_norm_rope_backward(c[0], c[1], *c[4:], gq, gk), gv]
    x = [a.double().requires_grad_() for a in (q, k, v, wq, wk)]
    turn = rc.turns(freq, range(t), n, d, False)

    def rotate(a, w):
        c, s, partner = turn
        y = a[0] / (a[0].square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        return (y * c + y[..., partner] * s).transpose(0, 1)
    qq, kk = rotate(x[0], x[3]), rotate(x[1], x[4]).repeat_interleave(hq // hkv, 0)
    mask = torch.ones(t, t, dtype=torch.bool).tril()
    p = torch.softmax((qq @ kk.transpose(1, 2) * d ** -0.5).masked_fill(~mask, -torch.inf), -1)
    out = (p @ x[2][0].transpose(0, 1).repeat_interleave(hq // hkv, 0)).transpose(0, 1)[None]
    out.backward(do.double())
    for name, a, b in zip(("o", "dq", "dk", "dwq", "dwk", "dv"), got,
                          (out.detach(), x[0].grad, x[1].grad, x[3].grad, x[4].grad, x[2].grad)):
        off = float((a.cpu().double() - b).abs().max() / b.abs().max())
        print(name, off, flush=True)
        assert off <= 6 * 2.0 ** -8, (name, off)
