"""Serving with keys given up, as a program runs an attention layer: prompts arrive in chunks whose tokens are
written to pages and attended, with the keys' weights accumulated; a row is forked; rows over their budgets give up
keys; single tokens go on at their own positions. Each step against the 64-bit attention over what each sequence
still holds; which keys go is the oracle's, from the weights that the GPU has accumulated."""
import numpy as np
import pytest
import torch

import dashmag_amd as dm
import rope_cases as rc
from chunk_cases import held_lse
from evict_oracle import Evicting
from shared_cases import U

pytestmark = pytest.mark.gpu


def _want(q, keys, values, n):
    """(out, lse, p, off, loff, poff) of the last n tokens of a row that holds `keys`: chunk_cases' bounds."""
    k, v = (torch.stack(x).double().transpose(0, 1) for x in (keys, values))
    x, d = k.shape[1], k.shape[2]
    seen = torch.arange(x) <= torch.arange(x - n, x)[:, None]
    y = q.double().unflatten(1, (k.shape[0], -1)).permute(1, 2, 0, 3)
    z = (y @ k.transpose(1, 2)[:, None] * d ** -0.5).masked_fill(~seen, -torch.inf)
    total = torch.logsumexp(z, -1, keepdim=True)
    p = torch.exp(z - total)
    s = ((y.abs() @ k.abs().transpose(1, 2)[:, None]) * d ** -0.5).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    e = (d + 16) * U * s
    half = torch.finfo(q.dtype).eps / 2 if q.dtype != torch.float32 else 0.0
    bound = (half + 2 * e + 2 * (x / 16 + 64) * U) * (p @ v[:, None].abs())
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -25 * seen.double() @ v[:, None].abs()
    g = e + (x / 16 + 64) * U + 8 * U * (total.abs() + 1)
    back = lambda t: t.permute(2, 0, 1, 3).flatten(1, 2)  # noqa: E731
    rows = p.shape[0] * p.shape[1] * n
    return (back(p @ v[:, None]), back(total)[..., 0], p.sum((0, 1, 2)), back(bound), back(g)[..., 0],
            (p * (e + g + (rows + 40) * U)).sum((0, 1, 2)))


@pytest.mark.parametrize("dtype,hq,hkv,d,n,page", [(torch.bfloat16, 8, 2, 128, 64, 16), (torch.float16, 4, 4, 64, 16, 32),
                                                   (torch.float32, 4, 1, 64, 32, 7)])
def test_serving(dtype, hq, hkv, d, n, page):
    gen = torch.Generator().manual_seed(d + page)
    rows, cols, pages = 5, 60 if page == 7 else 30, 400
    cap = cols * page
    kp, vp = (torch.full((pages, page, hkv, d), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    table = torch.full((rows, cols), -1, dtype=torch.int32, device="cuda")
    lengths, counts = (torch.zeros(x, dtype=torch.int32, device="cuda") for x in (rows, pages))
    weights = torch.zeros(rows, cap, device="cuda")
    wq, wk = (1 + 0.1 * torch.randn(d, generator=gen) for _ in range(2))
    freq = (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float()
    norms = [x.cuda() for x in (wq, wk, freq)]
    keys, values, places = ([[] for _ in range(rows)] for _ in range(3))
    told, off = (torch.zeros(rows, cap, dtype=torch.float64) for _ in range(2))  # the weights in 64 bits

    def step(new):
        want = [len(x) + m for x, m in zip(keys, new)]
        assert dm.cache_reserve(table, lengths, counts, torch.tensor(want, dtype=torch.int32), page).all()
        cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32).cuda()
        total = sum(new)
        q, k, v = (torch.randn(total, h, d, generator=gen).to(dtype) for h in (hq, hkv, hkv))
        at = torch.tensor([len(places[r]) + i for r, m in enumerate(new) for i in range(m)])
        qo = dm.qk_norm_rope_paged(q.cuda(), k.cuda(), v.cuda(), *norms, kp, vp, table, lengths, cu, None, at)
        qw, ko = (x[0] for x in dm.qk_norm_rope(q[None].cuda(), k[None].cuda(), *norms, at))
        assert torch.equal(qo, qw)
        out, lse = dm.attention_paged_with_weights(qo, kp, vp, table, lengths, weights, cu)
        x = 0
        for r, m in enumerate(new):
            for i in range(m):
                keys[r].append(ko[x + i].cpu()), values[r].append(v[x + i]), places[r].append(int(at[x + i]))
            if m:
                o, l, p, ob, lb, pb = _want(qo[x:x + m].cpu(), keys[r], values[r], m)
                rc.held(f"row {r}", out[x:x + m], o, ob)
                held_lse(f"row {r} lse", lse[x:x + m], l, lb)
                told[r, :len(p)] += p
                off[r, :len(p)] += pb + U * told[r, :len(p)]
            x += m
        worst = float(((weights.cpu().double() - told).abs() / off.clamp(min=1e-300)).max())
        print(f"weights: {worst:.3f} of the bound", flush=True)
        assert worst <= 1.0

    def evict(budgets, recent):
        state = weights.cpu().tolist(), table.tolist(), lengths.tolist(), counts.tolist()
        c = Evicting(state[1], state[2], state[3], page, weights=state[0])
        kept = dm.cache_evict([kp, vp], weights, table, lengths, counts, torch.tensor(budgets), recent)
        assert kept.tolist() == c.evict(budgets, recent)
        assert table.tolist() == c.table and lengths.tolist() == c.lengths and counts.tolist() == c.counts
        assert weights.tolist() == c.weights
        for r, row in enumerate(kept.tolist()):
            row = [j for j in row if j >= 0]
            keys[r], values[r] = [keys[r][j] for j in row], [values[r][j] for j in row]
            m = len(told[r, :]) - len(row)
            told[r], off[r] = (torch.cat([y[r, row], y.new_zeros(m)]) for y in (told, off))
            off[r, :len(row)] += 1e-300

    step([150, 40, 0, 3, 0])
    step([60, 1, 0, 90, 0])
    fresh = dm.cache_fork([kp, vp], table, lengths, counts, [0], [2])
    assert int(fresh[0]) >= 0 or 210 % page == 0
    keys[2], values[2], places[2] = list(keys[0]), list(values[0]), list(places[0])
    weights[2], told[2], off[2] = weights[0], told[0], off[0]
    step([1, 2, 5, 1, 0])
    evict([100, 30, 60, 40, 0], 8)
    for i in range(3):
        step([1, 1, 1, 1, 0])
    step([0, 70, 0, 33, 12])
    dm.cache_free(table, lengths, counts, [0], page)  # (what row 2 shares with it is its own now)
    keys[0], values[0], places[0] = [], [], []
    weights[0], told[0], off[0] = 0.0, 0.0, 0.0
    evict([0, 64, 50, 20, 12], 4)
    assert len(keys[2]) == 50
    step([9, 1, 1, 1, 1])
    dm.cache_compact([kp, vp], table, lengths, counts)
    step([1, 1, 40, 1, 1])
    dm.cache_free(table, lengths, counts, list(range(rows)), page)
    assert not counts.any()
