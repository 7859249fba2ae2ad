"""The queries' and keys' norms and rotation on the GPU, forward, backward and into pages, against
the 64-bit forms of rope_cases.py, whose bounds are derived there."""
import pytest
import torch

import dashmag_amd as dm
import rope_cases as rc

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# (dtype, weights' dtype or None, B, T, Hq, Hkv, D, n, interleaved, unit_offset, positions)
CASES = [
    (BF, BF, 1, 300, 8, 2, 128, 64, False, False, "none"),
    (BF, F32, 2, 77, 16, 2, 256, 32, False, True, "i32"),
    (F16, F16, 3, 65, 4, 4, 64, 32, True, False, "i64"),
    (BF, None, 1, 5, 5, 1, 128, 64, True, False, "row"),
    (F32, F32, 2, 129, 4, 2, 64, 32, False, False, "far"),
    (F32, F32, 1, 40, 3, 1, 128, 16, True, True, "far"),
    (F32, None, 1, 33, 2, 2, 256, 128, False, False, "negative"),
    (BF, BF, 1, 1, 1, 1, 64, 8, False, False, "none"),
    (BF, F32, 2, 31, 3, 1, 96, 48, False, False, "i32"),   # lanes without pieces
    (F16, F16, 1, 70, 5, 2, 80, 40, False, True, "far"),
    (BF, BF, 2, 333, 6, 3, 80, 16, True, False, "i32"),
    (F32, F32, 1, 45, 3, 3, 80, 8, False, False, "i64"),
    (F32, None, 2, 19, 4, 2, 96, 36, True, True, "far"),
    (BF, BF, 1, 2300, 12, 4, 96, 16, True, False, "none"),
    (F16, F32, 1, 61, 4, 2, 192, 96, False, False, "negative"),
    (BF, BF, 1, 200, 5, 1, 192, 32, True, True, "i32"),
    (F32, F32, 1, 26, 2, 1, 192, 64, False, False, "far"),
    (F16, F32, 1, 30, 3, 2, 104, 12, True, True, "i64"),    # the simple kernels: widths
    (BF, BF, 1, 30, 3, 2, 112, 56, False, False, "i64"),
    (F16, F32, 1, 30, 3, 2, 96, 12, True, True, "i64"),
    (F32, F32, 1, 9, 2, 1, 7, 3, False, False, "i32"),
    (BF, BF, 1, 64, 7, 3, 128, 20, False, False, "i32"),    # pairs of no whole piece
    (BF, BF, 1, 50, 6, 2, 64, 0, False, True, "none"),      # no rotation
    (F16, F16, 1, 1200, 4, 1, 64, 32, False, False, "far"),
    (BF, BF, 2, 1100, 40, 8, 128, 64, False, False, "i32"),
]


def _positions(kind, b, t, gen):
    if kind == "none":
        return None, torch.arange(t).repeat(b)
    if kind == "row":
        p = torch.randint(0, 5000, (t,), generator=gen)
        return p.to(torch.int32).cuda(), p.repeat(b)
    hi = {"i32": 9000, "i64": 9000, "far": (1 << 31) - 1, "negative": 3000}[kind]
    p = torch.randint(-3000 if kind == "negative" else 0, hi, (b, t), generator=gen)
    return (p if kind == "i64" else p.to(torch.int32)).cuda(), p.reshape(-1)


def _inputs(dtype, wd, b, t, hq, hkv, d, n, unit, seed):
    gen = torch.Generator().manual_seed(seed)
    q, k, gq, gk = (torch.randn(b, t, h, d, generator=gen).to(dtype) for h in (hq, hkv, hq, hkv))
    q *= torch.exp(2 * torch.randn(b, t, hq, 1, generator=gen)).to(dtype)
    wq, wk = (None if wd is None else ((0 if unit else 1) + 0.3 * torch.randn(d, generator=gen)).to(wd)
              for _ in range(2))
    freq = (10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float()
    return gen, q, k, gq, gk, wq, wk, freq


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_forward_and_backward(case):
    dtype, wd, b, t, hq, hkv, d, n, inter, unit, places = case
    gen, q, k, gq, gk, wq, wk, freq = _inputs(dtype, wd, b, t, hq, hkv, d, n, unit, 3 * t + d)
    at, p = _positions(places, b, t, gen)
    opts = dm.QkNormRopeOptions(interleaved=inter, unit_offset=unit)
    eps = opts.eps
    cq, ck, cgq, cgk, cwq, cwk, cf = _cuda(q, k, gq, gk, wq, wk, freq)
    qo, ko = dm.qk_norm_rope(cq, ck, cwq, cwk, cf, at, opts)
    dq, dk, dwq, dwk = dm.qk_norm_rope_backward(cq, ck, cwq, cwk, cf, cgq, cgk, at, opts)
    again = dm.qk_norm_rope_backward(cq, ck, cwq, cwk, cf, cgq, cgk, at, opts)
    turn = rc.turns(freq, p.numpy(), n, d, inter)
    for name, x, w, z, out, dx, dw in (("q", q, wq, gq, qo, dq, dwq), ("k", k, wk, gk, ko, dk, dwk)):
        x, z = x.flatten(0, 1), z.flatten(0, 1)
        rc.held(name, out.flatten(0, 1), *rc.forward(x, w, unit, eps, turn))
        want, bound, wantw, boundw = rc.backward(x, w, unit, eps, turn, z)
        rc.held("d" + name, dx.flatten(0, 1), want, bound)
        if w is None:
            assert dw is None
        else:
            assert dw.dtype == w.dtype
            rc.held("dw" + name, dw, wantw, boundw)
    for a, c in zip((dq, dk, dwq, dwk), again):
        assert a is None or torch.equal(a, c)


def test_gradients_against_differences():
    """The loss sum(z y) moved by a step along a direction of each input, in 64 bits on the host: the
    difference quotient is the gradient's product with the direction to the step's third power."""
    b, t, hq, hkv, d, n = 1, 6, 3, 2, 64, 24
    gen, q, k, gq, gk, wq, wk, freq = _inputs(F32, F32, b, t, hq, hkv, d, n, False, 9)
    dq, dk, dwq, dwk = (x.cpu().double() for x in dm.qk_norm_rope_backward(
        *_cuda(q, k, wq, wk, freq, gq, gk)))
    turn = rc.turns(freq, range(t), n, d, False)

    def loss(q, k, wq, wk):
        return sum((rc.forward(x[0], w, False, 1e-6, turn)[0] * z[0].double()).sum()
                   for x, w, z in ((q, wq, gq), (k, wk, gk)))
    args = [x.double() for x in (q, k, wq, wk)]
    for i, grad in enumerate((dq, dk, dwq, dwk)):
        u = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        up, down = ([a + s * h * u if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        want = float((loss(*up) - loss(*down)) / (2 * h))
        got = float((grad * u).sum())
        scale = float((grad.abs() * u.abs()).sum())
        # f32 gradients: 96 u of each term's parts, which are at most some tens of the term
        assert abs(got - want) <= 1e-4 * scale, (i, got, want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_views_are_read_in_place(dtype):
    """Slices of one projection, heads ahead of the time, a batch of which every second row is taken, an
    f32 base off 16 bytes: the contiguous call's bits."""
    b, t, hq, hkv, d, n = 2, 70, 4, 2, 128, 64
    gen, q, k, gq, gk, wq, wk, freq = _inputs(dtype, dtype, b, t, hq, hkv, d, n, False, 21)
    wq, wk, freq = _cuda(wq, wk, freq)
    want = dm.qk_norm_rope(*_cuda(q, k), wq, wk, freq)
    wantb = dm.qk_norm_rope_backward(*_cuda(q, k), wq, wk, freq, *_cuda(gq, gk))
    fused = torch.cat([q, k, k], 2).cuda()
    ahead = [x.cuda().transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, gq, gk)]
    second = [torch.stack([x, x], 1).flatten(0, 1).cuda()[::2] for x in (q, k, gq, gk)]
    off = []
    for x in (q, k, gq, gk):
        flat = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:]
        off.append(flat.copy_(x.reshape(-1)).view(x.shape))
    for x in ([fused[:, :, :hq], fused[:, :, hq:hq + hkv], gq.cuda(), gk.cuda()], ahead, second, off):
        got = dm.qk_norm_rope(x[0], x[1], wq, wk, freq)
        gotb = dm.qk_norm_rope_backward(x[0], x[1], wq, wk, freq, x[2], x[3])
        same = torch.equal if x is not off or dtype == BF else (
            lambda a, c: bool(((a - c).abs() <= 96 * rc.U * c.abs().max()).all()))
        assert all(same(a, c) for a, c in zip(got, want))
        assert all(same(a, c) for a, c in zip(gotb[:2], wantb[:2]))


def test_a_bad_value_stays_in_its_head():
    b, t, hq, hkv, d = 1, 20, 4, 2, 128
    gen, q, k, gq, gk, wq, wk, freq = _inputs(BF, BF, b, t, hq, hkv, d, 64, False, 4)
    q[0, 3, 1, 7], q[0, 5, 2, 0], q[0, 6, 0] = float("nan"), float("inf"), 0.0
    qo, ko = dm.qk_norm_rope(*_cuda(q, k, wq, wk, freq))
    bad = ~torch.isfinite(qo).all(-1).cpu()
    want = torch.zeros(b, t, hq, dtype=torch.bool)
    want[0, 3, 1] = want[0, 5, 2] = True
    assert torch.equal(bad, want) and torch.isfinite(ko).all()
    assert (qo[0, 6, 0] == 0).all()


@pytest.mark.parametrize("b,t,hq,hkv", [(0, 5, 2, 1), (2, 0, 2, 1), (1, 3, 0, 2), (1, 3, 2, 0)])
def test_nothing_to_do(b, t, hq, hkv):
    gen, q, k, gq, gk, wq, wk, freq = _inputs(BF, BF, b, t, hq, hkv, 64, 32, False, 4)
    qo, ko = dm.qk_norm_rope(*_cuda(q, k, wq, wk, freq))
    dq, dk, dwq, dwk = dm.qk_norm_rope_backward(*_cuda(q, k, wq, wk, freq, gq, gk))
    assert qo.shape == q.shape and ko.shape == k.shape and dq.shape == q.shape and dk.shape == k.shape
    for h, dw in ((hq, dwq), (hkv, dwk)):
        assert dw.shape == (64,) and (b * t * h > 0 or not dw.any())


# ------------------------------------------------------------------------------------------
# Into pages
# ------------------------------------------------------------------------------------------

def _paged_case(dtype, new, held, page, hq, hkv, d, seed, spare=4, cu=True):
    """Sequences of new[s] tokens behind held[s] others; pages of NaN; a table of shuffled pages."""
    gen = torch.Generator().manual_seed(seed)
    total = sum(new)
    lengths = [a + c for a, c in zip(new, held)]
    each = [-(-x // page) for x in lengths]
    perm = torch.randperm(sum(each) + spare, generator=gen)
    table = torch.full((len(new), max(each + [0]) + 1), -1, dtype=torch.int32)
    at = 0
    for s, x in enumerate(each):
        table[s, :x] = perm[at:at + x]
        at += x
    pages = [torch.full((len(perm), page, hkv, d), float("nan"), dtype=dtype) for _ in range(2)]
    q, k, v = (torch.randn(total, h, d, generator=gen).to(dtype) for h in (hq, hkv, hkv))
    cut = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    return q, k, v, pages, table, torch.tensor(lengths, dtype=torch.int32), cut


def _check_paged(case, page, opts, weights, freq, n, outs, skip=()):
    """The query and the pages after the call; sequences in ``skip`` wrote nothing."""
    q, k, v, pages, table, lengths, cut = case
    qo, kp, vp = outs
    d = q.shape[-1]
    p, seq = [], []
    for s in range(len(lengths)):
        m = int(cut[s + 1] - cut[s])
        p += range(int(lengths[s]) - m, int(lengths[s]))
        seq += [s] * m
    turn = rc.turns(freq, p, n, d, opts.interleaved)
    rc.held("q", qo[:len(p)], *rc.forward(q[:len(p)], weights[0], opts.unit_offset, opts.eps, turn))
    want, bound = rc.forward(k[:len(p)], weights[1], opts.unit_offset, opts.eps, turn)
    slots = torch.tensor([int(table[s, x // page]) * page + x % page for s, x in zip(seq, p)], dtype=torch.long)
    wrote = torch.tensor([s not in skip for s in seq], dtype=torch.bool)
    slots, kept = slots[wrote], torch.nonzero(wrote)[:, 0]
    rc.held("k", kp.cpu().flatten(0, 1)[slots], want[kept], bound[kept])
    assert torch.equal(vp.cpu().flatten(0, 1)[slots], v[kept])
    for x in (kp, vp):
        rest = torch.ones(x.shape[0] * page, dtype=torch.bool)
        rest[slots] = False
        assert torch.isnan(x.cpu().flatten(0, 1)[rest]).all()  # nothing else was written


PAGED = [
    (BF, [1] * 9, [0, 1, 14, 15, 16, 17, 400, 31, 2], 16, 8, 2, 128, 64, False),
    (F16, [5, 1, 0, 40, 16], [3, 15, 7, 0, 32], 16, 4, 4, 64, 32, True),
    (BF, [33, 2, 70], [100, 0, 5], 7, 6, 2, 256, 32, False),
    (F32, [3, 9], [0, 8], 32, 2, 1, 128, 64, False),
    (BF, [1, 4], [6, 0], 16, 3, 3, 96, 12, True),
    (BF, [1500, 1], [17, 30], 64, 4, 1, 64, 8, False),
    (F16, [40, 3], [9, 0], 16, 4, 2, 80, 40, False),
    (BF, [7, 21], [0, 50], 16, 4, 2, 96, 48, True),
    (F32, [7, 21], [0, 50], 16, 2, 2, 96, 48, False),
    (BF, [90, 5], [0, 50], 16, 6, 2, 192, 32, False),
]


@pytest.mark.parametrize("case", PAGED, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_paged(case):
    dtype, new, held, page, hq, hkv, d, n, inter = case
    c = _paged_case(dtype, new, held, page, hq, hkv, d, sum(new) + d)
    q, k, v, pages, table, lengths, cut = c
    gen = torch.Generator().manual_seed(5)
    wq, wk = ((0.2 * torch.randn(d, generator=gen)).to(dtype) for _ in range(2))
    freq = (500.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float()
    opts = dm.QkNormRopeOptions(eps=1e-5, interleaved=inter, unit_offset=True)
    kp, vp = (x.cuda() for x in pages)
    qo = dm.qk_norm_rope_paged(*_cuda(q, k, v, wq, wk, freq), kp, vp, table.cuda(), lengths.cuda(),
                               cut.cuda(), opts)
    _check_paged(c, page, opts, (wq, wk), freq, n, (qo, kp, vp))
    if all(x == 1 for x in new):
        kp2, vp2 = (x.cuda() for x in pages)
        one = dm.qk_norm_rope_paged(*_cuda(q, k, v, wq, wk, freq), kp2, vp2, table, lengths, None, opts)
        assert torch.equal(one, qo) and all(torch.equal(a.view(torch.int16), c.view(torch.int16))
                                            for a, c in ((kp2, kp), (vp2, vp)))


def test_paged_tokens_without_a_place():
    """The padding of a batch (length 0), rows behind the last sequence, a sequence of more tokens than
    its length, a page index outside the pages and a place past the table."""
    page, hq, hkv, d, n = 16, 4, 2, 128, 64
    new, held = [2, 3, 4, 2, 2], [30, 0, 0, 20, 8]
    c = _paged_case(BF, new, held, page, hq, hkv, d, 77)
    q, k, v, pages, table, lengths, cut = c
    q, k, v = (torch.cat([x, x[:3]]) for x in (q, k, v))  # three rows behind the last sequence
    lengths = lengths.clone()
    lengths[1] = 0            # padding: its rows have no place
    lengths[2] = 3            # the first of its four tokens has position -1
    table[3, 1] = 1000        # outside the pages
    long = lengths.clone()
    long[4] = page * table.shape[1] + 9  # past the table
    freq = (500.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float()
    opts = dm.QkNormRopeOptions()
    kp, vp = (x.cuda() for x in pages)
    qo = dm.qk_norm_rope_paged(*_cuda(q, k, v), None, None, freq.cuda(), kp, vp, table.cuda(), long.cuda(),
                               cut.cuda(), opts).cpu()
    zero = torch.zeros(len(q), dtype=torch.bool)
    zero[2:5] = zero[5] = zero[-3:] = True
    assert not qo[zero].any() and (qo[~zero].abs().amax((1, 2)) > 0).all()
    wrote = ~torch.isnan(vp).flatten(2).any(-1).cpu().flatten()
    slots = [int(table[0, 1]) * page + 14, int(table[0, 1]) * page + 15]
    slots += [int(table[2, 0]) * page + x for x in range(3)]
    want = torch.zeros_like(wrote)
    want[slots] = True
    assert torch.equal(wrote, want)
    assert torch.equal(wrote, ~torch.isnan(kp).flatten(2).any(-1).cpu().flatten())
    # positions of the last sequence: far past its table, its queries as any position's
    p = [30, 31] + [0] * 3 + [0] + [0, 1, 2] + [20, 21] + [int(long[4]) - 2, int(long[4]) - 1] + [0] * 3
    want, bound = rc.forward(q, None, False, 1e-6, rc.turns(freq, p, n, d, False))
    rc.held("q", qo[~zero], want[~zero], bound[~zero])


def test_paged_past_four_gigabytes():
    """Rows in the last pages of pools of 5 GB."""
    page, hq, hkv, d, n = 16, 4, 2, 128, 64
    c = _paged_case(BF, [20, 1, 3], [7, 8, 0], page, hq, hkv, d, 6)
    q, k, v, pages, table, lengths, cut = c
    used, total = len(pages[0]), 5 * 2 ** 30 // (pages[0][0].numel() * 2)
    far = [torch.empty(total, *x.shape[1:], dtype=x.dtype, device="cuda") for x in pages]
    for x, y in zip(far, pages):
        x[-used:] = y.cuda()
    freq = (100.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float()
    opts = dm.QkNormRopeOptions()
    at = torch.where(table >= 0, table + (total - used), table)
    qo = dm.qk_norm_rope_paged(*_cuda(q, k, v), None, None, freq.cuda(), *far, at.cuda(), lengths.cuda(),
                               cut.cuda(), opts)
    _check_paged(c, page, opts, (None, None), freq, n, (qo, far[0][-used:], far[1][-used:]))


def test_paged_offsets_that_do_not_go_up():
    """Offsets and lengths are read on the GPU whatever they hold: no row outside is touched."""
    page, hq, hkv, d = 16, 2, 1, 64
    c = _paged_case(BF, [4, 4, 4], [4, 4, 4], page, hq, hkv, d, 3)
    q, k, v, pages, table, lengths, cut = c
    for bad in ([9, -5, 1 << 30, 2], [0, 8, 4, 12], [5, 5, 5, 5], [-9, 2, 3, -1]):
        kp, vp = (x.cuda() for x in pages)
        qo = dm.qk_norm_rope_paged(*_cuda(q, k, v), None, None, torch.zeros(0).cuda(), kp, vp, table.cuda(),
                                   torch.tensor([1 << 30, -7, 8], dtype=torch.int32).cuda(),
                                   torch.tensor(bad, dtype=torch.int32).cuda())
        assert torch.isfinite(qo).all()
        wrote = set(torch.nonzero(~torch.isnan(vp).flatten(1).all(1).cpu())[:, 0].tolist())
        assert wrote <= set(table[table >= 0].tolist())


def test_paged_pages_of_one_pool_as_views():
    """Keys and values of one pool [P, 2, page, Hkv, D], and heads ahead of the rows."""
    page, hq, hkv, d = 16, 4, 2, 128
    c = _paged_case(BF, [20, 1, 3], [7, 8, 0], page, hq, hkv, d, 31)
    q, k, v, pages, table, lengths, cut = c
    freq = torch.ones(64)
    opts = dm.QkNormRopeOptions()
    both = torch.stack(pages, 1).cuda()
    ahead = torch.stack(pages, 1).transpose(2, 3).contiguous().cuda()
    for kp, vp in ((both[:, 0], both[:, 1]), (ahead[:, 0].transpose(1, 2), ahead[:, 1].transpose(1, 2))):
        qo = dm.qk_norm_rope_paged(*_cuda(q, k, v), None, None, freq.cuda(), kp, vp, table.cuda(),
                                   lengths.cuda(), cut.cuda(), opts)
        _check_paged(c, page, opts, (None, None), freq, 64, (qo, kp, vp))


def test_on_another_stream_and_captured():
    """Python calls captured as they are (nothing is read back): each replay takes the lengths that the
    program has moved on, and equals the eager call's bits."""
    page, hq, hkv, d, n = 16, 8, 2, 128, 64
    c = _paged_case(BF, [1] * 6, [3, 15, 16, 40, 0, 7], page, hq, hkv, d, 12)
    q, k, v, pages, table, lengths, cut = c
    q, k, v, table, freq = _cuda(q, k, v, table, torch.rand(n))
    ln = lengths.cuda()
    kp, vp = (x.cuda() for x in pages)
    gq, gk = torch.randn_like(q)[None], torch.randn_like(k)[None]

    def step():
        a = dm.qk_norm_rope_paged(q, k, v, None, None, freq, kp, vp, table, ln)
        return (a,) + dm.qk_norm_rope_backward(q[None], k[None], None, None, freq, gq, gk)[:2]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for r in range(3):
        ln.copy_(lengths + (r % 2))  # (a sequence without the page for one more writes nothing)
        kp.fill_(float("nan")), vp.fill_(float("nan"))
        junk = torch.randn(1 << 20, device="cuda").sum()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*outs, kp, vp)]
        kp.fill_(float("nan")), vp.fill_(float("nan"))
        want = [*step(), kp, vp]
        for a, b in zip(got, want):
            assert torch.equal(torch.nan_to_num(a, nan=77.0), torch.nan_to_num(b, nan=77.0)), r
        del junk
