"""The attention of new tokens over a paged cache, its log-sum-exps and the weights that the cached keys
get, against 64 bits (chunk_cases.py, which derives the bounds). Every cache row that no token sees holds NaN."""
import pytest
import torch

import dashmag_amd as dm
from dashmag_amd import _lib
from chunk_cases import Chunks, held_lse
from rope_cases import held

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# (new tokens, keys with them) of each sequence, window, tokens outside
SHAPES = {
    "one": ([(40, 300)], None, (0, 0)),
    "whole prompt": ([(257, 257)], None, (0, 0)),
    "single key": ([(1, 1)], None, (0, 0)),
    "ragged": ([(3, 100), (0, 50), (70, 71), (1, 1), (129, 700), (1, 640), (0, 0), (17, 17)], None, (0, 0)),
    "outside": ([(5, 64), (31, 33)], None, (3, 6)),
    "below zero": ([(40, 25), (3, 0), (2, 1)], None, (0, 0)),
    "window": ([(90, 400), (300, 333), (1, 90), (2, 40)], 50, (0, 0)),
    "window of one": ([(40, 90), (1, 33)], 0, (0, 0)),
    "tokens": ([(1, 700), (1, 1), (1, 64), (1, 333), (1, 2100)], None, (0, 0)),
    "drafts": ([(5, 900), (4, 31), (6, 6), (2, 1500)], None, (1, 0)),
    "long": ([(9, 9000), (1, 7000)], None, (0, 0)),
    "nothing": ([(0, 10), (0, 0)], None, (2, 1)),
}
FORMS = [(BF, 128, 2, 4, 16), (F16, 64, 1, 8, 32), (BF, 256, 2, 4, 16), (BF, 64, 2, 1, 64), (F16, 128, 1, 2, 7),
         (BF, 128, 1, 3, 16), (BF, 128, 1, 40, 48), (F16, 256, 1, 16, 1), (F32, 128, 2, 2, 16), (BF, 96, 1, 2, 16),
         (BF, 64, 1, 300, 16), (F32, 36, 1, 5, 3), (F32, 64, 4, 1, 7), (F32, 256, 1, 2, 16), (F16, 33, 2, 1, 5)]


def _all(b, opts=None, scale=None):
    """The three entry points: alike to the bit, and held to the bounds."""
    q, k, v, table, ln, cu = b.cuda()
    opts = opts or dm.AttentionOptions(window=None if b.window is None else dm.Window(b.window, 0), scale=scale)
    w = b.weights.cuda()
    out, lse = dm.attention_paged_with_weights(q, k, v, table, ln, w, cu, opts)
    o2, l2 = dm.attention_paged_with_lse(q, k, v, table, ln, cu, opts)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    assert torch.equal(out, dm.attention_paged(q, k, v, table, ln, cu, opts))
    w2 = b.weights.cuda()
    dm.attention_paged_with_weights(q, k, v, table, ln, w2, cu, opts)
    assert torch.equal(w, w2)  # nothing depends on the order of the workgroups
    want = b.want(scale)
    held("out", out, *want["out"])
    held_lse("lse", lse, *want["lse"])
    held("weights", w, *want["weights"])
    return out


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("shape", SHAPES)
def test_chunks(shape, form):
    dtype, d, hkv, rep, page = form
    seqs, window, gaps = SHAPES[shape]
    if rep > 32:  # (as many rows as the others have)
        seqs = [(min(n, 20), x) for n, x in seqs]
    print(f"chunks {shape} {dtype} D={d} Hkv={hkv} rep={rep} page={page}", flush=True)
    _all(Chunks(dtype, d, hkv, rep, page, seqs, seed=d + rep, window=window, gaps=gaps))


@pytest.mark.parametrize("dtype,d,page", [(BF, 128, 16), (F16, 64, 32), (BF, 256, 16), (F32, 64, 16)])
def test_one_token_each_without_offsets(dtype, d, page):
    """The paged decode's calls: the same results, up to its bounds."""
    seqs = [(1, x) for x in (1, 700, 16, 64, 0, 2049, 333, 900, 31)]
    for window in (None, 100):
        b = Chunks(dtype, d, 2, 4, page, seqs, seed=d, window=window, single=True)
        out = _all(b)
        q, k, v, table, ln, _ = b.cuda()
        opts = dm.AttentionOptions(window=None if window is None else dm.Window(window, 0))
        want, bound = b.want()["out"]
        held("paged decode", dm.attention_decode_paged(q, k.nan_to_num(0.0), v.nan_to_num(0.0), table, ln, opts), want,
             bound + 1e-3 * want.abs())
        assert not out[4].any()


def test_many_sequences():
    """More sequences than a workgroup has threads, some without tokens."""
    gen = torch.Generator().manual_seed(3)
    for count in (513, 1300):
        new = torch.randint(0, 4, (count,), generator=gen).tolist()
        seqs = [(n, n + int(x)) for n, x in zip(new, torch.randint(0, 90, (count,), generator=gen))]
        print(f"{count} sequences", flush=True)
        _all(Chunks(BF, 64, 1, 2, 16, seqs, seed=count, gaps=(1, 2)))
        _all(Chunks(F32, 64, 1, 1, 16, seqs, seed=count, gaps=(1, 2)))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256), (F32, 128)])
def test_a_long_chunk(dtype, d):
    """Tiles that many workers share, next to single tokens."""
    _all(Chunks(dtype, d, 2, 4, 16, [(700, 3000), (1, 2500), (333, 333), (1, 40)], seed=1))
    _all(Chunks(dtype, d, 1, 2, 16, [(900, 4000), (2, 600)], seed=2, window=1100))


@pytest.mark.parametrize("scale", [0.31, -0.2, 0.0])
def test_scales(scale):
    for dtype, d in ((BF, 128), (F32, 64), (F16, 256)):
        _all(Chunks(dtype, d, 2, 2, 16, [(60, 300), (1, 500), (200, 260)], seed=8), scale=scale)


def test_large_scores():
    """Scores hundreds apart: the running reference moves, and keys far below it count as nothing."""
    for dtype in (BF, F16, F32):
        _all(Chunks(dtype, 128, 1, 4, 16, [(130, 900), (1, 700), (3, 1400)], seed=8, scale=30.0))


def test_views():
    """Queries of a wider row, keys and values of one pool, heads ahead of the page's rows, values laid out
    otherwise than keys, weights of a wider array."""
    b = Chunks(BF, 128, 2, 4, 16, [(90, 300), (1, 500), (3, 40)], seed=3)
    q, k, v, *rest = b.cuda()
    want = dm.attention_paged(q, k, v, *rest)
    wide = torch.cat([q, q, q], 1)[:, 8:16]
    both = torch.stack([k, v], 1)
    ahead = torch.stack([k, v], 1).transpose(2, 3).contiguous()
    assert torch.equal(dm.attention_paged(wide, both[:, 0], both[:, 1], *rest), want)
    assert torch.equal(dm.attention_paged(q, ahead[:, 0].transpose(1, 2), ahead[:, 1].transpose(1, 2), *rest), want)
    held("apart", dm.attention_paged(q, k, ahead[:, 1].transpose(1, 2), *rest), *b.want()["out"])
    odd = torch.empty(q.numel() + 1, dtype=BF, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(dm.attention_paged(odd, k, v, *rest), want)
    w = torch.full((3, b.weights.shape[1] + 5), -7.0, device="cuda")
    w[:, 2:-3] = b.weights.cuda()
    dm.attention_paged_with_weights(q, k, v, *rest[:2], w[:, 2:-3], rest[2])
    held("weights", w[:, 2:-3], *b.want()["weights"])
    assert (w[:, :2] == -7).all() and (w[:, -3:] == -7).all()


@pytest.mark.parametrize("dtype,d,page,n", [(BF, 128, 16, 70), (F16, 64, 16, 300), (BF, 256, 32, 9), (F32, 64, 16, 40),
                                            (BF, 128, 16, 400), (BF, 64, 16, 1)])
def test_what_a_token_does_not_see_stays_out_of_it(dtype, d, page, n):
    """NaN and infinities in one key: the tokens in front of it, and those whose window is past it, are what they
    are without it; the others are not finite."""
    for window, length, bad in ((None, 500, 500 - n // 2 - 1), (100, 640, 640 - n // 2 - 60)):
        b = Chunks(dtype, d, 1, 4, page, [(n, length), (2, 90)], seed=d, window=window)
        opts = dm.AttentionOptions(window=None if window is None else dm.Window(window, 0))
        want, bound = b.want()["out"]
        q, k, v, table, ln, cu = b.cuda()
        pg, row = int(table[0, bad // page]), bad % page
        pos = torch.arange(length - n, length)
        sees = (pos >= bad) & (torch.tensor(True) if window is None else pos - window <= bad)
        sees = torch.cat([sees, torch.zeros(2, dtype=torch.bool)])
        for x in (float("nan"), float("inf"), -float("inf")):
            v2, k2 = v.clone(), k.clone()
            v2[pg, row, 0, 3] = x
            if x != x:
                k2[pg, row, 0, 5] = x
            w = b.weights.cuda()
            out, lse = dm.attention_paged_with_weights(q, k2, v2, table, ln, w, cu, opts)
            assert not torch.isfinite(out[sees.cuda()][:, :, 3]).any()
            held("others", out[~sees.cuda()], want[~sees], bound[~sees])
            if x != x:
                assert torch.isnan(lse[sees.cuda()]).all()
                gone = torch.isnan(w[0]).cpu()
                first = 0 if window is None else max(0, bad - window)
                last = int(pos[sees[:n]].max()) if sees.any() else -1
                if sees.any():
                    assert gone[max(first, int(pos[sees[:n]].min()) - (window or 10 ** 9)):last + 1].all()
                assert not gone[last + 1:].any() and not torch.isnan(w[1]).any()
            else:
                held("weights", w, *b.want()["weights"])


def test_a_query_of_nan_and_scores_of_infinity():
    """A token's NaN stays its own; a key whose score is -inf has no weight."""
    for dtype in (BF, F32):
        b = Chunks(dtype, 64, 1, 2, 16, [(80, 200), (1, 100)], seed=5)
        q, k, v, table, ln, cu = b.cuda()
        want, bound = b.want()["out"]
        q2 = q.clone()
        q2[17] = float("nan")
        out, lse = dm.attention_paged_with_lse(q2, k, v, table, ln, cu)
        others = torch.arange(81) != 17
        assert torch.isnan(out[17]).all() and torch.isnan(lse[17]).all()
        held("others", out[others.cuda()], want[others], bound[others])
        big = 3e38
        q3, k3 = torch.zeros_like(q), torch.zeros_like(k)
        q3[:, :, 0] = big
        k3[int(table[1, 0]), :, :, 0] = -big  # the first page of the second sequence: scores of -inf
        out, lse = dm.attention_paged_with_lse(q3, k3, v, table, ln, cu)
        mean = b.keys[1][1][16:].double().mean(0)  # [1, D]
        half = torch.finfo(dtype).eps
        off = (out[80].cpu().double() - mean).abs()
        assert (off <= half * (1 + b.keys[1][1][16:].double().abs().mean(0))).all()
        assert (lse[80].cpu().double() - torch.tensor(84.0).double().log()).abs().max() <= 1e-5


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F32, 64), (BF, 40)])
def test_offsets_lengths_and_pages_that_are_wrong(dtype, d):
    """Whatever the device arrays hold nothing outside is touched: offsets that do not go up leave no token in a
    sequence, lengths count as between 0 and the table's keys, pages outside read as zeros."""
    b = Chunks(dtype, d, 2, 2, 16, [(40, 70), (1, 90), (0, 16), (200, 210)], seed=4)
    q, k, v, table, ln, cu = b.cuda()
    for bad in ([0, 41, 40, 41, 241], [-1, 40, 41, 41, 241], [0, 40, 41, 41, 242], [5, 4, 3, 2, 1], [1 << 30] * 5):
        w = b.weights.cuda()
        out, lse = dm.attention_paged_with_weights(q, k, v, table, ln, w, torch.tensor(bad, dtype=torch.int32).cuda())
        assert not out.any() and (lse == -torch.inf).all() and torch.equal(w, b.weights.cuda())
    kz, vz = k.nan_to_num(0.0), v.nan_to_num(0.0)
    cap = table.shape[1] * 16
    many = torch.tensor([-5, cap + 77, 0, 2 ** 31 - 1], dtype=torch.int32).cuda()
    t2 = torch.where(table < 0, 0, table)
    assert torch.equal(dm.attention_paged(q, kz, vz, t2, many, cu),
                       dm.attention_paged(q, kz, vz, t2, many.clamp(0, cap), cu))
    t3 = table.clone()
    t3[0, 1], t3[1, 0], t3[3, 2] = -1, k.shape[0], 2 ** 31 - 1
    k4 = torch.cat([kz, torch.zeros_like(kz[:1])])
    v4 = torch.cat([vz, torch.zeros_like(vz[:1])])
    t4 = t3.clone()
    t4[0, 1] = t4[1, 0] = t4[3, 2] = k.shape[0]
    assert torch.equal(dm.attention_paged(q, kz, vz, t3, ln, cu), dm.attention_paged(q, k4, v4, t4, ln, cu))


def test_no_pages_and_no_columns():
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    none = torch.zeros(0, 16, 2, 64, dtype=BF, device="cuda")
    ln = torch.tensor([5, 0, 20], dtype=torch.int32).cuda()
    w = torch.zeros(3, 32, device="cuda")
    out, lse = dm.attention_paged_with_weights(q, none, none, torch.zeros(3, 2, dtype=torch.int32), ln, w)
    assert not out.any() and torch.allclose(lse[0], torch.tensor(5.0, device="cuda").log(), atol=1e-6)
    assert (lse[1] == -torch.inf).all() and torch.allclose(w[0, :5], torch.full((5,), 4 / 5, device="cuda"))
    assert not w[1].any() and not w[2, 20:].any()
    out, lse = dm.attention_paged_with_lse(q, none, none, torch.zeros(3, 0, dtype=torch.int32), ln)
    assert not out.any() and (lse == -torch.inf).all()
    k = torch.zeros(4, 16, 2, 64, dtype=BF, device="cuda")
    out, lse = dm.attention_paged_with_lse(q, k, k, torch.zeros(0, 2, dtype=torch.int32), [], [1])
    assert not out.any() and (lse == -torch.inf).all()
    assert dm.attention_paged(q[:0], k, k, torch.zeros(0, 2, dtype=torch.int32), []).shape == (0, 4, 64)


def test_streams_and_probes():
    """On a stream of the caller's own; the launches are counted."""
    b = Chunks(BF, 128, 2, 4, 16, [(90, 300), (1, 500)], seed=3)
    args = b.cuda()
    want = dm.attention_paged(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    _lib.probe_reset()
    with torch.cuda.stream(side):
        out = dm.attention_paged(*args)
        dm.attention_paged_with_weights(*args[:5], b.weights.cuda(), args[5])
    side.synchronize()
    assert torch.equal(out, want)
    counts = _lib.probe_counts()
    assert counts["attn_paged"] == 2 and counts["attn_weights"] == 1


def test_graph():
    """A captured call follows lengths, offsets and tables that move on, and adds to its weights at each replay."""
    a = Chunks(BF, 128, 2, 4, 16, [(60, 300), (1, 200), (1, 640)], seed=1, extra=4)
    c = Chunks(BF, 128, 2, 4, 16, [(1, 333), (60, 64), (1, 290)], seed=2, extra=4)
    cols = max(a.table.shape[1], c.table.shape[1])
    pages = max(len(a.k), len(c.k))

    def grown(b):
        t = torch.full((3, cols), -1, dtype=torch.int32)
        t[:, :b.table.shape[1]] = b.table
        kv = [torch.cat([x, x.new_zeros(pages - len(x), *x.shape[1:])]) for x in (b.k, b.v)]
        return [x.cuda() for x in (b.q, *kv, t, b.lengths, b.cu)]
    state, other = grown(a), grown(c)
    first = [x.clone() for x in state]
    w = torch.zeros(3, cols * 16, device="cuda")
    run = lambda: dm.attention_paged_with_weights(*state[:5], w, state[5])  # noqa: E731
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out, lse = run()
    for now in (other, first, other, other):
        for x, y in zip(state, now):
            x.copy_(y)
        w.fill_(0.5)
        g.replay()
        torch.cuda.synchronize()
        want_w = torch.full_like(w, 0.5)
        want, want_l = dm.attention_paged_with_weights(*now[:5], want_w, now[5])
        assert torch.equal(out, want) and torch.equal(lse, want_l) and torch.equal(w, want_w)
