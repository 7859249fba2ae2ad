"""The attention of new tokens over a paged cache and its keys' weights where sizes, places and workspaces are
unusual, against 64 bits (chunk_cases.py, which derives the bounds)."""
import pytest
import torch

import dashmag_amd as dm
from chunk_cases import Chunks, held_lse
from dashmag_amd import ops
from rope_cases import held

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
MIXED = [(90, 400), (1, 700), (16, 130), (17, 130), (3, 9), (0, 12)]  # (of 4 heads a key head: 360 to 4 rows)


def _weigh(b, q, k, v, table, ln, cu, w):
    opts = dm.AttentionOptions(window=None if b.window is None else dm.Window(b.window, 0))
    return dm.attention_paged_with_weights(q, k, v, table, ln, w, cu, opts)


def _held(b, out, lse, w):
    want = b.want()
    held("out", out, *want["out"])
    held_lse("lse", lse, *want["lse"])
    held("weights", w, *want["weights"])


@pytest.mark.parametrize("dtype,d,window", [(BF, 128, None), (F16, 64, 60), (BF, 256, None), (F32, 64, None), (BF, 40, 33)])
def test_what_the_workspace_holds(monkeypatch, dtype, d, window):
    """Nothing of a call's workspace is read before the call has written it."""
    for seqs in (MIXED, [(1, x) for x in (900, 1, 0, 64, 333)], [(4, 800), (2, 31)]):
        b = Chunks(dtype, d, 2, 4, 16, seqs, seed=d, window=window, gaps=(1, 2))
        got = []
        for fill in (0, 255, 127):
            monkeypatch.setattr(ops, "_workspace",
                                lambda n, dev: torch.full((max(int(n), 1),), fill, dtype=torch.uint8, device=dev))
            w = b.weights.cuda()
            got.append((*_weigh(b, *b.cuda(), w), w))
        _held(b, *got[0])
        for other in got[1:]:
            assert all(torch.equal(x, y) for x, y in zip(got[0], other))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256)])
@pytest.mark.parametrize("single", [False, True])
def test_tables_too_wide_to_keep_scores(dtype, d, single):
    """The weights by another pass over the keys: the call could need more scores than are kept."""
    seqs = [(1, x) for x in (700, 64, 0, 1, 2100)] if single else MIXED
    for window in (None, 50):
        b = Chunks(dtype, d, 2, 8 if single else 4, 16, seqs, seed=d + 1, window=window, single=single)
        q, k, v, table, ln, cu = b.cuda()
        cols = 1 << 19 if single else 1 << 16
        wide = torch.full((len(seqs), cols), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        w = torch.full((len(seqs), cols * 16), 0.25, device="cuda")
        w[:, :b.weights.shape[1]] = b.weights.cuda()
        out, lse = _weigh(b, q, k, v, wide, ln, cu, w)
        _held(b, out, lse, w[:, :b.weights.shape[1]])
        assert (w[:, b.weights.shape[1]:] == 0.25).all()
        assert torch.equal(out, dm.attention_paged(q, k, v, wide, ln, cu, dm.AttentionOptions(
            window=None if window is None else dm.Window(window, 0))))


@pytest.mark.parametrize("dtype,d,single", [(BF, 64, False), (BF, 64, True), (F32, 64, False)])
def test_weights_past_32_bits(dtype, d, single):
    """Rows of 2^30 keys: the last one's weights begin at 2^31."""
    seqs = [(1, 90), (1, 40), (1, 700)] if single else [(40, 90), (1, 40), (60, 700)]
    b = Chunks(dtype, d, 1, 4, 16, seqs, seed=5, single=single)
    q, k, v, table, ln, cu = b.cuda()
    wide = torch.full((3, 1 << 26), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    w = torch.zeros(3, 1 << 30, device="cuda")
    n = b.weights.shape[1]
    w[:, :n] = b.weights.cuda()
    out, lse = _weigh(b, q, k, v, wide, ln, cu, w)
    _held(b, out, lse, w[:, :n])
    assert not w[:, n:n + 4096].any() and not w[:, -4096:].any()


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F32, 64)])
@pytest.mark.parametrize("least", [24, 33])
def test_pools_past_32_bits(dtype, d, least):
    """Pools that span 24 and 33 GB: offsets of more than 32 bits, and more than the 16-bit kernels' places take."""
    b = Chunks(dtype, d, 2, 4, 16, [(90, 130), (1, 60), (5, 40)], seed=7)
    q, k, v, *rest = b.cuda()
    each = 16 * 2 * d
    apart = ((least << 30) // k.element_size() // len(k) + 7) // 8 * 8
    buf = torch.empty((len(k) - 1) * apart + 2 * each, dtype=dtype, device="cuda")
    kf, vf = (buf.as_strided(x.shape, (apart, 2 * d, d, 1), i * each).copy_(x) for i, x in enumerate((k, v)))
    w = b.weights.cuda()
    _held(b, *_weigh(b, q, kf, vf, *rest, w), w)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 256), (F32, 64)])
def test_rows_at_the_tiles_edges(dtype, d):
    """Sequences of one row more and less than a narrow tile, the most rows that narrow ones take and a wide tile; keys
    around a step's and a worker's least."""
    for rep in (1, 4):
        seqs = [(n, x) for n in (31, 32, 33, 63, 64, 65, 127, 128, 129, 256, 257) for x in (n, n + 64)]
        _held_all(Chunks(dtype, d, 1, rep, 16, seqs, seed=rep))
    _held_all(Chunks(dtype, d, 1, 4, 16, [(16, x) for x in (31, 32, 33, 95, 96, 97, 511, 513)], seed=3))
    _held_all(Chunks(dtype, d, 1, 4, 16, [(40, x) for x in (63, 64, 65, 511, 512, 513, 1023, 1025)], seed=4))


def _held_all(b):
    w = b.weights.cuda()
    _held(b, *_weigh(b, *b.cuda(), w), w)


def test_two_streams_at_once():
    """Calls in flight together, and a captured one beside an eager one, have workspaces of their own."""
    two = [Chunks(BF, 128, 2, 4, 16, [(300, 2000), (1, 700)], seed=1), Chunks(BF, 128, 2, 4, 16, [(200, 900), (40, 3000)], seed=2)]
    args = [b.cuda() for b in two]
    ws = [[b.weights.cuda() for _ in range(4)] for b in two]
    streams = [torch.cuda.Stream() for _ in two]
    torch.cuda.synchronize()
    got = [[], []]
    for n in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_weigh(two[i], *args[i], ws[i][n]))
    torch.cuda.synchronize()
    for i, b in enumerate(two):
        for n in range(4):
            assert torch.equal(got[i][n][0], got[i][0][0]) and torch.equal(ws[i][n], ws[i][0])
        _held(b, *got[i][0], ws[i][0])
    graphs, outs = [], []
    w = [b.weights.cuda() for b in two]
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(_weigh(two[i], *args[i], w[i]))
        graphs.append(g)
    for _ in range(3):
        for i, b in enumerate(two):
            w[i].copy_(b.weights.cuda())
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = _weigh(two[0], *args[0], ws[0][1].copy_(two[0].weights))
        torch.cuda.synchronize()
        assert torch.equal(eager[0], got[0][0][0])
        for i in range(2):
            assert torch.equal(outs[i][0], got[i][0][0]) and torch.equal(outs[i][1], got[i][0][1])
            assert torch.equal(w[i], ws[i][0])


def test_the_same_sequence_twice():
    """Rows that hold the same pages get the same, and a pool may be both keys and values."""
    b = Chunks(BF, 128, 2, 4, 16, [(70, 300)], seed=3)
    q, k, v, table, ln, cu = b.cuda()
    two = torch.tensor([0, 70, 140], dtype=torch.int32).cuda()
    w = torch.zeros(2, b.weights.shape[1], device="cuda")
    out, lse = _weigh(b, torch.cat([q, q]), k, v, torch.cat([table] * 2), torch.cat([ln] * 2), two, w)
    want = b.want()
    for at in (slice(0, 70), slice(70, 140)):
        held("out", out[at], *want["out"])
        held_lse("lse", lse[at], *want["lse"])
    for x in w:
        held("weights", (x + b.weights[0].cuda())[None], *want["weights"])
    same = dm.attention_paged(q, k, k, table, ln, cu)
    assert torch.equal(same, dm.attention_paged(q, k, k.clone(), table, ln, cu))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 256), (F16, 64), (F32, 64), (BF, 40)])
def test_the_weights_of_a_query_of_nan(dtype, d):
    """NaN in a token's query reaches the weights of the keys that it sees and no other's."""
    for seqs, tok, left in (([(80, 200), (1, 100)], 17, None), ([(5, 200), (1, 100)], 2, None), ([(5, 200), (70, 100)], 3, 40),
                            ([(90, 200), (2, 100)], 60, 30), ([(1, 90), (1, 64)], 0, 20)):
        b = Chunks(dtype, d, 2, 2, 16, seqs, seed=9, window=left)
        q, *rest = b.cuda()
        q[tok, 1] = float("nan")
        w = b.weights.cuda()
        _weigh(b, q, *rest, w)
        pos = seqs[0][1] - seqs[0][0] + tok
        seen = torch.zeros(b.weights.shape, dtype=torch.bool)
        seen[0, 0 if left is None else max(0, pos - left):pos + 1] = True
        assert torch.equal(torch.isnan(w).cpu(), seen)
        want, bound = b.want()["weights"]
        held("others", w[~seen.cuda()], want[~seen], bound[~seen])


@pytest.mark.parametrize("dtype,d,rep,seqs,window", [
    (BF, 128, 4, [(1, 20000)], None), (BF, 128, 4, [(8, 16000), (1, 50)], None), (F16, 64, 8, [(5, 30000)], 25000),
    (BF, 256, 2, [(3, 9000)], None), (F32, 64, 4, [(6, 9000)], None), (BF, 36, 3, [(2, 9000)], None),
    (BF, 128, 1, [(49, 31000)], None), (BF, 128, 40, [(2, 26000)], None), (BF, 33, 1, [(30, 5000)], None)])
def test_tiles_of_many_pieces(dtype, d, rep, seqs, window):
    """One sequence's keys over all workers: the pieces of its rows are joined by many."""
    _held_all(Chunks(dtype, d, 1, rep, 16, seqs, seed=rep, window=window))
