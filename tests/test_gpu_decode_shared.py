"""The paged decode of a batch whose rows share prefixes, against the 64-bit softmax of each row over
its own keys (shared_cases.py, which derives the bounds). Every cache row that no query sees holds NaN."""
import pytest
import torch

import dashmag_amd as dm
from dashmag_amd import _lib
from rope_cases import held
from shared_cases import Batch

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# groups (first row, lengths, prefix), rows of no group, rows, window
SHAPES = {
    "one": ([(0, [700, 650, 1400, 641], 640)], {}, 4, None),
    "odd prefix": ([(0, [1000, 998, 1030], 997)], {}, 3, None),
    "ragged": ([(1, [300], 256), (2, [90, 700, 91, 95, 400, 89], 89), (8, [2000, 1999], 1990)],
               {0: 33, 10: 17, 11: 0}, 13, None),
    "short members": ([(0, [0, 5, 640, 16, 2000, 1, 0, 639], 1024)], {}, 8, None),
    "no prefix": ([(0, [40, 0, 300], 0)], {3: 1}, 4, None),
    "nothing": ([(0, [0, 0], 64)], {}, 2, None),
    "no group": ([], {0: 100, 1: 1}, 2, None),
    "window": ([(0, [900, 1500, 0, 3000, 850], 800)], {5: 1200}, 6, 500),
    "window in the prefix": ([(0, [2100, 2300, 2047, 2200], 2000)], {}, 4, 333),
    "window of one": ([(0, [65, 64], 64)], {}, 2, 0),
    "many rows": ([(0, [513 + 7 * (i % 5) for i in range(70)], 512)], {}, 70, None),
    "two large groups": ([(0, [300 + i for i in range(37)], 290), (37, [1500 + 3 * i for i in range(66)], 1481)],
                         {}, 104, None),
    "long": ([(0, [9000, 9111], 8990)], {}, 2, None),
}


def _run(b, opts=None):
    return dm.attention_decode_shared(*b.cuda()[:4], *b.cuda()[4:], opts)


@pytest.mark.parametrize("dtype,d,hkv,rep,page", [
    (BF, 128, 2, 4, 16), (F16, 64, 1, 8, 32), (BF, 256, 2, 4, 16), (BF, 64, 2, 1, 64), (F16, 128, 1, 2, 16),
    (BF, 128, 1, 3, 16), (BF, 128, 1, 40, 48), (F16, 256, 1, 16, 16), (F32, 128, 2, 2, 16), (BF, 96, 1, 2, 16),
    (BF, 128, 2, 2, 7), (F32, 36, 1, 5, 3)], ids=str)
@pytest.mark.parametrize("shape", SHAPES)
def test_shared(shape, dtype, d, hkv, rep, page):
    groups, lone, rows, window = SHAPES[shape]
    b = Batch(dtype, d, hkv, rep, page, groups, lone, rows, seed=d + rep, window=window)
    print(f"shared {shape} {dtype} D={d} Hkv={hkv} rep={rep} page={page}", flush=True)
    opts = dm.AttentionOptions(window=None if window is None else dm.Window(window, 0))
    out = _run(b, opts)
    assert torch.equal(out, _run(b, opts))  # nothing depends on the order of the workgroups
    held("out", out, *b.want())


def test_without_groups_and_with_bad_ones():
    """Groups that do not go up within the batch share nothing: the results are right all the same."""
    groups, lone, rows, _ = SHAPES["ragged"]
    b = Batch(BF, 128, 2, 4, 16, groups, lone, rows, seed=2)
    q, k, v, table, ln, cu, pl = b.cuda()
    want = b.want()
    n = len(pl)
    for bad in ([3] * n + [1], [-1] + [2] * n, [0] * n + [rows + 1], list(range(n, -1, -1)), [1 << 30] * (n + 1)):
        at = torch.tensor(bad, dtype=torch.int32).cuda()
        held("bad groups", dm.attention_decode_shared(q, k, v, table, ln, at, pl), *want)
    none = torch.zeros(0, dtype=torch.int32).cuda()
    held("no groups", dm.attention_decode_shared(q, k, v, table, ln, none.new_zeros(1), none), *want)
    held("negative prefixes", dm.attention_decode_shared(q, k, v, table, ln, cu, -pl - 1), *want)
    held("paged", dm.attention_decode_paged(q, k, v, table, ln), *want)


def test_scale_and_no_lengths():
    b = Batch(BF, 128, 2, 4, 16, [(0, [640, 640, 640], 320)], {}, 3, seed=8)
    q, k, v, table, ln, cu, pl = b.cuda()
    table = table[:, :40].contiguous()
    out = dm.attention_decode_shared(q, k, v, table, None, cu, pl, dm.AttentionOptions(scale=0.31))
    held("out", out, *b.want(0.31))


def test_large_scores():
    """Scores hundreds apart: the running reference moves, and keys far below it count as nothing."""
    for dtype in (BF, F16, F32):
        b = Batch(dtype, 128, 1, 4, 16, [(0, [900, 700, 1400], 640)], {}, 3, seed=8, scale=30.0)
        held("out", _run(b), *b.want())


def test_views():
    """Queries of a wider row, keys and values of one pool, heads ahead of the page's rows."""
    groups, lone, rows, _ = SHAPES["ragged"]
    b = Batch(BF, 128, 2, 4, 16, groups, lone, rows, seed=3)
    q, k, v, *rest = b.cuda()
    want = _run(b)
    wide = torch.cat([q, q, q], 1)[:, 8:16]
    both = torch.stack([k, v], 1)
    ahead = torch.stack([k, v], 1).transpose(2, 3).contiguous()
    assert torch.equal(dm.attention_decode_shared(wide, both[:, 0], both[:, 1], *rest), want)
    assert torch.equal(dm.attention_decode_shared(q, ahead[:, 0].transpose(1, 2), ahead[:, 1].transpose(1, 2),
                                                  *rest), want)


@pytest.mark.parametrize("dtype,d,page", [(BF, 128, 16), (F16, 64, 16), (BF, 256, 32), (F32, 64, 16)])
def test_what_a_row_does_not_see_stays_out_of_it(dtype, d, page):
    """A prefix key that holds NaN and infinities, seen by the longer members alone: the shorter ones' and
    the windowed ones' results are what they are without it."""
    for window, lens, bad in ((None, [300, 520, 299, 305, 0], 301), (100, [600, 640, 610, 420], 330)):
        b = Batch(dtype, d, 1, 4, page, [(0, lens, 512)], {}, len(lens), seed=d, window=window)
        opts = dm.AttentionOptions(window=None if window is None else dm.Window(window, 0))
        want, bound = b.want()
        q, k, v, table, *rest = b.cuda()
        pg, row = int(table[1 if window is None else 3, bad // page]), bad % page
        sees = [bool(n > bad and (window is None or n - 1 - window <= bad)) for n in lens]
        assert any(sees) and not all(sees)
        for x in (float("nan"), float("inf"), -float("inf")):
            v[pg, row, 0, 3] = x
            k2 = k.clone()
            if x != x:
                k2[pg, row, 0, 5] = x
            out = dm.attention_decode_shared(q, k2, v, table, *rest, opts)
            for r, s in enumerate(sees):
                if s:
                    assert not torch.isfinite(out[r, :, 3]).any()
                else:
                    held(f"row {r}", out[r], want[r], bound[r])


@pytest.mark.parametrize("dtype,d,window", [(BF, 128, None), (F16, 64, 100), (BF, 256, None), (BF, 128, 40)])
def test_what_a_row_of_many_does_not_see_stays_out_of_it(dtype, d, window):
    """The same in a group of many rows, whose prefix is swept by all of them together."""
    lens = [300 + 7 * (i % 30) for i in range(40)]
    b = Batch(dtype, d, 1, 4, 16, [(0, lens, 480)], {}, len(lens), seed=d, window=window)
    opts = dm.AttentionOptions(window=None if window is None else dm.Window(window, 0))
    bad = 371
    want, bound = b.want()
    q, k, v, table, *rest = b.cuda()
    sees = [bool(n > bad and (window is None or n - 1 - window <= bad)) for n in lens]
    assert any(sees) and not all(sees)
    pg, row = int(table[lens.index(max(lens)), bad // 16]), bad % 16
    for x in (float("nan"), float("inf"), -float("inf")):
        v[pg, row, 0, 3] = x
        if x != x:
            k[pg, row, 0, 5] = x
        out = dm.attention_decode_shared(q, k, v, table, *rest, opts)
        if x != x:
            k[pg, row, 0, 5] = 0.5
        for r, s in enumerate(sees):
            if s:
                assert not torch.isfinite(out[r, :, 3]).any()
            else:
                held(f"row {r}", out[r], want[r], bound[r])


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256), (F32, 64)])
@pytest.mark.parametrize("rows", [3, 60])
def test_a_query_that_is_nan_gives_nan(dtype, d, rows):
    """In its own row and head, in groups of few rows and of many; the others are what they were."""
    b = Batch(dtype, d, 1, 4, 16, [(0, [600 + i for i in range(rows)], 590)], {}, rows, seed=4)
    want, bound = b.want()
    b.q[1, 2, 7] = float("nan")
    out = _run(b)
    assert torch.isnan(out[1, 2]).all()
    keep = torch.ones(out.shape[:2], dtype=torch.bool)
    keep[1, 2] = False
    held("others", out[keep.cuda()], want[keep], bound[keep])


@pytest.mark.parametrize("scale", [0.0, -0.2])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256), (F32, 64)])
@pytest.mark.parametrize("shape", ["ragged", "many rows", "two large groups"])
def test_scales_of_zero_and_below(shape, dtype, d, scale):
    groups, lone, rows, _ = SHAPES[shape]
    b = Batch(dtype, d, 1, 4, 16, groups, lone, rows, seed=6)
    held("out", _run(b, dm.AttentionOptions(scale=scale)), *b.want(scale))


@pytest.mark.parametrize("rows", [2, 40])
def test_pages_past_four_gigabytes(rows):
    """The last pages of a pool of 5 GB are the ones that are read."""
    b = Batch(BF, 128, 2, 4, 16, [(0, [200 + i for i in range(rows)], 180)], {}, rows, seed=9)
    q, k, v, table, *rest = b.cuda()
    n, pages = len(k), 5 * 2 ** 30 // (k[0].numel() * 2)
    far = [torch.empty(pages, *k.shape[1:], dtype=BF, device="cuda") for _ in range(2)]
    far[0][-n:], far[1][-n:] = k, v
    for pool in far:
        pool[:1].fill_(float("nan"))
    table = torch.where(table >= 0, table + (pages - n), table)
    held("out", dm.attention_decode_shared(q, *far, table, *rest), *b.want())


def test_pages_outside_read_as_zeros():
    """A page index outside the pages is a page of zeros, in the prefix and behind it."""
    b = Batch(BF, 128, 2, 4, 16, [(0, [200, 230], 160)], {}, 2, seed=5)
    q, k, v, table, *rest = b.cuda()
    table[0, 3], table[1, 3], table[0, 11] = 1 << 20, 1 << 20, -7
    for r, pages in ((0, (3, 11)), (1, (3,))):
        for c in pages:
            for x in b.keys[r][:2]:
                x[16 * c:16 * c + 16] = 0
    held("out", dm.attention_decode_shared(q, k, v, table, *rest), *b.want())


def test_captured():
    """A captured call of the mirror (nothing is read back) takes the lengths, groups and prefixes that the
    program moves on between replays, and gives the eager call's bits."""
    shapes = [SHAPES[x][:3] for x in ("ragged", "ragged")]
    b = Batch(BF, 128, 2, 4, 16, *shapes[0], seed=2)
    q, k, v, table, ln, cu, pl = b.cuda()
    call = lambda: dm.attention_decode_shared(q, k, v, table, ln, cu, pl)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for r in range(4):
        if r == 2:
            pl //= 2
        if r == 3:
            cu.zero_()
        out.fill_(7.0)
        junk = torch.randn(1 << 20, device="cuda").sum()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call()), r
        held(f"replay {r}", got, *b.want())
        del junk


def test_two_streams_at_once():
    """Two calls in flight on streams of their own have workspaces of their own."""
    bs = [Batch(BF, 128, 2, 4, 16, *SHAPES[x][:3], seed=i) for i, x in enumerate(("ragged", "two large groups"))]
    args = [b.cuda() for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(dm.attention_decode_shared(*args[i]))
    torch.cuda.synchronize()
    for b, got in zip(bs, outs):
        for x in got:
            held("out", x, *b.want())


def test_every_call_launches_its_kernels():
    b = Batch(BF, 128, 2, 4, 16, *SHAPES["one"][:3], seed=1)
    _lib.probe_reset()
    _run(b)
    assert _lib.probe_counts()["decode_shared"] == 1
