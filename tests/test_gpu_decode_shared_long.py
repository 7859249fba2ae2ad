"""The decode over shared prefixes on its long paths and in groups of many rows, against the 64-bit
softmax of each row (shared_cases.py): ranges of keys past what a kernel looks up at once, the checks of
groups, pages, views and captured calls in groups of many rows, odd widths, scores of minus infinity,
values that are not finite, long sums.

A call's ranges follow from the number of its tiles, so each long batch has enough short groups or rows
beside the long one that its keys are one range."""
import pytest
import torch

import dashmag_amd as dm
from rope_cases import held
from shared_cases import U, Batch

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _options(window):
    return dm.AttentionOptions(window=None if window is None else dm.Window(window, 0))


def _checked(b, window=None):
    out = dm.attention_decode_shared(*b.cuda(), _options(window))
    assert torch.equal(out, dm.attention_decode_shared(*b.cuda(), _options(window)))
    held("out", out, *b.want())


def _beside(long, groups, members):
    """The group ``long`` and short ones of ``members`` rows behind it."""
    n = len(long[1])
    return [long] + [(n + members * i, [5 + (i + j) % 13 for j in range(members)], 4) for i in range(groups)]


# 120 (at D = 256: 136) tiles and one range of 16700 keys: 261 tiles of 64 keys, two rounds of the 128 whose
# pages a workgroup holds. With the window a range of 14 tiles fewer that begins inside a page.
@pytest.mark.parametrize("window", [None, 15800])
@pytest.mark.parametrize("dtype,d,hkv,short", [(BF, 128, 8, 12), (F16, 64, 8, 12), (BF, 256, 4, 24)], ids=str)
def test_long_prefixes_of_groups_of_many_rows(dtype, d, hkv, short, window):
    groups = _beside((0, [16750, 16701, 9001], 16700), short, 3)
    b = Batch(dtype, d, hkv, 16, 16, groups, {}, 3 + 3 * short, seed=d, window=window)
    _checked(b, window)


# 124 tiles and one range of 9000 keys: four wavefronts of 2250, whose pages are looked up for 1024 at a time.
@pytest.mark.parametrize("window", [None, 8000])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256)], ids=str)
def test_long_prefixes_of_groups_of_few_rows(dtype, d, window):
    groups = _beside((0, [9040, 9001], 9000), 25, 2)
    b = Batch(dtype, d, 4, 4, 16, groups, {}, 52, seed=d, window=window)
    _checked(b, window)


# 1040 tiles of own keys, so one range a row, a wavefront's: 5000 and 2049 keys. As rows of no group, and
# (many) beside a group of many rows.
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256)], ids=str)
def test_long_own_keys(dtype, d, many):
    lone = {r: r % 4 for r in range(80 if many else 0, 260)}
    lone[100], lone[259] = 5000, 2049
    groups = [(0, [40 + r % 5 for r in range(80)], 37)] if many else []
    b = Batch(dtype, d, 4, 4, 16, groups, lone, 260, seed=d)
    _checked(b)


@pytest.mark.parametrize("dtype,d,hkv,rep,page", [(F32, 7, 2, 3, 5), (BF, 50, 1, 2, 16), (F16, 249, 1, 40, 16), (BF, 1, 2, 2, 16)],
                         ids=str)
def test_widths_that_are_no_multiple_of_four(dtype, d, hkv, rep, page):
    groups = [(1, [300], 256), (2, [90, 700, 91, 95, 400, 89], 89), (8, [2000, 1999], 1990)]
    _checked(Batch(dtype, d, hkv, rep, page, groups, {0: 33, 10: 17, 11: 0}, 13, seed=d))


def test_groups_of_many_rows_with_bad_groups():
    """Groups that do not go up within the batch share nothing, in a call that is planned for many rows."""
    rows = 70
    b = Batch(BF, 128, 2, 4, 16, [(0, [513 + 7 * (i % 5) for i in range(rows)], 512)], {}, rows, seed=2)
    q, k, v, table, ln, cu, pl = b.cuda()
    want = b.want()
    for bad in ([3, 1], [-1, 2], [0, rows + 1], [rows, 0], [1 << 30, 1 << 30]):
        at = torch.tensor(bad, dtype=torch.int32).cuda()
        held(f"groups {bad}", dm.attention_decode_shared(q, k, v, table, ln, at, pl), *want)
    held("negative prefix", dm.attention_decode_shared(q, k, v, table, ln, cu, -pl), *want)
    held("a longer prefix than the table", dm.attention_decode_shared(q, k, v, table[:1].expand(rows, -1), ln[:1].expand(rows),
                                                                      cu, pl + (1 << 30))[:1], want[0][:1], want[1][:1])


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256)], ids=str)
def test_groups_of_many_rows_with_pages_outside(dtype, d):
    """A page index outside the pages is a page of zeros, in the prefix of many rows and behind it."""
    rows = 44
    b = Batch(dtype, d, 2, 4, 16, [(0, [600 + i for i in range(rows)], 592)], {}, rows, seed=5)
    q, k, v, table, *rest = b.cuda()
    table[:, 3], table[:, 36], table[7, 37] = 1 << 20, -5, 1 << 30
    for r in range(rows):
        for c in (3, 36, 37) if r == 7 else (3, 36):
            for x in b.keys[r][:2]:
                x[16 * c:16 * c + 16] = 0
    held("out", dm.attention_decode_shared(q, k, v, table, *rest), *b.want())


def test_groups_of_many_rows_in_views():
    """Queries of a wider row, keys and values of one pool, heads ahead of the page's rows: the bits of the
    contiguous call."""
    rows = 70
    b = Batch(BF, 128, 2, 4, 16, [(0, [513 + 7 * (i % 5) for i in range(rows)], 512)], {}, rows, seed=3)
    q, k, v, *rest = b.cuda()
    want = dm.attention_decode_shared(q, k, v, *rest)
    held("contiguous", want, *b.want())
    wide = torch.cat([q, q, q], 1)[:, 8:16]
    both = torch.stack([k, v], 1)
    ahead = both.transpose(2, 3).contiguous()
    assert torch.equal(dm.attention_decode_shared(wide, both[:, 0], both[:, 1], *rest), want)
    assert torch.equal(dm.attention_decode_shared(q, ahead[:, 0].transpose(1, 2), ahead[:, 1].transpose(1, 2), *rest), want)


@pytest.mark.parametrize("dtype,d,groups,rows", [
    (BF, 128, [(0, [1500 + 3 * i for i in range(66)], 1481)], 66),          # many rows
    (BF, 256, [(0, [900 + 3 * i for i in range(40)], 887)], 40),
    (BF, 128, [(1, [300], 256), (2, [90, 700, 91, 95, 400, 89], 89)], 9),   # few
    (F32, 64, [(0, [200, 190, 313], 180)], 3)], ids=str)
def test_a_captured_call_follows_its_lengths(dtype, d, groups, rows):
    """Lengths that move on between the replays, to shorter rows and to none, and the prefixes and groups
    with them: each replay has the eager call's bits and the 64-bit result of these lengths."""
    b = Batch(dtype, d, 2, 4, 16, groups, {}, rows, seed=2)
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
    full = b.keys
    for i, (cut, first) in enumerate(((0, -1), (37, 0), (0, -1), (150, 2))):
        # every row `cut` keys shorter, row `first` without any
        lens = [0 if r == first else max(0, len(x[0]) - cut) for r, x in enumerate(full)]
        b.keys = [(x[0][:n], x[1][:n], 0) for x, n in zip(full, lens)]
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        if i == 3:
            cu.zero_()
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call()), i
        held(f"replay {i}", got, *b.want())


# ------------------------------------------------------------------------------------------
# Scores of minus infinity, values that are not finite
# ------------------------------------------------------------------------------------------

ALL = [(BF, 128, 16), (F16, 64, 16), (BF, 256, 16), (F32, 64, 16), (BF, 96, 16), (BF, 128, 7)]


@pytest.mark.parametrize("rows", [3, 60])
@pytest.mark.parametrize("dtype,d,page", ALL, ids=str)
def test_keys_of_minus_infinity_have_no_weight(dtype, d, page, rows):
    """Keys that a program has switched off with an element of minus infinity (the queries' are above 0
    there), the first ones of the prefix and the first ones behind it: the row's result is that of its other keys."""
    p = 592
    b = Batch(dtype, d, 1, 4, page, [(0, [p + 70 + i for i in range(rows)], p)], {}, rows, seed=4)
    b.q[:, :, 2] = b.q[:, :, 2].abs() + 0.125
    off = list(range(0, 150)) + list(range(p, p + 40))
    for r in range(rows):
        for j in off:
            b.k[int(b.table[r, j // page]), j % page, 0, 2] = -float("inf")
    on = torch.ones(p + 70 + rows, dtype=torch.bool)
    on[off] = False
    b.keys = [(k[on[:len(k)]], v[on[:len(v)]], 0) for k, v, _ in b.keys]
    held("out", dm.attention_decode_shared(*b.cuda()), *b.want())


@pytest.mark.parametrize("rows", [3, 60])
@pytest.mark.parametrize("dtype,d,page", ALL, ids=str)
def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it(dtype, d, page, rows):
    """Whatever its key's weight: e^-400 of the others' here, 0 in 32 bits, and zero times NaN is NaN. The row's
    other columns and the other rows are what they were."""
    lens = [2000 + i for i in range(rows)]
    b = Batch(dtype, d, 1, 4, page, [(0, lens, 1000)], {}, rows, seed=6)
    b.q[:, :, 0] = 40.0
    for k, _, _ in b.keys:
        k[:, :, 0] = 0.0
    b.k[:, :, :, 0] = torch.where(torch.isnan(b.k[:, :, :, 0].float()), b.k[:, :, :, 0], torch.zeros((), dtype=dtype))
    opts = dm.AttentionOptions(scale=1.0)
    b.q[:, :, 1:] *= 0.1
    for r in (1, 2):  # whole ranges of such keys
        for j in range(1400, lens[r]):
            b.k[int(b.table[r, j // page]), j % page, 0, 0] = -10.0
        b.keys[r][0][1400:, :, 0] = -10.0
    want, bound = b.want(1.0)
    b.v[int(b.table[1, 1990 // page]), 1990 % page, 0, 3] = float("nan")
    b.v[int(b.table[2, 1500 // page]), 1500 % page, 0, 5] = float("nan")
    out = dm.attention_decode_shared(*b.cuda(), opts)
    assert torch.isnan(out[1, :, 3]).all() and torch.isnan(out[2, :, 5]).all()
    keep = torch.ones(out.shape, dtype=torch.bool)
    keep[1, :, 3] = keep[2, :, 5] = False
    held("others", out[keep.cuda()], want[keep], bound[keep])


# ------------------------------------------------------------------------------------------
# Sums over many keys
# ------------------------------------------------------------------------------------------
#
# A key of score `scale`, then n - 1 of score 0: all weights but the first are w = e^-scale, so that every
# addition to a sum of them is off to the same side. Rounded sums of equal positive terms are off by at most
# u / 2 times their number of additions (the sum grows evenly), u = 2^-24.

def _equal_keys(dtype, d, n, w, values, rows, groups, rep):
    """Row 0 has n such keys, in its own pages if groups is None and as the prefix of a group otherwise; the
    other rows have one key. Returns (arrays, options, the result of row 0 in 64 bits)."""
    page = 16
    k, v = (torch.zeros(n // page + 1, page, 1, d, dtype=dtype, device="cuda") for _ in range(2))
    k[0, 0, 0, 0] = 1.0
    v[:] = values.to(dtype).cuda()
    table = torch.full((rows, n // page), -1, dtype=torch.int32, device="cuda")
    table[0] = torch.arange(n // page, dtype=torch.int32)
    table[1:, 0] = n // page
    lengths = torch.ones(rows, dtype=torch.int32, device="cuda")
    lengths[0] = n
    q = torch.zeros(rows, rep, d, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    if groups:
        cu = torch.arange(rows + 1, dtype=torch.int32, device="cuda")
        pl = torch.ones(rows, dtype=torch.int32, device="cuda")
        pl[0] = n
    else:
        cu, pl = (torch.zeros(i, dtype=torch.int32, device="cuda") for i in (1, 0))
    scale = float(-torch.log(torch.tensor(w, dtype=torch.float64)))
    return (q, k, v, table, lengths, cu, pl), dm.AttentionOptions(scale=scale), v[0, 0, 0].double().cpu()


def _sum_held(args, opts, want, bound):
    out = dm.attention_decode_shared(*args, opts)[0].flatten(0, -2)
    held("row 0", out, want.expand_as(out), bound * want.abs().expand_as(out))


def test_sums_of_a_long_prefix_of_many_rows():
    """2^19 keys in one range (100 groups, 115 tiles). Off by: the weights' rounding for the products, half a
    step; the products' sums over 16 keys a time, n / 16 additions; the weights' sum, in which a lane takes
    32 keys of a tile (at most 32 u) and n / 64 tiles; 64 u for the rest. w is 63.49 steps of a sum between 2^17 and 2^18: added
    one at a time the weights' sum is 0.4% short."""
    n = 1 << 19
    args = _equal_keys(F16, 64, n, 63.49 / 64, torch.ones(64), 100, True, 40)
    _sum_held(*args, 2.0 ** -11 + (n / 32 + n / 128 + 96) * U)


@pytest.mark.parametrize("groups", [True, False])
@pytest.mark.parametrize("dtype,d", [(F32, 64), (F32, 36), (BF, 96)], ids=str)
def test_sums_of_the_simple_form(dtype, d, groups):
    """2^14 keys in one range (520 tiles), 16 of them at a time. Off by: the sums of 16 keys' products and n / 16
    additions of those; the weights' sums, each of 8 threads' n / 16 additions of two; 128 u for the scores, the
    weights and the rest. (A result in bf16 is rounded once: the weights stay in f32 here.) With one addition a key
    the products' sums in f32 are 2.3e-4 short: a column's terms are a whole number and 0.49 of a step of them."""
    n, w = 1 << 14, 0.992
    values = (1000.49 + torch.arange(d, dtype=torch.float64)) / 1024 / w
    args = _equal_keys(dtype, d, n, w, values, 520, groups, 1)
    _sum_held(*args, (n / 32 + n / 32 + 128) * U)
