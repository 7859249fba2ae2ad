"""The attention of new tokens over a paged cache and its keys' weights where values, lengths and batches are
extreme, against 64 bits (chunk_cases.py, which derives the bounds)."""
import ctypes

import pytest
import torch

import dashmag_amd as dm
from dashmag_amd import _lib
from chunk_cases import Chunks, held_lse
from rope_cases import held
from shared_cases import U

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _without(b, gone):
    """b.want() of one sequence without a window, whose key `gone` has a score of -inf in every row."""
    (n, x), d = b.seqs[0], b.d
    k, v = (y.double().transpose(0, 1) for y in b.keys[0])
    k = k.clone()
    k[:, gone] = 0.0
    q = b.q.double().unflatten(1, (k.shape[0], b.rep)).permute(1, 2, 0, 3)  # [Hkv, rep, n, D]
    seen = (torch.arange(x) <= torch.arange(x - n, x)[:, None]) & (torch.arange(x) != gone)
    z = (q @ k.transpose(1, 2)[:, None] * d ** -0.5).masked_fill(~seen, -torch.inf)
    total = torch.logsumexp(z, -1, keepdim=True)
    p = torch.exp(z - total)
    s = ((q.abs() @ k.abs().transpose(1, 2)[:, None]) * d ** -0.5).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    e = (d + 16) * U * s
    half = 0.0 if b.q.dtype == F32 else torch.finfo(b.q.dtype).eps / 2
    bound = (half + 2 * e + 2 * (x / 16 + 64) * U) * (p @ v[:, None].abs())
    if b.q.dtype == F16:
        bound = bound + 2.0 ** -25 * seen.double() @ v[:, None].abs()
    g = e + (x / 16 + 64) * U + 8 * U * (total.abs() + 1)
    back = lambda y: y.permute(2, 0, 1, 3).flatten(1, 2)  # noqa: E731
    w, woff = b.weights.double(), torch.zeros(b.weights.shape, dtype=torch.float64)
    w[0, :x] += p.sum((0, 1, 2))
    woff[0, :x] = (p * (e + g + (p.shape[0] * p.shape[1] * n + 40) * U)).sum((0, 1, 2))
    return (back(p @ v[:, None]), back(bound)), (back(total)[..., 0], back(g)[..., 0]), (w, woff + U * w)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256), (F32, 64), (BF, 40)])
@pytest.mark.parametrize("rep,n", [(1, 5), (4, 3), (3, 15), (1, 33), (4, 24), (4, 25)])
def test_a_key_of_infinity_that_no_token_gives_weight(dtype, d, rep, n):
    """An infinite element of a key makes its scores -inf in every row: a weight of 0, whether or not the rows fill
    the steps that the keys are swept in."""
    x, gone = 300, 70
    b = Chunks(dtype, d, 2, rep, 16, [(n, x)], seed=d + n)
    b.q[..., 0] = b.q[..., 0].abs() + 0.5
    q, k, v, table, ln, cu = b.cuda()
    k[int(table[0, gone // 16]), gone % 16, :, 0] = -torch.inf
    w = b.weights.cuda()
    out, lse = dm.attention_paged_with_weights(q, k, v, table, ln, w, cu)
    want, want_lse, want_w = _without(b, gone)
    assert w[0, gone] == b.weights[0, gone]
    held("out", out, *want)
    held_lse("lse", lse, *want_lse)
    held("weights", w, *want_w)


def _held_all(b, scale=None):
    q, k, v, table, ln, cu = b.cuda()
    w = b.weights.cuda()
    opts = dm.AttentionOptions(window=None if b.window is None else dm.Window(b.window, 0), scale=scale)
    out, lse = dm.attention_paged_with_weights(q, k, v, table, ln, w, cu, opts)
    want = b.want(scale)
    held("out", out, *want["out"])
    held_lse("lse", lse, *want["lse"])
    held("weights", w, *want["weights"])


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256), (F32, 64)])
def test_rows_around_the_tiles_borders(dtype, d):
    """Sequences of a row more and less than one narrow tile, two of them, and what leaves its scores; keys around a
    narrow worker's least."""
    for rep, news in ((1, (7, 8, 9, 31, 32, 33, 47, 48, 49, 63, 64, 65)), (4, (1, 2, 3, 7, 8, 9, 11, 12, 13, 15, 16, 17))):
        for window in (None, 70):
            print(f"rep={rep} window={window}", flush=True)
            _held_all(Chunks(dtype, d, 1, rep, 16, [(n, x) for n in news for x in (n, n + 64, n + 130)], seed=rep, window=window))
    _held_all(Chunks(dtype, d, 1, 4, 16, [(8, x) for x in (8, 31, 32, 33, 63, 64, 65, 95, 96, 97, 511, 513)], seed=3))
    _held_all(Chunks(dtype, d, 1, 4, 16, [(9, x) for x in (9, 63, 64, 65, 191, 192, 193, 255, 256, 257)], seed=4))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256), (BF, 64)])
def test_calls_of_few_rows(dtype, d):
    """Calls of 31 to 65 rows a key head altogether: a sequence's, several sequences', tokens', in and out of a wide line."""
    for rep, rows in ((1, (31, 32, 33, 47, 48, 49, 63, 64, 65)), (4, (32, 36, 48, 52, 64, 68)), (40, (40, 80)), (33, (33, 66))):
        for n in (r // rep for r in rows):
            print(f"rep={rep} tokens={n}", flush=True)
            _held_all(Chunks(dtype, d, 2, rep, 16, [(n, n + 700)], seed=n))
            _held_all(Chunks(dtype, d, 2, rep, 7, [(1, 40 * i) for i in range(n)], seed=n, window=300))
            _held_all(Chunks(dtype, d, 2, rep, 16, [(1, 90 + i) for i in range(n)], seed=n, single=True))
            if n > 3:
                _held_all(Chunks(dtype, d, 2, rep, 16, [(2, 900), (0, 5), (n - 3, 400)], seed=n, gaps=(0, 1)))


def _weighing_workspace(b, cols):
    """Bytes of the call's workspace."""
    d = _lib.AttentionDesc(b=len(b.seqs), tq=len(b.q), tk=cols * b.page, hq=b.q.shape[1], hkv=b.k.shape[2], d=b.d,
                           dtype=_lib.DM_BF16 if b.q.dtype == BF else _lib.DM_F16, cu_seqlens_q=256)
    return _lib.lib().dm_attention_paged_workspace(ctypes.byref(d), b.page, 1)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256)])
@pytest.mark.parametrize("window", [None, 50])
def test_weights_of_few_rows_without_kept_scores(dtype, d, window):
    """Batches of prompts, drafts and tokens on a table so wide that no scores are kept: those of few rows too get their
    weights by another pass over the keys; the same on a narrow table, whose scores are kept."""
    seqs = [(90, 400), (1, 700), (2, 130), (17, 130), (3, 9), (0, 12), (8, 2100)]
    b = Chunks(dtype, d, 2, 4, 16, seqs, seed=d + 1, window=window)
    q, k, v, table, ln, cu = b.cuda()
    opts = dm.AttentionOptions(window=None if window is None else dm.Window(window, 0))
    want = b.want()
    scores = len(seqs) * 2 * 8 * table.shape[1] * 16 * 4  # (of 8 rows a sequence and key head: kept on the narrow table alone)
    assert _weighing_workspace(b, table.shape[1]) - _weighing_workspace(b, 1 << 19) >= scores
    for cols in (1 << 19, table.shape[1]):
        wide = torch.full((len(seqs), cols), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        w = torch.full((len(seqs), cols * 16), 0.25, device="cuda")
        w[:, :b.weights.shape[1]] = b.weights.cuda()
        out, lse = dm.attention_paged_with_weights(q, k, v, wide, ln, w, cu, opts)
        held("out", out, *want["out"])
        held_lse("lse", lse, *want["lse"])
        held("weights", w[:, :b.weights.shape[1]], *want["weights"])
        assert (w[:, b.weights.shape[1]:] == 0.25).all()


@pytest.mark.parametrize("dtype", [F16, BF])
@pytest.mark.parametrize("d,seqs,new", [(64, 2048, 1), (128, 2048, 1), (256, 1024, 1), (64, 256, 70), (128, 256, 70), (256, 256, 70)])
def test_many_small_weights_beside_a_large_one(dtype, d, seqs, new):
    """131072 keys of a weight of 2^-25.5 each beside a first of 1, as many sequences as workers: together they are 0.0028 of
    the sum. With values of 1 an output is 1 but for its rounding and its weights' (half a step each), f16 weights lost
    below 2^-32, and the f32 sums of its weights and products: chains of keys / 16 + 64 additions to sums near their last
    value, each off by u = 2^-24 of it, 2^13 u = 2^-11 a sum; E = 17 u S for scores of one product up to S = 17.7."""
    keys, page = 131073, 16
    pages = -(-keys // page)
    q = torch.zeros(seqs * new, 1, d, dtype=dtype, device="cuda")
    k = torch.zeros(pages, page, 1, d, dtype=dtype, device="cuda")
    v = torch.ones_like(k)
    q[..., 0] = 16.0
    k[0, 0, 0, 0] = 1.0
    scale = 25.5 * 0.6931471805599453 / 16
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(seqs, pages).contiguous()
    ln = torch.full((seqs,), keys, dtype=torch.int32, device="cuda")
    cu = torch.arange(0, seqs * new + 1, new, dtype=torch.int32, device="cuda")
    print(f"{dtype} D={d} {seqs} sequences of {new}", flush=True)
    out, lse = dm.attention_paged_with_lse(q, k, v, table, ln, cu, dm.AttentionOptions(scale=scale))
    half = torch.finfo(dtype).eps / 2
    off = (out.double() - 1).abs().max().item()
    seen = keys - new + 1 + (torch.arange(new, dtype=torch.float64) if new > 1 else torch.zeros(1, dtype=torch.float64))
    want = 25.5 * 0.6931471805599453 + torch.log1p((seen - 1) * 2.0 ** -25.5)
    loff = (lse.cpu().double().view(seqs, new) - want).abs().max().item()
    print(f"out {off:.2e}, lse {loff:.2e}", flush=True)
    chain, e = (keys / 16 + 64) * U, 17 * U * 17.7
    assert off <= 2 * half + keys * 2.0 ** -32 * (dtype == F16) + 2 * chain + 2 * e
    assert loff <= chain + e + 8 * U * (17.7 + 1)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (BF, 256), (F32, 64)])
@pytest.mark.parametrize("between", [1, 63, 64, 65, 127, 200, 1100])
def test_sequences_between_those_of_a_line(dtype, d, between):
    """Prompts with many sequences of few or no tokens between them and behind the last: a worker goes from one to the
    next past all of them, among the wide tiles, the narrow ones and the keys'."""
    few = [(0, 7), (1, 5), (0, 0), (2, 3)]
    gap = [few[i % 4] for i in range(between)]
    _held_all(Chunks(dtype, d, 1, 4, 16, [(90, 400), *gap, (41, 333), *gap[:between // 2], (130, 131), (0, 3)], seed=between))
    _held_all(Chunks(dtype, d, 1, 4, 16, [(3, 90), *[(0, 9)] * between, (5, 400), *[(0, 0)] * between, (12, 30)], seed=between))
