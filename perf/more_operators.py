"""Chunks of new tokens against a paged key-value cache, and what of the cache is kept, as measurable calls.

Three operators: the attention of ragged batches of new tokens (chunks of prompts, drafted tokens to be
verified, single tokens) over a paged cache, the same with the attention weights accumulated for each
cached key, and the eviction of a row's keys by those weights. With ``own`` false a pass runs in plain
torch operations, in 32 bits; with ``own`` true it calls ``dashmag_amd``.

Inputs are on the GPU: activations N(0, 1), accumulated weights log-normal (few keys get most of the
attention), offsets, lengths and tables int32 as the program's scheduler leaves them, pages of a sequence
scattered over the pool. The new tokens' keys and values lie in the pages already.
"""
import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------
# The cases
# ------------------------------------------------------------------------------------------
#
# prompts sequences get up to `new` tokens each, `singles` one; a sequence held up to `held` keys before.

def listed():
    return [
        # The last chunk of a long document's prefill: the largest call.
        dict(name="chunk_document_d128", kind="chunk", dtype="bf16", prompts=1, new=2048, singles=0,
             held=30720, hq=32, hkv=8, d=128, page=16, window=0, lay=1),
        # Prompts arriving at conversations of some length.
        dict(name="chunk_prompts_d128", kind="chunk", dtype="bf16", prompts=9, new=1400, singles=0,
             held=2048, hq=32, hkv=8, d=128, page=16, window=0, lay=2),
        # A scheduler's mixed step: chunks of two prompts beside the tokens of 62 conversations.
        dict(name="chunk_mixed_d128", kind="chunk", dtype="bf16", prompts=2, new=512, singles=62,
             held=8192, hq=32, hkv=8, d=128, page=16, window=0, lay=3),
        # Drafted tokens verified, two to six a sequence, narrow heads with a sliding window.
        dict(name="chunk_drafts_d64", kind="chunk", dtype="f16", prompts=32, new=6, singles=0,
             held=6000, hq=16, hkv=2, d=64, page=32, window=4000, lay=4),
        # Wide heads: the second chunk of four prompts.
        dict(name="chunk_prompts_d256", kind="chunk", dtype="bf16", prompts=4, new=1536, singles=0,
             held=6144, hq=8, hkv=2, d=256, page=16, window=0, lay=5),
        # Single precision and pages of an odd size: a small call.
        dict(name="chunk_f32_d64", kind="chunk", dtype="f32", prompts=3, new=70, singles=0,
             held=300, hq=4, hkv=4, d=64, page=7, window=0, lay=6),
        # One token for each of 64 conversations, and for each of four short ones, where latency counts.
        dict(name="token_d128", kind="chunk", dtype="bf16", prompts=0, new=1, singles=64,
             held=8192, hq=32, hkv=8, d=128, page=16, window=0, lay=7),
        dict(name="token_few_d128", kind="chunk", dtype="bf16", prompts=0, new=1, singles=4,
             held=1000, hq=8, hkv=2, d=128, page=16, window=0, lay=8),
        # The weights that eviction goes by, of a document's chunk and of 64 conversations' tokens.
        dict(name="weigh_document_d128", kind="weigh", dtype="bf16", prompts=1, new=1024, singles=0,
             held=15360, hq=32, hkv=8, d=128, page=16, window=0, lay=9),
        dict(name="weigh_token_d128", kind="weigh", dtype="bf16", prompts=0, new=1, singles=64,
             held=4096, hq=32, hkv=8, d=128, page=16, window=0, lay=10),
        # Half of each of 16 conversations' keys given up; two layers' pools.
        dict(name="evict_rows", kind="evict", dtype="bf16", rows=16, length=4096, budget=2048, recent=256,
             shared=0, spare=500, page=16, hkv=8, d=128, layers=2, lay=11),
        # One long document cut down to an eighth, behind a prefix that other rows hold too; one layer's pools.
        dict(name="evict_document", kind="evict", dtype="bf16", rows=2, length=32768, budget=4096, recent=512,
             shared=1024, spare=200, page=16, hkv=8, d=128, layers=1, lay=12),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "chunk", "weigh", "weigh", "evict"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
    hkv = rng.choice([1, 2, 4, 8])
    d = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64, 24, 7])
    if kind == "evict":
        length = _log(rng, 20, 8192)
        budget = _log(rng, 1, length)
        return dict(kind=kind, dtype=dtype, rows=max(1, _log(rng, 2, 65536) // length), length=length,
                    budget=budget, recent=rng.choice([0, budget // 8, budget // 2]),
                    shared=rng.choice([0, 0, length // 10]), spare=_log(rng, 5, 500), page=page, hkv=hkv, d=d,
                    layers=rng.choice([1, 1, 2]), lay=rng.randrange(1 << 30))
    hq = hkv * rng.choice([1, 2, 4, 4, 8])
    form = rng.choice(["one", "prompts", "drafts", "singles", "mixed"])
    prompts = {"one": 1, "prompts": _log(rng, 2, 16), "drafts": _log(rng, 2, 64), "singles": 0,
               "mixed": rng.choice([1, 2, 3])}[form]
    sequences = prompts if form in ("one", "prompts", "drafts") else prompts + 64
    # (as many cached values as the largest listed calls have, and as many scores; fewer in f32)
    held = _log(rng, 1, max(1, min(16384, (1 << 29) // (sequences * hkv * d) // (4 if dtype == "f32" else 1))))
    most = (1 << 30) // (d // 64) // (16 if dtype == "f32" else 1)
    new = max(1, min(_log(rng, 2, 8 if form == "drafts" else 4096),
                     most // (max(prompts, 1) * hq * (held + 512))))
    return dict(kind=kind, dtype=dtype, prompts=prompts, new=new if prompts else 1,
                singles=_log(rng, 1, 64) if form in ("singles", "mixed") else 0, held=held, hq=hq, hkv=hkv, d=d,
                page=page, window=rng.choice([0, 0, 0, 500, 3000]), lay=rng.randrange(1 << 30))


# ------------------------------------------------------------------------------------------
# What a case's sequences look like
# ------------------------------------------------------------------------------------------

def _layout(case):
    """(new tokens of each sequence, its length with them): the prompts first."""
    rng = random.Random(case["lay"])
    n, h = case["new"], case["held"]
    new = [rng.randint(1 + n // 4, n) if case["prompts"] > 1 and n > 1 else n for _ in range(case["prompts"])]
    new += [1] * case["singles"]
    return new, [x + (h if len(new) == 1 else rng.randint(h // 2, h)) for x in new]


def _evict_layout(case):
    """The rows' lengths."""
    rng = random.Random(case["lay"])
    n = case["length"]
    return [rng.randint(max(1, n * 7 // 8), n) for _ in range(case["rows"])]


def _pages_of(length, page):
    return -(-length // page)


# ------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------

def _i32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _table(gen, each, pages):
    """[rows, the most pages of a row] int32: ``each[r]`` pages of row ``r``, drawn without putting
    back, then -1."""
    taken = torch.randperm(pages, generator=gen, device="cuda")
    n = torch.tensor(each, device="cuda")
    j = torch.arange(max(each + [1]), device="cuda")
    at = (torch.cumsum(n, 0) - n)[:, None] + j
    return torch.where(j < n[:, None], taken[at.clamp(max=pages - 1)], -1).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape, dtype=DT[case["dtype"]]):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    s = dict(case)
    page, hkv, d = case["page"], case["hkv"], case["d"]
    if case["kind"] != "evict":
        new, lengths = _layout(case)
        each = [_pages_of(x, page) for x in lengths]
        pages = sum(each) + 5
        s["table"] = _table(gen, each, pages)
        s["q"] = randn(sum(new), case["hq"], d)
        s["kp"], s["vp"] = (randn(pages, page, hkv, d) for _ in range(2))
        s["lengths"] = _i32(lengths)
        s["starts"] = torch.cumsum(_i32([0] + new), 0, dtype=torch.int32)
        s["cu"] = s["starts"] if case["prompts"] else None
        p = case["prompts"]
        s["most"] = (max(new[:p] + [0]), max(lengths[:p] + [0]), max(lengths[p:] + [0]))
        if case["kind"] == "weigh":
            shape = len(new), s["table"].shape[1] * page
            s["weights"] = torch.exp(randn(*shape, dtype=torch.float32))
        return s
    lengths = _evict_layout(case)
    # whole pages that the first two rows both hold at their beginnings
    both = min(case["shared"], min(lengths)) // page if len(lengths) > 1 else 0
    each = [_pages_of(x, page) for x in lengths]
    pages = sum(each) + case["spare"]
    table = _table(gen, each, pages)
    if both:
        table[1, :both] = table[0, :both]
    held = table[table >= 0].long()
    s["table_from"], s["lengths_from"] = table, _i32(lengths)
    s["refcounts_from"] = torch.zeros(pages, dtype=torch.int32, device="cuda").index_add_(
        0, held, torch.ones_like(held, dtype=torch.int32))
    cap = table.shape[1] * page
    s["weights_from"] = torch.where(torch.arange(cap, device="cuda") < s["lengths_from"][:, None],
                                    torch.exp(2 * randn(len(lengths), cap, dtype=torch.float32)), 0.0)
    for x in ("table", "lengths", "refcounts", "weights"):
        s[x] = s[x + "_from"].clone()
    s["budgets"] = _i32([case["budget"]] * len(lengths))
    s["pools"] = torch.stack([randn(pages, page, hkv, d) for _ in range(2 * case["layers"])])
    return s


# ------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------

def _plain_group(s, first, last, most_new, most_len, out, lse):
    """The sequences first .. last - 1, padded to the most new tokens and keys; with the weights' array in the
    state, their weights are added."""
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], s["page"]
    rep, g = hq // hkv, last - first
    starts, lengths = s["starts"].long(), s["lengths"][first:last].long()
    new = starts[first + 1:last + 1] - starts[first:last]
    i = torch.arange(most_new, device="cuda")
    at = torch.arange(most_len, device="cuda")
    live = i < new[:, None]
    token = (starts[first:last, None] + i).clamp(max=s["q"].shape[0] - 1)
    where = (lengths - new)[:, None] + i  # [G, n]
    pages = s["table"][first:last][:, at // page].long().clamp(min=0)
    keys, values = (s[x][pages, at % page].float().permute(0, 2, 1, 3) for x in ("kp", "vp"))  # [G, Hkv, L, D]
    q = s["q"][token].float().view(g, most_new, hkv, rep, d).permute(0, 2, 1, 3, 4).reshape(g, hkv, -1, d)
    scores = torch.matmul(q * (1.0 / math.sqrt(d)), keys.transpose(-1, -2)).view(g, hkv, most_new, rep, most_len)
    seen = live[..., None] & (at <= where[..., None])
    if s["window"]:
        seen = seen & (at >= (where - s["window"])[..., None])
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.view(g, hkv, -1, most_len), values).view(g, hkv, most_new, rep, d)
    out[token[live]] = o.permute(0, 2, 1, 3, 4).reshape(g, most_new, hq, d)[live]
    lse[token[live]] = (top + total.log())[..., 0].permute(0, 2, 1, 3).reshape(g, most_new, hq)[live]
    if s["kind"] == "weigh":
        s["weights"][first:last, :most_len] += p.sum((1, 2, 3))


def _plain_chunk(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float32, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, device="cuda")
    new, prompts_len, singles_len = s["most"]
    if s["prompts"]:
        _plain_group(s, 0, s["prompts"], new, prompts_len, out, lse)
    if s["singles"]:
        _plain_group(s, s["prompts"], s["prompts"] + s["singles"], 1, singles_len, out, lse)
    return (out.to(s["q"].dtype), lse) + ((s["weights"],) if s["kind"] == "weigh" else ())


def _plain_evict(s):
    pools, weights, table, lengths, counts = (s[x] for x in ("pools", "weights", "table", "lengths", "refcounts"))
    page, cap = s["page"], weights.shape[1]
    held, old = lengths.long()[:, None], table.clone()
    j = torch.arange(cap, device="cuda").expand(weights.shape[0], -1)
    col = torch.arange(table.shape[1], device="cuda")
    mine = col < (held + page - 1) // page
    # always kept: the keys up to the last page that another row holds, and the recent ones
    others = mine & (counts[table.long().clamp(min=0)] > 1)
    fixed = torch.where(others, (col + 1) * page, 0).amax(1, keepdim=True)
    live = j < held
    budgets = s["budgets"].long()[:, None]
    always = live & ((j < fixed) | (j >= held - budgets.clamp(max=s["recent"])))
    n = torch.minimum(held, torch.maximum(budgets, always.sum(1, keepdim=True)))
    # the heaviest of the others, ties to the lowest index
    rank = torch.where(always, math.inf, torch.where(live, weights, -math.inf))
    order = torch.sort(rank, dim=1, descending=True, stable=True)[1]
    place = torch.empty_like(order).scatter_(1, order, j.contiguous())
    keep = live & (place < n)
    kept = torch.sort(torch.where(keep, j, cap), 1)[0]
    kept = torch.where(j < n, kept, -1)
    # the kept keys move down
    go = (kept >= 0) & (kept != j)
    r = torch.arange(weights.shape[0], device="cuda")[:, None].expand_as(j)[go]
    src, dst = kept[go], j[go]
    flat = pools.view(pools.shape[0], -1, pools.shape[-2] * pools.shape[-1])
    flat[:, table[r, dst // page].long() * page + dst % page] = flat[:, old[r, src // page].long() * page + src % page]
    weights.copy_(torch.where(j < n, weights.gather(1, kept.clamp(min=0)), torch.where(live, 0.0, weights)))
    # the pages behind them are given up
    gone = mine & (col >= (n + page - 1) // page)
    given = table[gone].long()
    counts.index_add_(0, given, torch.full_like(given, -1, dtype=torch.int32))
    table.masked_fill_(gone, -1)
    lengths.copy_(n[:, 0])
    return kept.to(torch.int32), weights, table, lengths, counts, pools


def run(s):
    if s["kind"] == "evict":
        # the rows as they were found; the pools still hold what is moved below
        for x in ("table", "lengths", "refcounts", "weights"):
            s[x].copy_(s[x + "_from"])
    if not own:
        return _plain_evict(s) if s["kind"] == "evict" else _plain_chunk(s)
    import dashmag_amd as dm
    if s["kind"] == "evict":
        kept = dm.cache_evict(list(s["pools"].unbind(0)), s["weights"], s["table"], s["lengths"], s["refcounts"],
                              s["budgets"], s["recent"])
        return kept, s["weights"], s["table"], s["lengths"], s["refcounts"], s["pools"]
    options = dm.AttentionOptions(window=dm.Window(s["window"], 0) if s["window"] else None)
    if s["kind"] == "chunk":
        return dm.attention_paged_with_lse(s["q"], s["kp"], s["vp"], s["table"], s["lengths"], s["cu"], options)
    out, lse = dm.attention_paged_with_weights(s["q"], s["kp"], s["vp"], s["table"], s["lengths"], s["weights"],
                                               s["cu"], options)
    return out, lse, s["weights"]


# ------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------

def work(case):
    e, page = SIZE[case["dtype"]], case["page"]
    if case["kind"] != "evict":
        new, lengths = _layout(case)
        w = case["window"]
        keys = seen = 0
        for n, x in zip(new, lengths):
            keys += x - (max(0, x - n - w) if w else 0)
            # token i sees min(x - n + i, w) + 1 keys
            whole = min(n, max(0, w + 1 - (x - n))) if w else n
            seen += whole * (x - n + 1) + whole * (whole - 1) // 2 + (n - whole) * (w + 1)
        rows = sum(new) * case["hq"]
        weights = 8 * keys if case["kind"] == "weigh" else 0
        return {"bytes": 2 * keys * case["hkv"] * case["d"] * e + 2 * rows * case["d"] * e + 4 * rows +
                4 * keys // page + weights, "flops": 4 * seen * case["hq"] * case["d"]}
    lengths = _evict_layout(case)
    row = case["hkv"] * case["d"] * e * 2 * case["layers"]  # one key's bytes in every pool
    moved = kept = 0
    both = min(case["shared"], min(lengths)) // page * page if len(lengths) > 1 else 0
    for r, x in enumerate(lengths):
        fixed = both if r < 2 else 0
        n = min(x, max(case["budget"], min(x, fixed + min(case["recent"], case["budget"]))))
        kept += n
        moved += n - fixed if n < x else 0
    # the moved keys; the weights read once, the kept ones and the indices written
    return {"bytes": 2 * moved * row + 4 * sum(lengths) + 8 * kept, "flops": 0}


# ------------------------------------------------------------------------------------------
# In 64 bits, from the definitions
# ------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"]
    if case["kind"] != "evict":
        new, lengths = _layout(case)
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
        weights = s["weights"].double() if case["kind"] == "weigh" else None
        rep, first = case["hq"] // case["hkv"], 0
        for r, (n, x) in enumerate(zip(new, lengths)):
            key = torch.arange(x, device="cuda")
            slot = s["table"][r, key // page].long() * page + key % page
            at = torch.arange(x - n, x, device="cuda")[:, None]
            hidden = (key > at) | ((key < at - case["window"]) if case["window"] else key < 0)
            for h in range(case["hkv"]):
                k, v = (s[y].flatten(0, 1)[slot, h].double() for y in ("kp", "vp"))
                for a in range(h * rep, (h + 1) * rep):
                    z = torch.matmul(s["q"][first:first + n, a].double(), k.T) / math.sqrt(case["d"])
                    z[hidden] = -math.inf
                    total = torch.logsumexp(z, 1)
                    p = torch.exp(z - total[:, None])
                    out[first:first + n, a], lse[first:first + n, a] = torch.matmul(p, v), total
                    if weights is not None:
                        weights[r, :x] += p.sum(0)
            first += n
        return (out, lse) + (() if weights is None else (weights,))
    pools, cap = s["pools"], s["weights"].shape[1]
    counts, table, weights = s["refcounts"].tolist(), s["table"].tolist(), s["weights"].tolist()
    lengths, before, after = s["lengths"].tolist(), s["refcounts"].tolist(), []
    kept = [[-1] * cap for _ in lengths]
    for r, x in enumerate(lengths):
        fixed = max([0] + [(c + 1) * page for c in range(_pages_of(x, page)) if before[table[r][c]] > 1])
        always = {k for k in range(x) if k < fixed or k >= x - min(case["recent"], case["budget"])}
        rest = sorted((k for k in range(x) if k not in always), key=lambda k: (-weights[r][k], k))
        keep = sorted(always | set(rest[:max(0, case["budget"] - len(always))]))
        slot = [table[r][k // page] * page + k % page for k in range(x)]
        flat = pools.view(pools.shape[0], -1, case["hkv"] * case["d"])
        to, of = (torch.tensor(y, device="cuda") for y in (slot[:len(keep)], [slot[k] for k in keep]))
        flat[:, to] = flat[:, of].clone()
        kept[r][:len(keep)] = keep
        weights[r][:x] = [weights[r][k] for k in keep] + [0.0] * (x - len(keep))
        for c in range(_pages_of(len(keep), page), _pages_of(x, page)):
            counts[table[r][c]] -= 1
            table[r][c] = -1
        after.append(len(keep))
    return (_i32(kept), torch.tensor(weights, dtype=torch.float64, device="cuda"), _i32(table), _i32(after),
            _i32(counts), pools.double())
