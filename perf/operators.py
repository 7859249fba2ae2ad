"""An attention layer around its paged key-value cache, as measurable calls.

Three operators: the norms and the rotation of queries and keys (for training, with their
gradients, and for serving, where the new keys and values go to the cache's pages), the decoding
attention of a batch whose sequences share a long prefix, and the pages themselves (reserved,
forked, freed, compacted). With ``own`` false a pass runs in plain torch operations, in 32 bits
(angles in 64); with ``own`` true it calls ``dashmag_amd``.

Inputs are on the GPU: activations N(0, 1), norm weights 1 + N(0, 0.1) (N(0, 0.1) around a unit
offset), offsets, lengths and tables int32 as the program's scheduler leaves them, pages of a
sequence scattered over the pool.
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

def listed():
    return [
        # The attention layers of a training step over a packed batch of documents, whose
        # positions start again at each: the batch of the benchmark, forward and backward.
        dict(name="rotate_packed_d128", kind="rotate", dtype="bf16", b=1, t=16384, hq=32, hkv=8,
             d=128, n=64, interleaved=False, unit=False, fused=False, weight="bf16", places="packed"),
        dict(name="rotate_grad_packed_d128", kind="rotate_grad", dtype="bf16", b=1, t=16384, hq=32,
             hkv=8, d=128, n=64, interleaved=False, unit=False, fused=False, weight="bf16",
             places="packed"),
        # The wide heads of a hybrid Gated DeltaNet model: a quarter of each head rotates, the
        # weights sit around one, q and k are slices of one projection.
        dict(name="rotate_grad_part_d256", kind="rotate_grad", dtype="bf16", b=1, t=6144, hq=16,
             hkv=2, d=256, n=32, interleaved=False, unit=True, fused=True, weight="f32",
             places="count"),
        # Single precision, adjacent pairs, far positions, an odd batch: a small call.
        dict(name="rotate_f32_d64", kind="rotate", dtype="f32", b=3, t=257, hq=4, hkv=4, d=64, n=32,
             interleaved=True, unit=False, fused=False, weight="f32", places="far"),
        # Serving: prompts arriving at sequences that hold some already (a chunked prefill).
        dict(name="append_prompts_d128", kind="append", dtype="bf16", seqs=9, tokens=8192, held=2048,
             hq=32, hkv=8, d=128, n=64, page=16, interleaved=False, unit=False, lay=1),
        # Serving: one token for each of 64 sequences, a call of microseconds.
        dict(name="append_token_d128", kind="append", dtype="bf16", seqs=64, tokens=64, held=2048,
             hq=32, hkv=8, d=128, n=64, page=16, interleaved=False, unit=False, lay=2),
        # Eight answers to one prompt, wide heads: the smallest shared decode.
        dict(name="shared_samples_d256", kind="shared", dtype="bf16", batch=8, groups=1, prefix=6144,
             own=200, hq=8, hkv=2, d=256, page=16, window=0, idle=0, lay=3),
        # A system prompt in front of 64 conversations.
        dict(name="shared_prompt_d128", kind="shared", dtype="bf16", batch=64, groups=1, prefix=16384,
             own=1024, hq=32, hkv=8, d=128, page=16, window=0, idle=0, lay=4),
        # Several prompts, a ragged number of answers to each, narrow heads with a sliding
        # window, the last rows of the batch without a request.
        dict(name="shared_groups_d64", kind="shared", dtype="f16", batch=45, groups=5, prefix=8000,
             own=700, hq=16, hkv=2, d=64, page=32, window=6000, idle=3, lay=5),
        # 256 agents with the same tools and documents in front: the largest call.
        dict(name="shared_agents_d128", kind="shared", dtype="bf16", batch=256, groups=1,
             prefix=32768, own=512, hq=32, hkv=8, d=128, page=16, window=0, idle=0, lay=6),
        # The scheduler's round of sampling: eight answers to each of eight prompts forked, pages
        # for their tokens reserved, the finished ones freed. Four layers' pools.
        dict(name="pages_round", kind="round", dtype="bf16", rows=128, parents=8, samples=8,
             length=1500, grow=40, pages=4096, page=16, hkv=8, d=128, layers=4, lay=7),
        # A pool half in use closed up after many sequences have ended. Two layers' pools.
        dict(name="pages_compact", kind="compact", dtype="bf16", rows=96, length=1000, pages=6000,
             page=16, hkv=8, d=128, layers=2, lay=8),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "rotate_grad", "rotate_grad", "append", "append", "shared",
                       "shared", "shared", "round", "compact"])
    half = rng.choice(["bf16", "bf16", "f16"])
    hkv = rng.choice([1, 2, 4, 8])
    d = rng.choice([64, 128, 128, 256])
    if kind in ("rotate", "rotate_grad"):
        dtype = rng.choice([half, half, half, "f32"])
        d = rng.choice([64, 96, 128, 128, 256])
        b = rng.choice([1, 1, 2, 3])
        return dict(kind=kind, dtype=dtype, b=b,
                    t=_log(rng, 1, (4096 if dtype == "f32" else 16384) // (b * max(1, d // 128))),
                    hq=hkv * rng.choice([1, 2, 4]), hkv=hkv, d=d,
                    n=d // 2 if rng.random() < 0.7 else d // 8, interleaved=rng.random() < 0.3,
                    unit=rng.random() < 0.3, fused=rng.random() < 0.4, weight=rng.choice([dtype, "f32"]),
                    places=rng.choice(["count", "packed", "far"]))
    if kind == "append":
        seqs = _log(rng, 1, 128)
        return dict(kind="append", dtype=half, seqs=seqs,
                    tokens=seqs if rng.random() < 0.5 else _log(rng, seqs, 8192),
                    held=_log(rng, 1, 2048), hq=hkv * rng.choice([1, 2, 4]), hkv=hkv, d=d,
                    n=d // 2 if rng.random() < 0.7 else d // 8, page=rng.choice([16, 16, 32, 64, 7]),
                    interleaved=rng.random() < 0.3, unit=rng.random() < 0.3, lay=rng.randrange(1 << 30))
    if kind == "shared":
        batch = _log(rng, 2, 128)
        return dict(kind="shared", dtype=half, batch=batch, groups=min(batch, rng.choice([1, 1, 2, 5, 9])),
                    prefix=_log(rng, 100, 16384), own=_log(rng, 1, 1024), hq=hkv * rng.choice([1, 2, 4, 8]),
                    hkv=hkv, d=d, page=rng.choice([16, 16, 32, 64]),
                    window=rng.choice([0, 0, 0, 1000, 5000]), idle=rng.choice([0, 0, 1]) if batch > 9 else 0,
                    lay=rng.randrange(1 << 30))
    if kind == "round":
        parents, samples = rng.choice([1, 3, 8, 16]), _log(rng, 1, 16)
        length = _log(rng, 20, 2000)
        return dict(kind="round", dtype=half, rows=parents * (1 + samples) + rng.randrange(40),
                    parents=parents, samples=samples, length=length, grow=_log(rng, 1, 100),
                    pages=parents * (length // 16 + 1) + parents * samples * 8 + _log(rng, 100, 4000),
                    page=rng.choice([16, 32, 64]), hkv=hkv, d=d, layers=rng.choice([1, 2, 4]),
                    lay=rng.randrange(1 << 30))
    rows, length = _log(rng, 4, 100), _log(rng, 50, 800)
    return dict(kind="compact", dtype=half, rows=rows, length=length,
                pages=rows * (length // 16 + 1) + _log(rng, 50, 1500), page=rng.choice([16, 16, 32]),
                hkv=hkv, d=d, layers=rng.choice([1, 2]), lay=rng.randrange(1 << 30))


# ------------------------------------------------------------------------------------------
# What a case's sequences look like
# ------------------------------------------------------------------------------------------

def _cut(rng, total, n, least):
    """``total`` in ``n`` parts of at least ``least``."""
    spare = total - n * least
    at = [0] + sorted(rng.randint(0, spare) for _ in range(n - 1)) + [spare]
    return [least + y - x for x, y in zip(at, at[1:])]


def _append_layout(case):
    """(tokens of each sequence in this call, its length after the call)"""
    rng = random.Random(case["lay"])
    new = _cut(rng, case["tokens"], case["seqs"], 1)
    return new, [n + rng.randint(case["held"] // 4, case["held"]) for n in new]


def _shared_layout(case):
    """(rows of each group, the groups' prefix lengths, the rows' lengths): the idle rows, of length
    0, come last and belong to no group."""
    rng = random.Random(case["lay"])
    live = case["batch"] - case["idle"]
    members = _cut(rng, live, min(case["groups"], live), 1)
    prefix = [case["prefix"] if len(members) == 1 else rng.randint(case["prefix"] // 4, case["prefix"])
              for _ in members]
    lengths = [p + rng.randint(min(case["own"], 1 + case["own"] // 8), case["own"])
               for p, m in zip(prefix, members) for _ in range(m)]
    return members, prefix, lengths + [0] * case["idle"]


def _round_layout(case):
    """(the parents' lengths): rows 0 .. parents - 1 of the table."""
    rng = random.Random(case["lay"])
    return [rng.randint(case["length"] // 2, case["length"]) for _ in range(case["parents"])]


def _compact_layout(case):
    """(the rows' lengths, the pages of the pool in the order that the rows take them): every fourth
    row is empty."""
    rng = random.Random(case["lay"])
    lengths = [0 if r % 4 == 3 else rng.randint(case["length"] // 2, case["length"])
               for r in range(case["rows"])]
    order = list(range(case["pages"]))
    rng.shuffle(order)
    return lengths, order


def _pages_of(length, page):
    return -(-length // page)


def _moved_pages(case):
    """How many pages of a pool compaction moves."""
    lengths, order = _compact_layout(case)
    n = sum(_pages_of(x, case["page"]) for x in lengths)
    return sum(1 for p in order[:n] if p >= n)


# ------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------

def _frequencies(n, device):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float().to(device)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape, dtype=DT[case["dtype"]]):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    def weight(d, unit, dtype):
        return ((0.0 if unit else 1.0) + 0.1 * randn(d, dtype=torch.float32)).to(DT[dtype])

    s = dict(case)
    kind = case["kind"]
    if kind in ("rotate", "rotate_grad"):
        b, t, hq, hkv, d = case["b"], case["t"], case["hq"], case["hkv"], case["d"]
        if case["fused"]:
            x = randn(b, t, hq + 2 * hkv, d)
            s["q"], s["k"] = x[:, :, :hq], x[:, :, hq:hq + hkv]
        else:
            s["q"], s["k"] = randn(b, t, hq, d), randn(b, t, hkv, d)
        if kind == "rotate_grad":
            s["gq"], s["gk"] = randn(b, t, hq, d), randn(b, t, hkv, d)
        s["wq"], s["wk"] = (weight(d, case["unit"], case["weight"]) for _ in range(2))
        s["freq"] = _frequencies(case["n"], "cuda")
        s["at"] = None
        if case["places"] == "packed":
            cuts = torch.randint(0, t, (1 + t // 1500,), generator=gen, device="cuda")
            starts = torch.zeros(t, dtype=torch.int64, device="cuda").index_fill_(0, cuts, 1)
            here = torch.arange(t, device="cuda")
            at = here - torch.cummax(here * starts, 0)[0]
            s["at"] = at.to(torch.int32).expand(b, t).contiguous()
        elif case["places"] == "far":
            s["at"] = torch.randint(0, 1 << 20, (b, t), generator=gen, device="cuda", dtype=torch.int32)
        return s
    if kind == "append":
        new, lengths = _append_layout(case)
        page, hq, hkv, d, n = case["page"], case["hq"], case["hkv"], case["d"], case["tokens"]
        each = [_pages_of(x, page) for x in lengths]
        s["table"] = _table(gen, each, sum(each) + 5)
        s["q"], s["k"], s["v"] = randn(n, hq, d), randn(n, hkv, d), randn(n, hkv, d)
        s["wq"], s["wk"] = (weight(d, case["unit"], case["dtype"]) for _ in range(2))
        s["freq"] = _frequencies(case["n"], "cuda")
        s["kp"], s["vp"] = (randn(sum(each) + 5, page, hkv, d) for _ in range(2))
        s["lengths"] = _i32(lengths)
        s["cu"] = None
        if case["tokens"] != case["seqs"]:
            s["cu"] = torch.cumsum(_i32([0] + new), 0, dtype=torch.int32)
        return s
    if kind == "shared":
        members, prefix, lengths = _shared_layout(case)
        page, b, hkv, d = case["page"], case["batch"], case["hkv"], case["d"]
        # the pages of each group's whole prefix pages, then each row's own
        shared = [p // page for p in prefix]
        of = [g for g, m in enumerate(members) for _ in range(m)]
        each = shared + [_pages_of(lengths[r], page) - shared[g] for r, g in enumerate(of)]
        rows = _table(gen, each, sum(each) + 5)
        table = torch.full((b, max(_pages_of(x, page) for x in lengths)), -1, dtype=torch.int32,
                           device="cuda")
        for r, g in enumerate(of):
            table[r, :shared[g]] = rows[g, :shared[g]]
            mine = rows[len(shared) + r, :each[len(shared) + r]]
            table[r, shared[g]:shared[g] + mine.numel()] = mine
        s["table"] = table
        s["q"] = randn(b, case["hq"], d)
        s["kp"], s["vp"] = (randn(sum(each) + 5, page, hkv, d) for _ in range(2))
        s["lengths"] = _i32(lengths)
        starts = [0]
        for m in members:
            starts.append(starts[-1] + m)
        # (a prefix that ends inside a page: its last page's rows are each sequence's own)
        s["groups"], s["prefix_lengths"] = _i32(starts), _i32([x * page for x in shared])
        s["most"] = (max(members), max(1, max(shared) * page), max([lengths[r] - shared[g] * page
                                                             for r, g in enumerate(of)]))
        return s
    page, rows = case["page"], case["rows"]
    s["pools"] = torch.stack([randn(case["pages"], page, case["hkv"], case["d"])
                              for _ in range(2 * case["layers"])])
    s["refcounts"] = torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
    if kind == "round":
        lengths = _round_layout(case)
        each = [_pages_of(x, page) for x in lengths]
        s["table"] = torch.full((rows, _pages_of(max(lengths) + case["grow"], page) + 3), -1,
                                dtype=torch.int32, device="cuda")
        held = _table(gen, each, case["pages"])
        s["table"][:len(each), :held.shape[1]] = held
        s["lengths"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["lengths"][:len(lengths)] = _i32(lengths)
        s["refcounts"][held[held >= 0].long()] = 1
        n = case["parents"]
        forks = n * case["samples"]
        # the children take the table's rows from its end
        s["parents"] = _i32([i % n for i in range(forks)])
        s["children"] = _i32([rows - 1 - i for i in range(forks)])
        want = [0] * rows
        for i in range(forks):
            want[rows - 1 - i] = lengths[i % n] + case["grow"]
        s["want"] = _i32(want)
        return s
    lengths, order = _compact_layout(case)
    each = [_pages_of(x, page) for x in lengths]
    table, at = [], 0
    for n in each:
        table.append(order[at:at + n] + [-1] * (max(each) - n))
        at += n
    s["table_from"], s["lengths"] = _i32(table), _i32(lengths)
    s["refcounts"][_i32(order[:at]).long()] = 1
    s["refcounts_from"] = s["refcounts"].clone()
    s["table"] = s["table_from"].clone()
    return s


def _table(gen, each, pages):
    """[rows, the most pages of a row] int32: ``each[r]`` pages of row ``r``, drawn without putting
    back, then -1."""
    taken = torch.randperm(pages, generator=gen, device="cuda")
    n = torch.tensor(each, device="cuda")
    j = torch.arange(max(each + [1]), device="cuda")
    at = (torch.cumsum(n, 0) - n)[:, None] + j
    return torch.where(j < n[:, None], taken[at.clamp(max=pages - 1)], -1).to(torch.int32)


# ------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------

def _turns(freq, at, interleaved):
    """cos and sin [..., 1, 2 n] of the positions ``at``, in the order of the rotated elements, and
    the sines' signs in it; the angles in 64 bits."""
    angle = at.double().unsqueeze(-1) * freq.double()
    c, s = angle.cos().float(), angle.sin().float()
    if interleaved:
        return c.repeat_interleave(2, -1).unsqueeze(-2), torch.stack((-s, s), -1).flatten(-2).unsqueeze(-2)
    return torch.cat((c, c), -1).unsqueeze(-2), torch.cat((-s, s), -1).unsqueeze(-2)


def _partner(x, interleaved):
    """Each rotated element's other one of its pair."""
    if interleaved:
        return x.unflatten(-1, (-1, 2)).flip(-1).flatten(-2)
    return torch.roll(x, x.shape[-1] // 2, -1)


def _rotate(y, turns, interleaved):
    c, s = turns
    r = c.shape[-1]
    x = y[..., :r]
    return torch.cat((x * c + _partner(x, interleaved) * s, y[..., r:]), -1)


def _norm_rope(x, w, turns, case):
    x = x.float()
    w = w.float() + 1 if case["unit"] else w.float()
    return _rotate(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w, turns,
                   case["interleaved"])


def _norm_rope_grad(x, w, z, turns, case):
    x = x.float()
    w = w.float() + 1 if case["unit"] else w.float()
    c, s = turns
    u = _rotate(z.float(), (c, -s), case["interleaved"])
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    g = u * w
    dx = r * (g - x * r.square() * (g * x).mean(-1, keepdim=True))
    return dx, (u * x * r).sum((0, 1, 2))


def _plain_rotate(s):
    at = s["at"] if s["at"] is not None else torch.arange(s["t"], device="cuda").expand(s["b"], -1)
    turns = _turns(s["freq"], at, s["interleaved"])
    q, k = s["q"], s["k"]
    if s["kind"] == "rotate":
        return (_norm_rope(q, s["wq"], turns, s).to(q.dtype), _norm_rope(k, s["wk"], turns, s).to(k.dtype))
    dq, dwq = _norm_rope_grad(q, s["wq"], s["gq"], turns, s)
    dk, dwk = _norm_rope_grad(k, s["wk"], s["gk"], turns, s)
    return dq.to(q.dtype), dk.to(k.dtype), dwq.to(s["wq"].dtype), dwk.to(s["wk"].dtype)


def _plain_append(s):
    token = torch.arange(s["tokens"], device="cuda")
    lengths = s["lengths"].long()
    if s["cu"] is None:
        seq, at = token, lengths - 1
    else:
        ends = s["cu"][1:].long()
        seq = torch.searchsorted(ends, token, right=True)
        at = lengths[seq] - ends[seq] + token
    turns = _turns(s["freq"], at, s["interleaved"])
    page, row = s["table"][seq, at // s["page"]].long(), at % s["page"]
    s["kp"][page, row] = _norm_rope(s["k"], s["wk"], turns, s).to(s["kp"].dtype)
    s["vp"][page, row] = s["v"]
    return _norm_rope(s["q"], s["wq"], turns, s).to(s["q"].dtype), s["kp"], s["vp"]


def _plain_shared(s):
    """The groups' prefixes gathered once for each group, padded to the largest, the rows' own keys
    for each row; one softmax over both."""
    b, hq, hkv, d, page = s["batch"], s["hq"], s["hkv"], s["d"], s["page"]
    most, prefix, mine = s["most"]
    rep, g = hq // hkv, s["groups"].numel() - 1
    starts, lengths = s["groups"].long(), s["lengths"].long()
    live = b - s["idle"]
    row = torch.arange(b, device="cuda")
    of = torch.searchsorted(starts[1:], row[:live], right=True)
    member = row[:live] - starts[of]
    start = torch.zeros_like(lengths)
    start[:live] = s["prefix_lengths"].long()[of]
    low = (lengths - 1 - s["window"]).clamp(min=0) if s["window"] else torch.zeros_like(lengths)

    def gather(pages, rows, first, n):
        at = first[:, None] + torch.arange(n, device="cuda")
        pg = s["table"][rows[:, None], (at // page).clamp(max=s["table"].shape[1] - 1)].long()
        return pages[pg.clamp(min=0), at % page].float().permute(0, 2, 1, 3), at  # [rows, Hkv, n, D]

    def weigh(scores, at, below):
        keep = (at < below[:, None]) & (at >= low[:scores.shape[0], None])
        return scores.masked_fill(~keep[:, None, None], -math.inf)

    def grouped(x):  # [G, Hkv, members x rep, ...] of each live row: [live, Hkv, rep, ...]
        return x.unflatten(2, (most, rep)).transpose(1, 2)[of, member]

    q = s["q"].float().view(b, hkv, rep, d) * (1.0 / math.sqrt(d))
    nothing = torch.zeros(g, dtype=torch.int64, device="cuda")
    first = starts[:-1]
    qg = torch.zeros(g, most, hkv, rep, d, device="cuda")
    qg[of, member] = q[:live]
    keys, at = gather(s["kp"], first, nothing, prefix)
    ps = torch.matmul(qg.transpose(1, 2).flatten(2, 3), keys.transpose(-1, -2))
    ps = weigh(grouped(ps), at[:1], torch.minimum(start, lengths)[:live])
    keys, at = gather(s["kp"], row, start, mine)
    os = weigh(torch.matmul(q, keys.transpose(-1, -2)), at, lengths)
    top = os.amax(-1, keepdim=True)
    top[:live] = torch.maximum(top[:live], ps.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    ps, os = (ps - top[:live]).exp(), (os - top).exp()
    total = os.sum(-1, keepdim=True)
    total[:live] += ps.sum(-1, keepdim=True)
    out = torch.matmul(os, gather(s["vp"], row, start, mine)[0])
    pg = torch.zeros(g, most, hkv, rep, prefix, device="cuda")
    pg[of, member] = ps
    values = gather(s["vp"], first, nothing, prefix)[0]
    out[:live] += grouped(torch.matmul(pg.transpose(1, 2).flatten(2, 3), values))
    out = out / torch.where(total > 0, total, 1.0)
    return out.reshape(b, hq, d).to(s["q"].dtype)


def _plain_round(s):
    pools, table, lengths, counts, page = s["pools"], s["table"], s["lengths"], s["refcounts"], s["page"]
    parents, children = s["parents"].long(), s["children"].long()
    j = torch.arange(table.shape[1], device="cuda")
    # fork: the parents' whole pages shared, a copy of the partly filled one
    held = lengths[parents].long()
    whole, rest = held // page, held % page
    free = (counts <= 0).nonzero()[:, 0]
    rank = (torch.cumsum(rest > 0, 0) - 1).clamp(min=0)
    made = (rest == 0) | (rank < free.numel())
    fresh = torch.where(made & (rest > 0), free[rank.clamp(max=free.numel() - 1)], torch.where(made, -1, -2))
    entries = torch.where(j < whole[:, None], table[parents].long(), -1)
    last = (j == whole[:, None]) & (fresh >= 0)[:, None]
    before = table[parents, whole.clamp(max=table.shape[1] - 1)].long().clamp(min=0)
    entries = torch.where(last, fresh[:, None], entries)
    take = (torch.arange(page, device="cuda") < rest[:, None])[..., None, None]
    to = fresh[fresh >= 0]
    pools[:, to] = torch.where(take[fresh >= 0], pools[:, before[fresh >= 0]], pools[:, to])
    table[children] = torch.where(made[:, None], entries, -1).to(torch.int32)
    lengths[children] = torch.where(made, held, 0).to(torch.int32)
    used = entries[made]
    counts.index_add_(0, used[used >= 0], torch.ones_like(used[used >= 0], dtype=torch.int32))
    # reserve: pages for the children's next tokens
    want = torch.maximum(s["want"], lengths).long()
    have = (lengths.long() + page - 1) // page
    need = (want + page - 1) // page - have
    fits = want <= table.shape[1] * page
    need = torch.where(fits, need, 0)
    free = (counts <= 0).nonzero()[:, 0]
    ends = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (ends <= free.numel()))
    k = j - have[:, None]
    place = granted[:, None] & (k >= 0) & (k < need[:, None])
    page_of = free[((ends - need)[:, None] + k).clamp(0, free.numel() - 1)]
    table.copy_(torch.where(place, page_of, table))
    counts[page_of[place]] = 1
    lengths.copy_(torch.where(granted, want, lengths))
    # free: the children end
    used = (j < ((lengths[children].long() + page - 1) // page)[:, None])
    gone = table[children][used].long()
    counts.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    table[children] = torch.where(used, -1, table[children])
    lengths[children] = 0
    return fresh.to(torch.int32), granted, table, lengths, counts, pools


def _plain_compact(s):
    pools, table, lengths, counts, page = s["pools"], s["table"], s["lengths"], s["refcounts"], s["page"]
    live = counts > 0
    n = live.sum()
    index = torch.arange(counts.numel(), device="cuda")
    to = (~live & (index < n)).nonzero()[:, 0]
    src = (live & (index >= n)).nonzero()[:, 0]
    moved = torch.where(live, index, -1)
    moved[src] = to
    pools[:, to] = pools[:, src]
    counts[to] = counts[src]
    counts[src] = 0
    used = torch.arange(table.shape[1], device="cuda") < ((lengths.long() + page - 1) // page)[:, None]
    table.copy_(torch.where(used, moved[table.long().clamp(min=0)], table))
    return moved.to(torch.int32), table, counts, pools


def run(s):
    kind = s["kind"]
    if kind == "compact":
        # the pool as it was found; its pages still hold what the rows below move
        s["table"].copy_(s["table_from"])
        s["refcounts"].copy_(s["refcounts_from"])
    if not own:
        return {"rotate": _plain_rotate, "rotate_grad": _plain_rotate, "append": _plain_append,
                "shared": _plain_shared, "round": _plain_round, "compact": _plain_compact}[kind](s)
    import dashmag_amd as dm
    if kind in ("rotate", "rotate_grad", "append"):
        options = dm.QkNormRopeOptions(interleaved=s["interleaved"], unit_offset=s["unit"])
        if kind == "rotate":
            return dm.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["freq"], s["at"], options)
        if kind == "rotate_grad":
            return dm.qk_norm_rope_backward(s["q"], s["k"], s["wq"], s["wk"], s["freq"], s["gq"], s["gk"],
                                            s["at"], options)
        q = dm.qk_norm_rope_paged(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["freq"], s["kp"], s["vp"],
                                  s["table"], s["lengths"], s["cu"], options)
        return q, s["kp"], s["vp"]
    if kind == "shared":
        options = dm.AttentionOptions(window=dm.Window(s["window"], 0) if s["window"] else None)
        return dm.attention_decode_shared(s["q"], s["kp"], s["vp"], s["table"], s["lengths"], s["groups"],
                                          s["prefix_lengths"], options)
    pools, table, lengths, counts = list(s["pools"].unbind(0)), s["table"], s["lengths"], s["refcounts"]
    if kind == "round":
        fresh = dm.cache_fork(pools, table, lengths, counts, s["parents"], s["children"])
        granted = dm.cache_reserve(table, lengths, counts, s["want"], s["page"])
        dm.cache_free(table, lengths, counts, s["children"], s["page"])
        return fresh, granted, table, lengths, counts, s["pools"]
    moved = dm.cache_compact(pools, table, lengths, counts)
    return moved, table, counts, s["pools"]


# ------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------

def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind in ("rotate", "rotate_grad"):
        x = case["b"] * case["t"] * (case["hq"] + case["hkv"]) * case["d"]
        places = 0 if case["places"] == "count" else 4 * case["b"] * case["t"]
        if kind == "rotate":
            return {"bytes": 2 * x * e + places, "flops": 8 * x}
        return {"bytes": 3 * x * e + places, "flops": 16 * x}
    if kind == "append":
        x = case["tokens"] * (case["hq"] + case["hkv"]) * case["d"]
        v = case["tokens"] * case["hkv"] * case["d"]
        return {"bytes": 2 * (x + v) * e + 4 * case["tokens"], "flops": 8 * x}
    if kind == "shared":
        members, prefix, lengths = _shared_layout(case)
        page, window = case["page"], case["window"]
        keys = seen = at = 0
        for m, p in zip(members, prefix):
            p = p // page * page
            low = [max(0, x - 1 - window) if window else 0 for x in lengths[at:at + m]]
            keys += max(0, p - min(low)) + sum(x - max(p, y) for x, y in zip(lengths[at:at + m], low))
            seen += sum(x - y for x, y in zip(lengths[at:at + m], low))
            at += m
        q = case["batch"] * case["hq"] * case["d"]
        return {"bytes": 2 * keys * case["hkv"] * case["d"] * e + 2 * q * e + 4 * keys // page,
                "flops": 4 * seen * case["hq"] * case["d"]}
    row = case["hkv"] * case["d"] * e * 2 * case["layers"]  # one token's bytes in every pool
    if kind == "round":
        lengths, page = _round_layout(case), case["page"]
        forks = case["samples"]
        copied = forks * sum(x % page for x in lengths)
        pages = forks * sum(_pages_of(x + case["grow"], page) for x in lengths)
        # the rows' copies; the table entries read, written, read again and cleared with their
        # counts; the counts looked through for free pages
        return {"bytes": 2 * copied * row + 24 * pages + 4 * case["pages"] + 8 * case["rows"], "flops": 0}
    lengths, _ = _compact_layout(case)
    pages = sum(_pages_of(x, case["page"]) for x in lengths)
    return {"bytes": 2 * _moved_pages(case) * case["page"] * row + 12 * case["pages"] + 8 * pages, "flops": 0}


# ------------------------------------------------------------------------------------------
# In 64 bits, from the definitions
# ------------------------------------------------------------------------------------------

def _pairs(n, interleaved):
    """The first and second elements of the n rotated pairs."""
    i = torch.arange(n, device="cuda")
    return (2 * i, 2 * i + 1) if interleaved else (i, i + n)


def _exact_head(x, w, freq, at, case, z=None):
    """One tensor [tokens, heads, D] normalised and rotated at the positions ``at``; with the gradient
    ``z`` of that, the gradients of x and w."""
    x, w = x.double(), w.double() + (1.0 if case["unit"] else 0.0)
    a, b = _pairs(freq.numel(), case["interleaved"])
    angle = at.double()[:, None, None] * freq.double()
    c, s = torch.cos(angle), torch.sin(angle)
    scale = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6)
    if z is None:
        y = x * scale * w
        out = y.clone()
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., a] * s + y[..., b] * c
        return out
    z = z.double()
    u = z.clone()
    u[..., a] = z[..., a] * c + z[..., b] * s
    u[..., b] = z[..., b] * c - z[..., a] * s
    dw = (u * x * scale).flatten(0, 1).sum(0)
    h = x * scale
    gh = u * w
    return (gh - h * (gh * h).sum(-1, keepdim=True) / x.shape[-1]) * scale, dw


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("rotate", "rotate_grad"):
        b, t = case["b"], case["t"]
        at = torch.arange(t, device="cuda").repeat(b) if s["at"] is None else s["at"].reshape(-1)
        if kind == "rotate":
            return tuple(_exact_head(s[x].flatten(0, 1), s["w" + x], s["freq"], at, case).unflatten(0, (b, t))
                         for x in "qk")
        (dq, dwq), (dk, dwk) = (_exact_head(s[x].flatten(0, 1), s["w" + x], s["freq"], at, case,
                                            s["g" + x].flatten(0, 1)) for x in "qk")
        return dq.unflatten(0, (b, t)), dk.unflatten(0, (b, t)), dwq, dwk
    if kind == "append":
        new, lengths = _append_layout(case)
        at = torch.cat([torch.arange(x - n, x) for n, x in zip(new, lengths)]).cuda()
        seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
        kp, vp = s["kp"].double(), s["vp"].double()
        slot = s["table"][seq, at // case["page"]].long() * case["page"] + at % case["page"]
        kp.flatten(0, 1)[slot] = _exact_head(s["k"], s["wk"], s["freq"], at, case)
        vp.flatten(0, 1)[slot] = s["v"].double()
        return _exact_head(s["q"], s["wq"], s["freq"], at, case), kp, vp
    if kind == "shared":
        _, _, lengths = _shared_layout(case)
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        rep = case["hq"] // case["hkv"]
        for r, n in enumerate(lengths):
            lo = max(0, n - 1 - case["window"]) if case["window"] else 0
            if n <= lo:
                continue
            j = torch.arange(lo, n, device="cuda")
            slot = s["table"][r, j // case["page"]].long() * case["page"] + j % case["page"]
            k, v = (s[x].flatten(0, 1)[slot].double().transpose(0, 1) for x in ("kp", "vp"))
            q = s["q"][r].double().view(case["hkv"], rep, case["d"])
            p = torch.softmax(torch.matmul(q, k.transpose(1, 2)) / math.sqrt(case["d"]), -1)
            out[r] = torch.matmul(p, v).reshape(case["hq"], case["d"])
        return out
    pools, page = s["pools"], case["page"]
    counts, lengths = s["refcounts"].tolist(), s["lengths"].tolist()
    table = s["table"].tolist()
    if kind == "round":
        fresh, granted = [], []
        for p, c in zip(s["parents"].tolist(), s["children"].tolist()):
            whole, rest = divmod(lengths[p], page)
            new = -1
            if rest:
                new = counts.index(0)
                pools[:, new, :rest] = pools[:, table[p][whole], :rest]
                counts[new] = 1
                table[c][whole] = new
            for x in range(whole):
                table[c][x] = table[p][x]
                counts[table[p][x]] += 1
            lengths[c] = lengths[p]
            fresh.append(new)
        for r, n in enumerate(s["want"].tolist()):
            granted.append(True)
            for x in range(_pages_of(lengths[r], page), _pages_of(n, page)):
                table[r][x] = counts.index(0)
                counts[table[r][x]] = 1
            lengths[r] = max(lengths[r], n)
        for c in s["children"].tolist():
            for x in range(_pages_of(lengths[c], page)):
                counts[table[c][x]] -= 1
                table[c][x] = -1
            lengths[c] = 0
        return (_i32(fresh), torch.tensor(granted).cuda(), _i32(table), _i32(lengths), _i32(counts),
                pools.double())
    n = sum(x > 0 for x in counts)
    moved = [x if counts[x] > 0 else -1 for x in range(len(counts))]
    holes = [x for x in range(n) if counts[x] == 0]
    late = [x for x in range(n, len(counts)) if counts[x] > 0]
    for x, y in zip(late, holes):
        pools[:, y] = pools[:, x]
        moved[x], counts[y], counts[x] = y, counts[x], 0
    for r, x in enumerate(lengths):
        for i in range(_pages_of(x, page)):
            table[r][i] = moved[table[r][i]]
    return _i32(moved), _i32(table), _i32(counts), pools.double()
