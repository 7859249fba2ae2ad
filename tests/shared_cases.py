"""Batches whose rows share prefixes, in pages, with the decode's result in 64 bits and what an output
may be off by.

A row's output is sum p_j v_j / sum p_j. With u = 2^-24: a score's products are summed in f32 over D
terms, scaled and taken against a reference: off by at most (D + 16) u S, S the largest scale sum |q k|
of the row; a weight is e^ of it, off by that and 4 u, and (16-bit inputs) rounded once for its
product with the values, half a step of the type; the sums' chains are at most a sixteenth of the keys and
64 long. So an output is off by at most (half step + 2 (D + 16) u S + 2 (keys / 16 + 64) u) A, A = sum p |v| /
sum p; f16 weights below the smallest normal lose 2^-25 each of a sum of at least 1. Then it is
rounded once."""
import torch

U = 2.0 ** -24


class Batch:
    """groups: (first row, [rows' lengths], prefix length) of each, rows in between and behind share
    nothing; lone: {row: length}. Pages that no row sees and rows behind the lengths hold NaN."""

    def __init__(self, dtype, d, hkv, rep, page, groups, lone, rows, seed, window=None, ahead=False, scale=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.window, self.d, self.page = window, d, page
        lengths = [0] * rows
        for first, lens, _ in groups:
            for i, x in enumerate(lens):
                lengths[first + i] = x
        for r, x in lone.items():
            lengths[r] = x
        cols = max(1, max(-(-x // page) for x in lengths) + 1)
        need = sum(-(-x // page) for x in lengths) + sum(-(-p // page) for _, _, p in groups) + 3
        order = torch.randperm(need, generator=gen).tolist()
        k, v = (torch.full((need, page, hkv, d), float("nan")).to(dtype) for _ in range(2))
        table = torch.full((rows, cols), -1, dtype=torch.int32)
        prefix_of = {}
        for first, lens, p in groups:
            pk, pv = (torch.randn(p, hkv, d, generator=gen).to(dtype) for _ in range(2))
            whole = [order.pop() for _ in range(p // page)]
            for i, x in enumerate(lens):
                prefix_of[first + i] = (p, pk, pv, whole)
        self.keys = []
        for r, x in enumerate(lengths):
            p, pk, pv, whole = prefix_of.get(r, (0, None, None, []))
            dk, dv = (torch.randn(x, hkv, d, generator=gen).to(dtype) for _ in range(2))
            if p:
                dk[:p], dv[:p] = pk[:x], pv[:x]
            low = max(0, x - 1 - window) if window is not None else 0
            for c in range(-(-x // page)):
                pg = whole[c] if c < len(whole) else order.pop()
                table[r, c] = pg
                # (the prefix's last keys, on a page of the row's own, are read through the longest row)
                a = max(c * page, low if not len(whole) <= c < -(-p // page) else 0)
                b = min((c + 1) * page, x)
                if a < b:
                    k[pg, a - c * page:b - c * page] = dk[a:b]
                    v[pg, a - c * page:b - c * page] = dv[a:b]
            self.keys.append((dk, dv, low))
        self.q = (scale * torch.randn(rows, hkv * rep, d, generator=gen)).to(dtype)
        self.k, self.v, self.table = k, v, table
        self.lengths = torch.tensor(lengths, dtype=torch.int32)
        cut, pl, at = [groups[0][0] if groups else 0], [], 0
        for first, lens, p in groups:
            if first != cut[-1]:  # rows in between: a group without a prefix
                cut.append(first), pl.append(0)
            cut.append(first + len(lens)), pl.append(p)
        self.groups, self.prefix = (torch.tensor(x, dtype=torch.int32) for x in (cut, pl))

    def want(self, scale=None):
        """(output, bound) [rows, Hq, D] in 64 bits, before rounding."""
        q = self.q.double()
        out, bound = torch.zeros_like(q), torch.zeros_like(q)
        scale = self.d ** -0.5 if scale is None else scale
        dt = self.q.dtype
        for r, (k, v, low) in enumerate(self.keys):
            k, v = (x[low:].double().transpose(0, 1) for x in (k, v))  # [Hkv, n, D]
            n = k.shape[1]
            if n == 0:
                continue
            x = q[r].unflatten(0, (k.shape[0], -1))
            p = torch.softmax(x @ k.transpose(1, 2) * scale, -1)
            out[r] = (p @ v).flatten(0, 1)
            big = (p @ v.abs()).flatten(0, 1)
            s = (x.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True).flatten(0, 1) * abs(scale)
            half = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
            bound[r] = (half + 2 * (self.d + 16) * U * s + 2 * (n / 16 + 64) * U) * big
            if dt == torch.float16:
                bound[r] += 2.0 ** -25 * v.abs().sum(1, keepdim=True).expand(-1, x.shape[1], -1).flatten(0, 1)
        return out, bound

    def cuda(self):
        return [x.cuda() for x in (self.q, self.k, self.v, self.table, self.lengths, self.groups, self.prefix)]
