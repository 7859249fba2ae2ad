"""Ragged batches of new tokens over a paged cache, with their attention in 64 bits and what each result
may be off by.

With u = 2^-24 a score's products are summed in f32 over D terms, scaled and taken against a reference: off by
at most E = (D + 16) u S, S the largest scale sum |q k| of the row. A softmax weight is e^ of it, off by that
and 4 u, its sums' chains at most a sixteenth of the n keys and 64 long, and for 16-bit inputs it is
rounded once for its product with the values, half a step of the type; so an output is off by at most
(half step + 2 E + 2 (n / 16 + 64) u) A, A = sum p |v|; f16 weights below the smallest normal lose 2^-25 each of a
sum of at least 1. The log-sum-exp is off by at most G = E + (n / 16 + 64) u + 8 u (|lse| + 1). A key's weight is a
sum of f32 weights e^(score - lse), each off by (E + G + 8 u) of itself (the score is not rounded to fewer bits), over
R rows in chains of at most R, and is added to what was there: sum p (E + G + (R + 40) u) + u |result|."""
import torch

from shared_cases import U


class Chunks:
    """seqs: (new tokens, keys with them) of each sequence; gaps: tokens in front of the first sequence and
    behind the last that belong to none. Cache rows that no token sees hold NaN, and so do the tokens' that see
    none."""

    def __init__(self, dtype, d, hkv, rep, page, seqs, seed, window=None, gaps=(0, 0), scale=1.0, single=False,
                 spare=3, extra=2):
        gen = torch.Generator().manual_seed(seed)
        self.window, self.d, self.page, self.rep, self.seqs, self.gaps = window, d, page, rep, seqs, gaps
        cols = max([-(-x // page) for _, x in seqs] + [0]) + extra
        need = sum(-(-x // page) for _, x in seqs) + spare
        order = torch.randperm(need, generator=gen).tolist()
        self.k, self.v = (torch.full((need, page, hkv, d), float("nan")).to(dtype) for _ in range(2))
        self.table = torch.full((len(seqs), cols), -1, dtype=torch.int32)
        self.keys = []
        for r, (n, x) in enumerate(seqs):
            k, v = (torch.randn(x, hkv, d, generator=gen).to(dtype) for _ in range(2))
            low = max(0, x - n - window) if window is not None else 0
            for c in range(-(-x // page)):
                pg = order.pop()
                self.table[r, c] = pg
                a, b = max(c * page, low), min((c + 1) * page, x)
                if n and a < b:
                    self.k[pg, a - c * page:b - c * page] = k[a:b]
                    self.v[pg, a - c * page:b - c * page] = v[a:b]
            self.keys.append((k, v))
        total = gaps[0] + sum(n for n, _ in seqs) + gaps[1]
        self.q = (scale * torch.randn(total, hkv * rep, d, generator=gen)).to(dtype)
        self.lengths = torch.tensor([x for _, x in seqs], dtype=torch.int32)
        cu = [gaps[0]]
        for n, _ in seqs:
            cu.append(cu[-1] + n)
        self.cu = None if single else torch.tensor(cu, dtype=torch.int32)
        self.start = cu
        self.weights = torch.rand(len(seqs), cols * page, generator=gen)

    def want(self, scale=None):
        """{"out", "lse", "weights"}: (result, bound) in 64 bits, before rounding."""
        dt, d = self.q.dtype, self.d
        scale = d ** -0.5 if scale is None else scale
        half = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        lse = torch.full(self.q.shape[:2], -torch.inf, dtype=torch.float64)
        off, loff = torch.zeros_like(out), torch.zeros_like(lse)
        w, woff = self.weights.double(), torch.zeros(self.weights.shape, dtype=torch.float64)
        for r, (n, x) in enumerate(self.seqs):
            k, v = (y.double().transpose(0, 1) for y in self.keys[r])  # [Hkv, x, D]
            if n == 0 or x == 0:
                continue
            at = slice(self.start[r], self.start[r] + n)
            pos = torch.arange(x - n, x)
            seen = torch.arange(x) <= pos[:, None]
            if self.window is not None:
                seen &= torch.arange(x) >= pos[:, None] - self.window
            any_ = seen.any(1)
            q = self.q[at].double().unflatten(1, (k.shape[0], self.rep)).permute(1, 2, 0, 3)  # [Hkv, rep, n, D]
            z = (q @ k.transpose(1, 2)[:, None] * scale).masked_fill(~seen, -torch.inf)
            total = torch.logsumexp(z, -1, keepdim=True)
            p = torch.where(seen, torch.exp(z - total), 0.0)
            p = torch.where(any_[:, None], p, 0.0)
            o, big = p @ v[:, None], p @ v[:, None].abs()
            s = ((q.abs() @ k.abs().transpose(1, 2)[:, None]) * abs(scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            e = (d + 16) * U * s
            back = lambda y: y.permute(2, 0, 1, 3).flatten(1, 2)  # noqa: E731
            out[at], lse[at] = back(o), back(total)[..., 0]
            bound = (half + 2 * e + 2 * (x / 16 + 64) * U) * big
            if dt == torch.float16:
                bound = bound + 2.0 ** -25 * seen.double() @ v[:, None].abs()
            g = e + (x / 16 + 64) * U + 8 * U * (torch.where(any_[:, None], total, 0.0).abs() + 1)
            off[at], loff[at] = back(bound), back(g)[..., 0]
            w[r, :x] += p.sum((0, 1, 2))
            woff[r, :x] = (p * (e + g + (p.shape[0] * p.shape[1] * n + 40) * U)).sum((0, 1, 2))
        return {"out": (out, off), "lse": (lse, loff), "weights": (w, woff + U * w)}

    def cuda(self):
        return [x if x is None else x.cuda() for x in (self.q, self.k, self.v, self.table, self.lengths, self.cu)]


def held_lse(name, got, want, bound):
    """As rope_cases.held, and -inf where the log-sum-exp of no key is."""
    got = got.cpu().double()
    none = want == -torch.inf
    assert torch.equal(got == -torch.inf, none), name
    off = torch.where(none, 0.0, (got - torch.where(none, 0.0, want)).abs())
    worst = float((off / bound.clamp(min=1e-300)).max()) if off.numel() else 0.0
    print(f"{name}: {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, (name, worst)
