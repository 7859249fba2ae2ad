"""The eviction of keys, one row and one key after another: what the device's operation has to give, to the
bit. A row's keys are told by their weights (a list a row), NaN above all."""
import math

from pages_oracle import Cache, pages


class Evicting(Cache):
    def __init__(self, *args, weights=()):
        super().__init__(*args)
        self.weights = [list(w) for w in weights]

    def evict(self, budgets, recent):
        kept, before = [], list(self.counts)
        for r, budget in enumerate(budgets):
            held, budget, page, row = self.keys(r), max(budget, 0), self.page, self.table[r]
            out = [-1] * (self.cols * page)
            kept.append(out)
            out[:held] = range(held)
            if held <= budget:
                continue
            fixed = max([0] + [(c + 1) * page for c in range(pages(held, page))
                               if 0 <= row[c] < len(before) and before[row[c]] > 1])
            w = self.weights[r]
            must = {j for j in range(held) if j < fixed or j >= held - min(recent, budget)}
            rest = sorted((j for j in range(held) if j not in must),
                          key=lambda j: (0, 0, j) if math.isnan(w[j]) else (1, -w[j], j))
            keep = sorted(must | set(rest[:max(0, budget - len(must))]))
            if len(keep) == held:
                continue
            for to, j in enumerate(keep):
                p, q = row[j // page], row[to // page]
                if 0 <= p < len(before) and 0 <= q < len(before):
                    for x in self.pools:
                        x[q, to % page] = x[p, j % page]
            out[:] = keep + [-1] * (len(out) - len(keep))
            w[:held] = [w[j] for j in keep] + [0.0] * (held - len(keep))
            for c in range(pages(len(keep), page), pages(held, page)):
                if 0 <= row[c] < len(before):
                    self.counts[row[c]] -= 1
                row[c] = -1
            self.lengths[r] = len(keep)
        return kept
