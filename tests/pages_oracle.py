"""The pages of a cache, one row and one page after another: what the device's operations have to give,
to the bit. Tables are lists of lists, pools numpy arrays [P, page_size, ...]."""


def pages(n, page):
    return -(-n // page)


class Cache:
    def __init__(self, table, lengths, counts, page, pools=()):
        self.table, self.lengths = [list(r) for r in table], list(lengths)
        self.counts, self.page, self.pools = list(counts), page, [p.copy() for p in pools]
        self.cols = len(table[0]) if table else 0

    def keys(self, r):
        return max(0, min(self.lengths[r], self.cols * self.page))

    def _free(self):
        return [p for p, c in enumerate(self.counts) if c <= 0]

    def reserve(self, new):
        free, granted, short = self._free(), [], False
        for r, n in enumerate(new):
            have = pages(self.keys(r), self.page)
            if n > self.cols * self.page:
                granted.append(False)
                continue
            need = max(0, pages(n, self.page) - have) if n > self.keys(r) else 0
            if need and (short or need > len(free)):
                short = True
                granted.append(False)
                continue
            for i in range(need):
                p = free.pop(0)
                self.table[r][have + i], self.counts[p] = p, 1
            if n > self.keys(r):
                self.lengths[r] = n
            granted.append(True)
        return granted

    def fork(self, parents, children):
        free, fresh, short, named = self._free(), [], False, set()
        before, rows = [self.keys(r) for r in range(len(self.table))], [list(r) for r in self.table]
        empty = [x <= 0 for x in self.lengths]
        for p, c in zip(parents, children):
            ok = 0 <= p < len(rows) and 0 <= c < len(rows) and empty[c] and c not in named
            named.add(c)
            if not ok:
                fresh.append(-2)
                continue
            whole, rest = divmod(before[p], self.page)
            own = -1
            if rest:
                if short or not free:
                    short = True
                    fresh.append(-2)
                    continue
                own = free.pop(0)
                self.counts[own] = 1
                self.table[c][whole] = own
                if 0 <= rows[p][whole] < len(self.counts):
                    for x in self.pools:
                        x[own, :rest] = x[rows[p][whole], :rest]
            for j in range(whole):
                self.table[c][j] = rows[p][j]
                if 0 <= rows[p][j] < len(self.counts):
                    self.counts[rows[p][j]] += 1
            self.lengths[c] = before[p]
            fresh.append(own)
        return fresh

    def free(self, rows):
        for r in rows:
            if not 0 <= r < len(self.table):
                continue
            for j in range(pages(self.keys(r), self.page)):
                p = self.table[r][j]
                self.table[r][j] = -1
                if 0 <= p < len(self.counts):
                    self.counts[p] -= 1
            self.lengths[r] = 0

    def compact(self):
        n = sum(c > 0 for c in self.counts)
        moved = [p if c > 0 else -1 for p, c in enumerate(self.counts)]
        holes = [p for p in range(n) if self.counts[p] <= 0]
        for p in range(n, len(self.counts)):
            if self.counts[p] > 0:
                to = holes.pop(0)
                moved[p], self.counts[to], self.counts[p] = to, self.counts[p], 0
                for x in self.pools:
                    x[to] = x[p]
        for r, row in enumerate(self.table):
            for j in range(pages(self.keys(r), self.page)):
                if 0 <= row[j] < len(moved):
                    row[j] = moved[row[j]]
        return moved
