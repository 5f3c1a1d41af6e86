"""A page pool in plain Python, one entry after the other, for the tests."""
import numpy as np


class Pool:
    """refs as a list; content[p] stands for what page p's bytes are."""

    def __init__(self, n_pages, page):
        self.n, self.page, self.refs, self.short = n_pages, page, np.zeros(n_pages, np.int64), 0
        self.content = np.arange(n_pages)

    def lowest(self, taken):
        for p in range(self.n):
            if self.refs[p] == 0 and p not in taken:
                return p
        self.short += 1
        return -1

    def reserve(self, table, start, lens):
        """Pages of the newest start[b+1] - start[b] tokens of each sequence."""
        for b in range(len(lens)):
            n = start[b + 1] - start[b]
            for p in range(table.shape[1]):
                holds_new = any(x // self.page == p for x in range(max(lens[b] - n, 0), max(lens[b], 0)))
                if holds_new and not 0 <= table[b, p] < self.n:
                    table[b, p] = self.lowest(())
                    if table[b, p] >= 0:
                        self.refs[table[b, p]] = 1

    def fork(self, table, lens, parents, width=None):
        width = table.shape[1] if width is None else width
        out, out_lens, taken = np.full((len(parents), width), -1), np.zeros(len(parents), int), {}
        shared = np.zeros_like(self.refs)
        for i, j in enumerate(parents):
            if not 0 <= j < len(table):
                continue
            n = out_lens[i] = min(max(lens[j], 0), table.shape[1] * self.page)
            for p in range(min(width, -(-n // self.page))):
                old = table[j, p]
                if not 0 <= old < self.n:
                    continue
                if (p + 1) * self.page <= n:
                    out[i, p] = old
                    shared[old] += 1
                else:
                    new = self.lowest(taken)
                    if new >= 0:
                        taken[new] = old
                    out[i, p] = new
        for new, old in taken.items():
            self.refs[new] = 1
            self.content[new] = self.content[old]
        self.refs += shared
        return out, out_lens

    def free(self, table):
        for e in np.ndindex(table.shape):
            p = table[e]
            if 0 <= p < self.n:
                self.refs[p] = max(self.refs[p] - 1, 0)
            table[e] = -1

    def compact(self, *tables):
        live = [p for p in range(self.n) if self.refs[p] > 0]
        high = [p for p in live if p >= len(live)]
        low = [p for p in range(len(live)) if self.refs[p] <= 0]
        to = dict(zip(high, low))
        for t in tables:
            for e in np.ndindex(t.shape):
                if len(live) <= t[e] < self.n:
                    t[e] = to.get(t[e], -1)
        for s, d in to.items():
            self.content[d], self.refs[d], self.refs[s] = self.content[s], self.refs[s], 0
        return len(live)
