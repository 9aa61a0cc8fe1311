"""Plain models of the paged cache for its tests: the page bookkeeping on
Python lists, and attention in 64 bits over rows gathered position by position."""
import numpy as np


class Refused(Exception):
    pass


class PageModel:
    """table / length / refs and the rows of one cache, changed as
    include/kestrel_cuda.h describes. rows[(layer, page)] is [n_kv, page, hd]."""

    def __init__(self, n_layer, n_pages, page, n_kv, hd, n_seq, max_pages, k, v):
        self.n_layer, self.n_pages, self.page = n_layer, n_pages, page
        self.n_seq, self.max_pages = n_seq, max_pages
        self.table = [[-1] * max_pages for _ in range(n_seq)]
        self.length = [0] * n_seq
        self.refs = [0] * n_pages
        self.k, self.v = k.copy(), v.copy()  # [n_layer, n_pages, n_kv, page, hd]

    def held(self, n):
        return -(-n // self.page)

    def fork(self, src, dst):
        for i, (s, d) in enumerate(zip(src, dst)):
            if not (0 <= s < self.n_seq and 0 <= d < self.n_seq) or d in src or s in dst or d in dst[:i] \
                    or self.length[d]:
                raise Refused
        for s, d in zip(src, dst):
            self.table[d], self.length[d] = list(self.table[s]), self.length[s]
            for p in self.table[d][:self.held(self.length[d])]:
                self.refs[p] += 1

    def free(self, seqs, keep=None):
        for i, s in enumerate(seqs):
            n = min(self.length[s], keep[i] if keep is not None else 0)
            for j in range(self.held(n), self.held(self.length[s])):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.length[s] = n

    def extend(self, seqs, n_new):
        if len(set(seqs)) < len(seqs) or any(a < 0 for a in n_new):
            raise Refused
        if any(self.length[s] + a > self.max_pages * self.page for s, a in zip(seqs, n_new)):
            raise Refused
        plan, refs = [], list(self.refs)
        for s, a in zip(seqs, n_new):
            n = self.length[s]
            copy = False
            if a and n % self.page:
                p = self.table[s][n // self.page]
                copy = refs[p] > 1
                refs[p] -= copy
            plan.append((copy, self.held(n + a) - self.held(n) + copy))
        free = [p for p in range(self.n_pages) if self.refs[p] == 0]
        if sum(c for _, c in plan) > len(free):
            raise Refused
        for (s, a), (copy, count) in zip(zip(seqs, n_new), plan):
            n = self.length[s]
            take, free = free[:count], free[count:]
            if copy:
                j, r = n // self.page, n % self.page
                old = self.table[s][j]
                self.refs[old] -= 1
                for x in (self.k, self.v):
                    x[:, take[0], :, :r] = x[:, old, :, :r]
            col = self.held(n + a) - count
            for t, p in enumerate(take):
                self.table[s][col + t] = p
                self.refs[p] = 1
            self.length[s] = n + a

    def write(self, layer, seqs, counts, k, v):
        r = 0
        for s, c in zip(seqs, counts):
            for i in range(c):
                pos = self.length[s] - c + i
                p = self.table[s][pos // self.page]
                self.k[layer, p, :, pos % self.page] = k[r]
                self.v[layer, p, :, pos % self.page] = v[r]
                r += 1

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        moving = [p for p in range(live, self.n_pages) if self.refs[p] > 0]
        to = dict(zip(moving, holes))
        for a, b in to.items():
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return live

    def check(self):
        """Every page's refs are the sequences that hold it."""
        held = [0] * self.n_pages
        for s in range(self.n_seq):
            for j, p in enumerate(self.table[s]):
                assert (p >= 0) == (j < self.held(self.length[s]))
                if p >= 0:
                    held[p] += 1
        assert held == self.refs

    def rows(self, layer, s):
        """(k, v) of sequence s's positions, [len, n_kv, hd]."""
        pos = range(self.length[s])
        get = lambda x: np.stack([x[layer, self.table[s][j // self.page], :, j % self.page] for j in pos]) \
            if self.length[s] else np.zeros((0,) + x.shape[2:3] + x.shape[4:])
        return get(self.k), get(self.v)


def attention(q, k, v, first, scale, window=0, sinks=0):
    """64-bit attention of q [rows, n_head, hd] at positions first, first + 1,
    ... over k, v [len, n_kv, hd]: only what a row sees is touched."""
    rows, nh, hd = q.shape
    nkv = k.shape[1]
    out = np.zeros((rows, nh, hd))
    for r in range(rows):
        i = first + r
        see = [j for j in range(min(i + 1, len(k))) if not window or j > i - window or j < sinks]
        if i < 0 or not see:
            continue
        kk, vv = k[see].astype(np.float64), v[see].astype(np.float64)
        for h in range(nh):
            s = scale * (kk[:, h // (nh // nkv)] @ q[r, h].astype(np.float64))
            p = np.exp(s - s.max())
            out[r, h] = p @ vv[:, h // (nh // nkv)] / p.sum()
    return out
