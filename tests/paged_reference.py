"""The paged cache's operators (append, attention, accept) from their definitions, in 64 bits, request by request."""
import math

import numpy as np

D = 128


class Step:
    """A step's requests: `lengths` tokens cached, `parents` per request (a list for each; None: a chain of `rows`),
    pages in random order over a pool with a few that belong to nobody."""

    def __init__(self, rng, page, lengths, rows, trees=None, pad=0, spare=3, extra_ld=1):
        self.page, self.lengths, self.rows = page, list(lengths), list(rows)
        self.trees = trees
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int64)
        self.total = int(self.start[-1]) + pad
        need = [-(-(n + t) // page) for n, t in zip(lengths, rows)]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(need), max(need + [0]) + extra_ld), -7, np.int64)
        at = 0
        for s, m in enumerate(need):
            self.table[s, :m] = order[at:at + m]
            at += m

    def parents(self, s):
        return list(range(-1, self.rows[s] - 1)) if self.trees is None else list(self.trees[s])

    def flat_parents(self):
        p = np.full(self.total, -1)
        for s in range(len(self.rows)):
            p[self.start[s]:self.start[s + 1]] = self.parents(s)
        return p

    def depths(self, s):
        d = []
        for p in self.parents(s):
            d.append(0 if p < 0 else d[p] + 1)
        return np.array(d, np.int64)

    def place(self, s, j):
        """Page and place of slots j of request s."""
        j = np.asarray(j)
        return self.table[s, j // self.page], j % self.page

    def sees(self, s):
        """[row, slot]: whether the row sees the slot."""
        n, t = self.lengths[s], self.rows[s]
        see = np.zeros((t, n + t), bool)
        see[:, :n] = True
        for i, p in enumerate(self.parents(s)):
            if p >= 0:
                see[i, n:] = see[p, n:]
            see[i, n + i] = True
        return see


def tree(rng, kind, t):
    """Parents of t rows."""
    if kind == "line":
        return list(range(-1, t - 1))
    if kind == "star":
        return [-1] + [0] * (t - 1)
    if kind == "forest":
        return [-1 if rng.random() < 0.3 else int(rng.integers(-1, i)) if i else -1 for i in range(t)]
    return [-1] + [int(rng.integers(max(0, i - 9), i)) for i in range(1, t)]


def rotate(x, pos, cos, sin):
    """x [rows, heads, 128] by the tables' rows at pos; and the magnitudes that the sums are made of."""
    c, s = cos[pos].astype(np.float64)[:, None], sin[pos].astype(np.float64)[:, None]
    lo, hi = x[..., :64], x[..., 64:]
    y = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
    mag = np.concatenate([abs(lo * c) + abs(hi * s), abs(hi * c) + abs(lo * s)], -1)
    return y, mag


def norm(x, w, eps):
    x = x.astype(np.float64)
    return x if w is None else x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * w.astype(np.float64)


def attention(q, k, v, see):
    """q [t, heads, D] of one KV head's group, k and v [slots, D], see [t, slots]: outputs, sum of p |v|, and the sum of
    |q k| / sqrt(D) of each row's largest slot; slots that a row does not see are not looked at."""
    t, heads, _ = q.shape
    out, pv, mag = np.zeros((t, heads, D)), np.zeros((t, heads, D)), np.zeros((t, heads))
    for i in range(t):
        at = np.nonzero(see[i])[0]
        if at.size == 0:
            continue
        with np.errstate(all="ignore"):
            x = q[i] @ k[at].T / math.sqrt(D)
            m = x.max(1, keepdims=True)
            e = np.where(x == -np.inf, 0.0, np.exp(x - m))
            p = e / e.sum(1, keepdims=True)
            p = np.where(m == -np.inf, 0.0, p)
            out[i], pv[i] = p @ v[at], p @ abs(v[at])
            mag[i] = (abs(q[i]) @ abs(k[at]).T).max(1) / math.sqrt(D)
    return out, pv, mag


def accept(parents, tokens, picks):
    path = [0]
    while True:
        more = [i for i, p in enumerate(parents) if p == path[-1] and tokens[i] == picks[path[-1]]]
        if not more:
            return path
        path.append(more[0])
