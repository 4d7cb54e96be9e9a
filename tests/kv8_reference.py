"""The 8-bit K/V cache and the log probabilities in 64 bits: what the kernels' tests compare with."""
import numpy as np

D = 128
TOP = {"e4m3": 448.0, "int8": 127.0}

# the E4M3 numbers of codes 0..126 (127 is NaN), ascending
E4M3 = np.array([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])


def scale_of(amax, fmt):
    """Smallest power of two s with amax <= TOP s (0 for 0)."""
    amax = np.asarray(amax, np.float64)
    out = np.zeros_like(amax)
    for e in range(-40, 20):
        s = 2.0 ** e
        hit = (out == 0) & (amax > 0) & (amax <= TOP[fmt] * s)
        out[hit] = s
    return out


def rounded(y, fmt):
    """Numbers (in units of the scale) rounded to nearest even in the format; NaN stays in E4M3 and is 0 in INT8."""
    if fmt == "int8":
        return np.clip(np.rint(np.nan_to_num(y, nan=0.0)), -127, 127)
    a = np.abs(y)
    i = np.clip(np.searchsorted(E4M3, np.nan_to_num(a), side="right") - 1, 0, 126)
    j = np.minimum(i + 1, 126)
    lo, hi = a - E4M3[i], E4M3[j] - a
    up = (hi < lo) | ((hi == lo) & (i % 2 == 1))
    v = np.where(up, E4M3[j], E4M3[i])
    return np.where(np.isnan(y), np.nan, np.copysign(v, y))


def numbers(codes, fmt):
    """uint8 codes to the numbers they stand for."""
    if fmt == "int8":
        return codes.view(np.int8).astype(np.float64)
    table = np.concatenate([E4M3, [np.nan]])
    v = table[codes & 127]
    return np.where(codes & 128, -v, v)


class Cache:
    """Numbers (units of the scale) and scales, with the store and the eviction by their definitions."""

    def __init__(self, fmt, block, cap, hkv):
        self.fmt, self.block, self.cap, self.hkv = fmt, block, cap, hkv
        nb = -(-cap // block)
        self.num = {x: np.zeros((hkv, cap, D)) for x in "kv"}
        self.scale = {x: np.zeros((hkv, nb)) for x in "kv"}

    def store(self, k, v, slot):
        """k, v [t][hkv][128] float64 (FP16 values)."""
        for x, new in (("k", k), ("v", v)):
            new = np.clip(new.transpose(1, 0, 2), -65504, 65504)
            t = new.shape[1]
            for b in range(slot // self.block, (slot + t - 1) // self.block + 1):
                lo, hi = max(slot, b * self.block), min(slot + t, (b + 1) * self.block)
                part = new[:, lo - slot:hi - slot]
                s = scale_of(np.nan_to_num(np.abs(part)).max((1, 2)), self.fmt)
                if lo > b * self.block:
                    old = self.scale[x][:, b]
                    s = np.maximum(s, old)
                    one = np.where(s > 0, s, 1)
                    was = self.num[x][:, b * self.block:lo]
                    self.num[x][:, b * self.block:lo] = rounded(was * (old / one)[:, None, None], self.fmt)
                self.num[x][:, lo:hi] = rounded(part / np.where(s > 0, s, 1)[:, None, None], self.fmt)
                self.scale[x][:, b] = s

    def values(self, x, n):
        return self.num[x][:, :n] * np.repeat(self.scale[x], self.block, 1)[:, :n, None]

    def evict(self, acc, n, n_keep, n_sink, n_recent, cap):
        """(kept [hkv][n_keep], the new cache, its weights)."""
        d = Cache(self.fmt, self.block, cap, self.hkv)
        kept = np.zeros((self.hkv, n_keep), np.int64)
        out = np.zeros((self.hkv, cap))
        for g in range(self.hkv):
            a = np.where(np.isnan(acc[g, :n]), -np.inf, acc[g, :n])
            rank = [(0 if i < n_sink or i >= n - n_recent else 1, -a[i], bool(np.isnan(acc[g, i])), i)
                    for i in range(n)]
            kept[g] = sorted(r[3] for r in sorted(rank)[:n_keep])
            out[g, :n_keep] = acc[g, kept[g]]
            for x in "kv":
                for b in range(-(-n_keep // self.block)):
                    at = kept[g, b * self.block:(b + 1) * self.block]
                    old = self.scale[x][g, at // self.block]
                    d.scale[x][g, b] = s = old.max()
                    d.num[x][g, b * self.block:b * self.block + at.size] = \
                        rounded(self.num[x][g, at] * (old / (s if s > 0 else 1))[:, None], self.fmt)
        return kept, d, out


def attention(q, k, v, t, hidden):
    """q [t][hq][128], k, v [hkv][n][128], hidden [n] bool. Output [t][hq][128], weight [hkv][n], and per output and
    slot what the error bounds need: sum p |v| and the largest sum |q k| / sqrt(128) of a row."""
    hq, (hkv, n, _) = q.shape[1], k.shape
    G = hq // hkv
    out, pv = np.zeros((t, hq, D)), np.zeros((t, hq, D))
    acc, mag = np.zeros((hkv, n)), np.zeros((t, hq))
    for h in range(hq):
        g = h // G
        for i in range(t):
            see = ~hidden & (np.arange(n) <= n - t + i)
            if not see.any():
                continue
            x = k[g, see] @ q[i, h] / np.sqrt(D)
            mag[i, h] = (np.abs(k[g, see]) @ np.abs(q[i, h])).max() / np.sqrt(D)
            p = np.exp(x - x.max())
            p /= p.sum()
            out[i, h] = p @ v[g, see]
            pv[i, h] = p @ np.abs(v[g, see])
            acc[g, see] += p
    return out, acc, pv, mag


def logprobs(x, seen):
    """Log probabilities [rows][vocab] (-inf where not seen), entropy, and per row m and z (the sum without one maximum)."""
    x = np.where(seen, x, -np.inf)
    m = x.max(1, keepdims=True)
    m0 = np.where(np.isfinite(m), m, 0)
    e = np.exp(x - m0)
    first = x.argmax(1)
    e[np.arange(len(x)), first] = 0
    z = e.sum(1, keepdims=True)
    lz = np.log1p(z)
    lp = np.where(np.isfinite(x), x - m0 - lz, -np.inf)
    w = np.where(e > 0, e * (m0 - np.where(np.isfinite(x), x, 0)), 0).sum(1, keepdims=True)
    return lp, (lz + w / (1 + z))[:, 0], m0[:, 0], z[:, 0]


def top(x, seen, k):
    """The k best ids of one row by value, then by id; -1 where there is none above -inf."""
    ok = np.nonzero(seen & (x > -np.inf))[0]
    best = ok[np.lexsort((ok, -x[ok]))][:k]
    return np.concatenate([best, np.full(k - best.size, -1, np.int64)])
