"""Plain 64-bit forms of the batch attention operators, and bounds of their rounding.

EPS is half a step of fp32 (2^-24), the error of one rounding."""
import numpy as np

EPS = 2.0 ** -24


def starts(lens, first=0):
    return np.concatenate([[first], first + np.cumsum(lens)]).astype(np.int32)


def attention(q, k, v, scale, hidden):
    """One head: q [nq, D], k and v [nk, D] float64, hidden [nq, nk]; (out, weights, score error)."""
    nq, nk = q.shape[0], k.shape[0]
    out, w = np.zeros((nq, v.shape[1])), np.zeros((nq, nk))
    with np.errstate(all="ignore"):
        for i in range(nq):
            s = np.flatnonzero(~hidden[i])
            if len(s) == 0:
                continue
            a = k[s] @ q[i] * scale
            p = np.exp(a - a.max())
            w[i, s] = p / p.sum()
            out[i] = w[i, s] @ v[s]
    return out, w


def row_bound(q, k, v, scale, hidden):
    """How far an fp32 row may be off: a score is a sum of D products (D + 16 roundings of
    the sum of their sizes), an error d in the scores moves a weight by at most 2 d of
    it, and the sums over the keys run in chains of nk / 16 + 64 roundings."""
    nk = k.shape[0]
    if nk == 0:
        return np.zeros(q.shape[0])
    size = abs(scale) * np.abs(q).max(1, keepdims=True) * np.abs(k).sum(1)[None, :]
    size = np.where(hidden, 0, size).max(1)
    d = (q.shape[1] + 16) * EPS * size
    top = np.where(hidden[:, :, None], 0, np.abs(v)[None]).max((1, 2)) if v.size < 1 << 16 else np.abs(v).max()
    return (2 * d + (nk / 16 + 64) * EPS) * top


def packed(q, k, v, qs, ks, scale, group):
    """attention_packed in 64 bits: (out, bound per row and head), NaN where no row belongs."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape[:2])
    for s in range(len(qs) - 1):
        a, b, c, d = qs[s], qs[s + 1], ks[s], ks[s + 1]
        nq, nk = b - a, d - c
        hidden = np.arange(nk)[None, :] > np.arange(nq)[:, None] + nk - nq
        for h in range(q.shape[1]):
            kk, vv = k[c:d, h // group], v[c:d, h // group]
            out[a:b, h], _ = attention(q[a:b, h], kk, vv, scale, hidden)
            with np.errstate(all="ignore"):
                tol[a:b, h] = row_bound(q[a:b, h], kk, vv, scale, hidden)
    return out, tol


def quotient(x, s):
    """x / s to the nearest whole number in 64 bits, 0 where s is not a positive number."""
    live = (s > 0) & (s < np.inf)
    with np.errstate(all="ignore"):
        return np.where(live, np.rint(x / np.where(live, s, 1)), 0)


class Cache:
    """The 8-bit cache in numpy: codes int8 [B, H, cap, D], scales float32 [B, H, blocks]."""

    def __init__(self, kc, vc, ks, vs, block):
        self.kc, self.vc, self.ks, self.vs, self.block = kc, vc, ks, vs, block

    def append(self, k, v, st, lengths):
        t, cap = self.block, self.kc.shape[2]
        for x, c, z in ((k, self.kc, self.ks), (v, self.vc, self.vs)):
            for b, end in enumerate(lengths):
                n = st[b + 1] - st[b]
                have = int(end) - int(n)
                lo, hi = max(have, 0), min(int(end), cap)
                if lo >= hi:
                    continue
                for h in range(c.shape[1]):
                    for p0 in range(lo - lo % t, hi, t):
                        f, e = max(p0, lo), min(p0 + t, hi)
                        y = x[st[b] + f - have:st[b] + e - have, h]
                        with np.errstate(all="ignore"):
                            s = np.abs(y).max() / np.float32(127)
                            before = z[b, h, p0 // t] if f > p0 else np.float32(0)
                            if np.isnan(before) or not np.isfinite(y).all():
                                s = np.float32(np.nan)
                            s = np.float32(np.maximum(before, s))
                            old = c[b, h, p0:f].astype(np.float64)
                            if not before == s:
                                live = 0 < s < np.inf
                                old = np.rint(old * (np.float64(before) / np.float64(s))) if live else old * 0
                            new = np.clip(quotient(y.astype(np.float64), np.float64(s)), -127, 127)
                        c[b, h, p0:f] = old
                        c[b, h, f:e] = new
                        z[b, h, p0 // t] = s

    def values(self, c, z):
        of = np.arange(c.shape[2]) // self.block
        with np.errstate(all="ignore"):
            return c.astype(np.float32) * z[:, :, of][..., None]

    def read(self, st, lengths, k, v):
        for out, c, z in ((k, self.kc, self.ks), (v, self.vc, self.vs)):
            x = self.values(c, z)
            for b, end in enumerate(lengths):
                n = int(st[b + 1]) - int(st[b])
                for i in range(n):
                    p = int(end) - n + i
                    out[st[b] + i] = x[b, :, p] if 0 <= p < c.shape[2] else 0

    def attention(self, q, lengths, scale, seen=None):
        """(out, seen, bound of out, bound of seen) in 64 bits."""
        B, heads, _ = q.shape
        H, cap = self.kc.shape[1:3]
        g = heads // H
        k, v = self.values(self.kc, self.ks).astype(np.float64), self.values(self.vc, self.vs).astype(np.float64)
        out, tol = np.zeros(q.shape), np.zeros(q.shape[:2])
        seen = None if seen is None else seen.astype(np.float64)
        stol = np.zeros((B, H, cap))
        for b in range(B):
            n = min(max(int(lengths[b]), 0), cap)
            for h in range(heads):
                qq = q[b, h:h + 1].astype(np.float64)
                hid = np.zeros((1, n), bool)
                kk, vv = k[b, h // g, :n], v[b, h // g, :n]
                o, w = attention(qq, kk, vv, scale, hid)
                out[b, h] = o[0]
                with np.errstate(all="ignore"):
                    tol[b, h] = row_bound(qq, kk, vv, scale, hid)[0]
                    one = row_bound(qq, kk, np.ones((n, 1)), scale, hid)[0]
                if seen is not None:
                    seen[b, h // g, :n] += w[0]
                    stol[b, h // g, :n] += w[0] * one
        if seen is not None:
            # an fp32 exponential below 2^-126 has no relative error (it is subnormal or 0):
            # each head's weight may be off by that much, whatever its size
            stol += (g + 1) * EPS * np.abs(seen) + g * 2.0 ** -126
        return out, seen, tol, stol

    def evict(self, to, lengths, seen, budget, recent, new_seen, kept):
        t = self.block
        for b in range(self.kc.shape[0]):
            n = min(max(int(lengths[b]), 0), self.kc.shape[2])
            for h in range(self.kc.shape[1]):
                key = np.where(np.isnan(seen[b, h, :n]), np.inf, seen[b, h, :n]).astype(np.float64)
                nan = np.isnan(seen[b, h, :n])
                i = np.arange(n)
                at = i if n <= budget else np.sort(np.lexsort((i, -key, ~nan, i < n - recent))[:budget])
                m = len(at)
                kept[b, h, :m], kept[b, h, m:] = at, -1
                new_seen[b, h, :m] = seen[b, h, at]
                for c, z, c2, z2 in ((self.kc, self.ks, to.kc, to.ks), (self.vc, self.vs, to.vc, to.vs)):
                    for p in range(0, m, t):
                        a = at[p:p + t]
                        z1 = z[b, h, a // t]
                        s = np.maximum.reduce(z1)       # a NaN comes through
                        live = 0 < s < np.inf
                        r = z1.astype(np.float64) / np.float64(s) if live else np.zeros(len(a))
                        c2[b, h, p:p + len(a)] = np.rint(c[b, h, a] * r[:, None])
                        z2[b, h, p // t] = s
