"""The operators of include/sp_hipkv.h on numpy arrays in 64 bits, and paged caches
to run them on."""
import numpy as np

import spkv
from devmem import Dev

PAGE = 64


def spinor_chunks(hd):
    nb = -(-hd // 55)
    base, extra = hd // nb, hd % nb
    return np.repeat(np.arange(nb), [base + (b < extra) for b in range(nb)]), nb, (hd + 4 * nb + 15) // 16 * 16


class Cache:
    """A pool of pages in shuffled order and a table for every sequence; every row
    that no position maps to holds NaN (exact rows: large numbers)."""

    def __init__(self, g, rows, nkv, hd, lens, ring=0, scale=1.0):
        self.rows, self.nkv, self.hd, self.ring, self.lens = rows, nkv, hd, ring, lens
        need = [max(1, -(-n // PAGE)) for n in lens]
        if ring:
            need = [min(n, ring) for n in need]
        order = g.permutation(sum(need))
        self.page = [order[sum(need[:i]):sum(need[:i + 1])] for i in range(len(lens))]
        chunk, nb, rb = spinor_chunks(hd)
        n = sum(need)
        if rows == spkv.ROWS_SPINOR:
            self.pool = np.zeros((n, 2, nkv, PAGE, rb), np.uint8)
            self.pool[..., hd:hd + 4 * nb] = np.full((n, 2, nkv, PAGE, nb), np.nan, np.float32).view(np.uint8)
            self.pool[..., :hd] = 77
        elif rows == spkv.ROWS_EXACT:
            self.pool = np.full((n, 2, nkv, PAGE, hd), 0x7FFFFF, np.int32)
        else:
            self.pool = np.full((n, 2, nkv, PAGE, hd), np.nan, np.float32)
        for s, ln in enumerate(lens):
            first = max(0, ln - ring * PAGE) if ring else 0
            for p in range(first, ln):
                at = self._at(s, p)
                if rows == spkv.ROWS_SPINOR:
                    code = np.clip(np.rint(g.standard_normal((2, nkv, hd)) * 40), -127, 127).astype(np.int8)
                    mul = (0.02 * scale + 0.01 * g.random((2, nkv, nb))).astype(np.float32)
                    self.pool[at[0], :, :, at[1], :hd] = code.view(np.uint8)
                    self.pool[at[0], :, :, at[1], hd:hd + 4 * nb] = mul.view(np.uint8)
                elif rows == spkv.ROWS_EXACT:
                    self.pool[at[0], :, :, at[1]] = np.rint(g.standard_normal((2, nkv, hd)) * scale * 65536)
                else:
                    self.pool[at[0], :, :, at[1]] = g.standard_normal((2, nkv, hd)) * scale

    def _at(self, s, p):
        lp = p // PAGE
        return self.page[s][lp % self.ring if self.ring else lp], p % PAGE

    def set(self, s, p, value):
        """Every element of position p's K and V rows."""
        a, b = self._at(s, p)
        if self.rows == spkv.ROWS_SPINOR:
            chunk, nb, rb = spinor_chunks(self.hd)
            self.pool[a, :, :, b, self.hd:self.hd + 4 * nb] = np.full((2, self.nkv, nb), value, np.float32).view(np.uint8)
        else:
            self.pool[a, :, :, b] = value

    def values(self, s, positions, v):
        """[positions][kv head][hd] of K (v = 0) or V (1)."""
        out = np.stack([self.pool[a, v, :, b] for a, b in (self._at(s, p) for p in positions)])
        if self.rows == spkv.ROWS_SPINOR:
            chunk, nb, rb = spinor_chunks(self.hd)
            mul = np.ascontiguousarray(out[..., self.hd:self.hd + 4 * nb]).view(np.float32)
            out = out[..., :self.hd].view(np.int8).astype(np.float64) * mul[..., chunk]
        return out

    def upload(self):
        self.dev = Dev(self.pool)
        size = self.pool[0].nbytes
        self.tabs = Dev(np.concatenate([self.dev.at + p.astype(np.int64) * size for p in self.page]))
        starts = np.cumsum([0] + [len(p) for p in self.page])[:-1]
        self.lists = Dev(self.tabs.at + 8 * starts.astype(np.int64))
        return self


def masks(g, kind, nodes):
    """Rows of visible nodes, and each node's depth."""
    see, depth = [], []
    for j in range(nodes):
        if kind == "chain":
            see.append(set(range(j + 1))); depth.append(j)
        elif kind == "none":
            see.append(set()); depth.append(0)
        elif kind == "random":
            see.append({k for k in range(nodes) if g.random() < 0.3}); depth.append(int(g.integers(0, 5)))
        else:
            up = -1 if j == 0 else int(g.integers(max(0, (j - 1) // 3 - 1), max(1, (j + 2) // 2)))
            see.append((see[up] if up >= 0 else set()) | {j}); depth.append(depth[up] + 1 if up >= 0 else 0)
    return see, depth


def words(see, n):
    out = np.zeros((len(see), n), np.uint64)
    for i, s in enumerate(see):
        for j in s:
            out[i, j // 64] |= np.uint64(1 << (j % 64))
    return out


def tree_attention(cache, cached, trees, q, window, scale, exact_head=None):
    """[nodes][heads][hd] in 64 bits, and a bound on what f32 sums in any order are
    off by.  trees: (see, depth) of each sequence.

    u = 2^-24.  A score sums hd products, each rounded once or not at all: off by
    at most (hd + 4) u scale |q|.|k|, d in all (the factors 4: the scale, the
    subtraction of the maximum, the exponential's argument and result).  A weight is
    then off by a factor of at most e^(2 d), numerator and denominator by n u more
    for the sums over n positions and the products: (4 d + (2 n + 64) u) sum p |v|
    (twice 2 d, as e^(2 d) - 1 < 4 d for the small d here)."""
    out, tol, i = np.zeros(q.shape), np.zeros(q.shape), 0
    NH, hd = q.shape[1:]
    G, u = NH // cache.nkv, 2.0 ** -24
    for s, (see, depth) in enumerate(trees):
        for j, nodes in enumerate(see):
            low = max(0, min(cached[s], cached[s] + depth[j] - window + 1)) if window else 0
            pos = list(range(low, cached[s])) + [cached[s] + k for k in sorted(nodes)]
            if pos:
                K, V = cache.values(s, pos, 0), cache.values(s, pos, 1)
                for h in range(NH):
                    k, v = K[:, h // G], V[:, h // G]
                    if exact_head:
                        out[i, h] = exact_head(q[i, h], k, v)
                        continue
                    k, v, x = k.astype(np.float64), v.astype(np.float64), q[i, h].astype(np.float64)
                    z = k @ x * scale
                    w = np.exp(z - z.max())
                    w /= w.sum()
                    out[i, h] = w @ v
                    d = (hd + 4) * u * scale * (np.abs(k) @ np.abs(x)).max() + 4 * u * np.abs(z - z.max()).max()
                    tol[i, h] = (4 * d + (2 * len(pos) + 64) * u) * (w @ np.abs(v))
            i += 1
    return out, tol


def logprobs(x, scale, given, top):
    """given, entropy, lse, ids, top log p in 64 bits (long double sums)."""
    y = x.astype(np.longdouble) * np.longdouble(np.float32(scale))
    m = y.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.exp(y - m)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    big = np.argmax(y, axis=1)
    e[np.arange(len(x)), big] = 0
    r = e.sum(1)
    lse = m[:, 0] + np.log1p(r)
    d = np.where(e > 0, y - m, 0)
    ent = np.log1p(r) - (e * d).sum(1) / (1 + r)
    rows = np.arange(len(x))[:, None]
    return ((y[rows, given] - m) - np.log1p(r)[:, None], ent, lse, order, (y[rows, order] - m) - np.log1p(r)[:, None])
