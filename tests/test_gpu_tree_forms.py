"""Tree attention in every form that is built: each number of row tiles a workgroup takes,
one part and several, with windows and ragged sequences.  The sizes' plans are asked for
on the CPU (test_tree_plans.py), so that another choice of them cannot leave a form out."""
import numpy as np
import pytest

import tree_ref
from test_gpu_tree_ops import EXACT, F32, SPINOR, Tree

pytestmark = pytest.mark.gpu

# rows, head_dim, q heads for each kv head, kv heads, sequences, cached, nodes, window
FLOAT = [
    (F32, 64, 3, 2, 2, 7, 11, 0), (F32, 64, 3, 2, 2, 333, 11, 90), (F32, 64, 3, 2, 2, 700, 5, 0), (F32, 64, 3, 1, 2, 1100, 5, 700),
    (F32, 64, 4, 4, 33, 7, 5, 0), (F32, 64, 16, 4, 5, 333, 13, 90), (F32, 64, 8, 2, 2, 1100, 25, 0), (F32, 64, 8, 1, 5, 1100, 25, 700),
    (F32, 64, 4, 4, 33, 7, 9, 0), (F32, 64, 16, 4, 5, 333, 25, 90), (F32, 64, 5, 2, 3, 1100, 67, 0),
    (F32, 64, 4, 4, 33, 7, 13, 0), (F32, 64, 4, 4, 33, 333, 13, 90), (F32, 64, 16, 1, 3, 1100, 67, 0),
    (F32, 128, 3, 2, 2, 7, 11, 0), (F32, 128, 3, 2, 2, 333, 11, 90), (F32, 128, 3, 2, 2, 700, 5, 0), (F32, 128, 3, 1, 2, 1100, 5, 700),
    (F32, 128, 4, 4, 33, 7, 5, 0), (F32, 128, 16, 4, 5, 333, 13, 90), (F32, 128, 8, 2, 2, 1100, 25, 0), (F32, 128, 8, 1, 5, 1100, 25, 700),
    (F32, 128, 4, 4, 33, 7, 9, 0), (F32, 128, 16, 4, 5, 333, 25, 90), (F32, 128, 5, 2, 9, 1100, 13, 0), (F32, 128, 16, 4, 3, 1100, 9, 700),
    (F32, 256, 3, 2, 2, 7, 11, 0), (F32, 256, 3, 2, 2, 333, 11, 90), (F32, 256, 3, 2, 2, 700, 5, 0), (F32, 256, 3, 1, 2, 1100, 5, 700),
    (F32, 256, 4, 4, 33, 7, 5, 0), (F32, 256, 16, 4, 5, 333, 13, 90), (F32, 256, 8, 1, 2, 700, 67, 0), (F32, 256, 8, 1, 2, 700, 67, 700),
    (SPINOR, 64, 3, 2, 2, 7, 11, 0), (SPINOR, 64, 3, 2, 2, 333, 11, 90), (SPINOR, 64, 3, 2, 2, 700, 5, 0), (SPINOR, 64, 3, 1, 2, 1100, 5, 700),
    (SPINOR, 64, 16, 8, 1, 7, 67, 0), (SPINOR, 64, 16, 8, 2, 333, 67, 90), (SPINOR, 64, 16, 4, 1, 700, 67, 0), (SPINOR, 64, 16, 4, 1, 700, 67, 700),
    (SPINOR, 64, 16, 16, 1, 7, 67, 0), (SPINOR, 64, 16, 16, 2, 333, 67, 90), (SPINOR, 64, 16, 4, 1, 1100, 67, 0),
    (SPINOR, 128, 3, 2, 2, 7, 11, 0), (SPINOR, 128, 3, 2, 2, 333, 11, 90), (SPINOR, 128, 3, 2, 2, 700, 5, 0), (SPINOR, 128, 3, 1, 2, 1100, 5, 700),
    (SPINOR, 128, 16, 8, 1, 7, 67, 0), (SPINOR, 128, 16, 8, 2, 333, 67, 90), (SPINOR, 128, 8, 8, 1, 1100, 25, 0), (SPINOR, 128, 16, 2, 1, 1100, 67, 700),
    (SPINOR, 256, 3, 2, 2, 7, 11, 0), (SPINOR, 256, 3, 2, 2, 333, 11, 90), (SPINOR, 256, 3, 2, 2, 700, 5, 0), (SPINOR, 256, 3, 1, 2, 1100, 5, 700),
    (SPINOR, 256, 16, 2, 3, 333, 13, 0),
]
INTEGER = [(EXACT, hd, 4, 1, s, cached, nodes, window) for hd in (64, 128, 256)
           for nodes, s, cached, window in ((3, 1, 20, 0), (4, 1, 700, 0), (7, 1, 20, 0), (8, 2, 300, 90), (11, 1, 300, 0), (12, 1, 20, 0), (15, 2, 20, 0),
                                            (16, 1, 300, 0), (19, 1, 20, 0), (20, 1, 300, 90), (23, 1, 20, 0), (24, 2, 200, 0), (27, 1, 300, 0))]


def lengths(S, cached, nodes):
    """Ragged: the first sequence has the largest counts, which the plan goes by."""
    return [cached if s == 0 else cached * (s * 7 % 11) // 11 for s in range(S)], [nodes if s == 0 else 1 + (nodes - 1) * (s * 5 % 9) // 9 for s in range(S)]


def build(case, seed=51):
    rows, hd, G, nkv, S, cached, nodes, window = case
    c, n = lengths(S, cached, nodes)
    return Tree(rows, hd, G, c, n, window=window, nkv=nkv, seed=seed)


def values(cache, s, n, kv):
    """[positions][kv head][hd] of a sequence's first n positions."""
    p = np.arange(n)
    out = cache.pool[np.asarray(cache.page[s])[p // 64], kv, :, p % 64]
    if cache.rows == SPINOR:
        chunk, nb, rb = tree_ref.spinor_chunks(cache.hd)
        mul = np.ascontiguousarray(out[..., cache.hd:cache.hd + 4 * nb]).view(np.float32)
        out = out[..., :cache.hd].view(np.int8).astype(np.float64) * mul[..., chunk]
    return out.astype(np.float64)


def reference(t):
    """tree_ref.tree_attention and its bound, whole matrices at a time.  Values that no
    compared row sees may be anything: they are 0 here."""
    G, u, hd = t.NH // t.cache.nkv, 2.0 ** -24, t.hd
    q = t.q[:, :t.NH * hd].reshape(-1, t.NH, hd).astype(np.float64)
    out, tol, at = np.zeros(q.shape), np.zeros(q.shape), 0
    for s, (see, depth) in enumerate(t.trees):
        n, c = len(see), t.cached[s]
        seen = np.zeros((n, c + n), bool)
        for j in range(n):
            seen[j, (max(0, min(c, c + depth[j] - t.window + 1)) if t.window else 0):c] = True
            seen[j, [c + k for k in see[j]]] = True
        seen = np.repeat(seen, G, 0)
        K, V = values(t.cache, s, c + n, 0), values(t.cache, s, c + n, 1)
        for x in (K, V):
            x[~(np.abs(x) < 1e30)] = 0
        for h in range(t.cache.nkv):
            x = q[at:at + n, h * G:(h + 1) * G].reshape(n * G, hd)
            z = np.where(seen, x @ K[:, h].T * t.scale, -np.inf)
            d = np.where(seen, np.abs(x) @ np.abs(K[:, h]).T, 0).max(1)
            off = z.max(1, keepdims=True) - z
            w = np.exp(-off)
            w /= w.sum(1, keepdims=True)
            d = (hd + 4) * u * t.scale * d + 4 * u * np.where(seen, off, 0).max(1)
            out[at:at + n, h * G:(h + 1) * G] = (w @ V[:, h]).reshape(n, G, hd)
            e = (4 * d + (2 * seen.sum(1) + 64) * u)[:, None] * (w @ np.abs(V[:, h]))
            tol[at:at + n, h * G:(h + 1) * G] = e.reshape(n, G, hd)
        at += n
    return out, tol


@pytest.mark.parametrize("case", FLOAT, ids=str)
def test_float_forms(case):
    """As it is, then with values that nobody but its own node sees: the last node of each
    sequence, places before every window, unused places."""
    t = build(case).ready()
    got, (want, tol) = t.run(), reference(t)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all(), (np.abs(got - want) - tol).max()
    last = np.cumsum(t.nodes) - 1
    for bits in (0x7F7F8000, 0xFF7FFFFF, 0x7F800000, 0x7FC00000):
        bad = np.array([bits], np.uint32).view(np.float32)[0]
        t = build(case)
        with np.errstate(all="ignore"):
            for s, (c, n) in enumerate(zip(t.cached, t.nodes)):
                if n > 1:
                    t.cache.set(s, c + n - 1, bad)
                for p in range(max(0, c - t.window + 1) if t.window else 0):
                    t.cache.set(s, p, bad)
            t.ready()
            rest = np.delete(np.arange(len(got)), [i for i, n in zip(last, t.nodes) if n > 1])
            again = t.run()
        assert np.isfinite(again[rest]).all() and (np.abs(again - want) <= tol)[rest].all()


@pytest.mark.parametrize("case", INTEGER, ids=str)
def test_exact_forms(case):
    build(case).ready().check()
