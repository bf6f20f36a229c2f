"""Tree attention of rows that hold extreme values: what a node does not see never
reaches it, what it sees and is not finite always does.  Tolerances: tree_ref."""
import numpy as np
import pytest

import tree_ref
from helpers import prompt
from test_gpu_tree_ops import EXACT, F32, SPINOR, Tree
from test_gpu_tree_step import Rig, close, path, tree

pytestmark = pytest.mark.gpu


def f32(bits):
    return np.array([bits], np.uint32).view(np.float32)[0]


# 0x7F7F8000 is the least magnitude that rounds to an infinite bf16, 0x7F7F7FFF the largest that does not
HUGE = [0x7F7FFFFF, 0xFF7FFFFF, 0x7F7F8000, 0xFF7F8000, 0x7F7F7FFF, 0xFF7F7FFF, 0x7F800000, 0xFF800000, 0x7FC00000, 0x7F800001]


def fill_unused(t, value):
    """Places of the pool that no position maps to (Cache marks them with NaN)."""
    if t.cache.rows == SPINOR:
        chunk, nb, rb = tree_ref.spinor_chunks(t.hd)
        mul = np.ascontiguousarray(t.cache.pool[..., t.hd:t.hd + 4 * nb]).view(np.float32)
        mul[np.isnan(mul)] = value
        t.cache.pool[..., t.hd:t.hd + 4 * nb] = mul.view(np.uint8)
    elif t.cache.rows == F32:
        t.cache.pool[np.isnan(t.cache.pool)] = value
    else:
        t.cache.pool[t.cache.pool == 0x7FFFFF] = value


def hidden(rows, hd, value, cached=300, nodes=40, window=64):
    """A tree whose hidden positions and unused places all hold a value: below every
    window, and a last node that only it sees itself."""
    t = Tree(rows, hd, 2, [cached], [nodes], window=window, seed=31)
    with np.errstate(all="ignore"):
        fill_unused(t, value)
        for p in range(cached - window - 20 if window else 0):
            t.cache.set(0, p, value)
        t.cache.set(0, cached + nodes - 1, value)
    assert all(nodes - 1 not in see for see in t.trees[0][0][:-1])
    return t.ready()


def same_but_the_last(t):
    with np.errstate(all="ignore"):
        got, (want, tol) = t.run(), t.want()
    n = len(got) - 1
    assert np.isfinite(got[:n]).all()
    assert (np.abs(got[:n] - want[:n]) <= tol[:n]).all()
    return got


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [F32, SPINOR])
def test_unseen_values_of_any_size(rows, hd):
    """Largest numbers beside infinities and NaN, with a window and without."""
    for bits in HUGE:
        same_but_the_last(hidden(rows, hd, f32(bits)))
    same_but_the_last(hidden(rows, hd, f32(0x7F7FFFFF), cached=2900, nodes=9, window=0))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_unseen_values_of_exact_rows(hd):
    """... and the largest integers: the bits of a cache without them."""
    clean = hidden(EXACT, hd, 0).run()
    for value in (0x7FFFFFFF, -0x80000000, 0x7FFFFF, -1):
        assert np.array_equal(hidden(EXACT, hd, value).run()[:-1].view(np.uint32), clean[:-1].view(np.uint32))


def test_unseen_words_of_any_bits():
    """Whatever memory held before: random words in every hidden and unused place."""
    g = np.random.default_rng(5)
    t = Tree(F32, 128, 2, [300], [40], window=64, seed=32)
    bits = g.integers(0, 1 << 32, t.cache.pool.shape, np.uint64).astype(np.uint32)
    some = g.random(bits.shape) < 0.5                     # half of them among the values that round up to infinity
    bits[some] = 0x7F7F8000 | (bits[some] & 0x80007FFF)
    unused = np.isnan(t.cache.pool)
    t.cache.pool.view(np.uint32)[unused] = bits[unused]
    for p in list(range(200)) + [339]:
        a, b = t.cache._at(0, p)
        t.cache.pool.view(np.uint32)[a, :, :, b] = bits[a, :, :, b]
    same_but_the_last(t.ready())


def test_seen_values_that_pieces_do_not_hold():
    """The header counts magnitudes from 2^127 on as not finite: a node that sees one is
    without a finite value in its column, in whole tiles and in others."""
    for p in (5, 200, 339):
        t = Tree(F32, 128, 2, [300], [40], kind="chain", seed=33)
        a, b = t.cache._at(0, p)
        t.cache.pool[a, 1, :, b, 17] = f32(0x7F7F9000)
        t.ready()
        got, (want, tol) = t.run(), t.want()
        hit = np.arange(40) >= p - 300
        assert not np.isfinite(got[hit][..., 17]).any()
        got[hit, :, 17], want[hit, :, 17] = 0, 0
        assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("shape", ["qwen3-tiny", "qwen3-hd128", "gemma3-hd256"])
def test_steps_over_pages_that_held_large_values(tmpdir_models, shape):
    """A handle's pages keep what was written and rewound: decode steps, which read no
    unused place, say what a tree step gives on them."""
    r = Rig(tmpdir_models, shape)
    b = r.backend(False)
    big = np.full((128, r.kvd), f32(0x7F7F8000), np.float32)
    big[::2] = f32(0xFF7FFFFF)
    for l in range(r.d["n_layers"]):
        b.write_kv(l, 0, big, big)
    assert b.rewind(128) == 0
    b.prefill(prompt(37, r.V, seed=3))
    parents, toks = tree(9, 4), prompt(9, r.V, seed=8)
    lg, nxt, _ = b.tree_step(toks, parents, r.V)
    ref = np.zeros(r.V, np.float32)
    for leaf in [i for i in range(9) if i not in parents]:
        f = b.fork()
        for i in path(parents, leaf):
            f.decode(int(toks[i]), ref)
            assert close(lg[i], ref), i
        f.close()
    b.close(); r.close()


def lifted(rows, cached, nodes, p0, hd=128):
    """Position p0 scores far above all others, 2^-300 or less of whose weight is left."""
    t = Tree(rows, hd, 2, [cached], [nodes], kind="chain", seed=34)
    t.q[:] = 1.0
    t.dq.put(t.q)
    a, b = t.cache._at(0, p0)
    k = np.float32(600 * np.sqrt(hd) / hd * np.log(2))
    if rows == F32:
        t.cache.pool[a, 0, :, b] = k
    else:
        chunk, nb, rb = tree_ref.spinor_chunks(hd)
        t.cache.pool[a, 0, :, b, :hd] = 100
        t.cache.pool[a, 0, :, b, hd:hd + 4 * nb] = np.full(nb, k / 100, np.float32).view(np.uint8)
    return t


def spoil(t, p, kv, value, column=0):
    """One V (1) or K (0) column of position p, of Spinor rows its chunk; the columns hit."""
    a, b = t.cache._at(0, p)
    if t.cache.rows == F32:
        t.cache.pool[a, kv, :, b, column] = value
        return np.arange(t.hd) == column
    chunk, nb, rb = tree_ref.spinor_chunks(t.hd)
    at = t.hd + 4 * chunk[column]
    t.cache.pool[a, kv, :, b, at:at + 4] = np.array([value], np.float32).view(np.uint8)
    return chunk == chunk[column]


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("rows", [F32, SPINOR])
@pytest.mark.parametrize("cached,p0,p1", [(300, 10, 12), (300, 10, 40), (300, 200, 5), (300, 10, 299), (300, 10, 302), (300, 302, 33), (5000, 100, 4000),
                                          (5000, 4000, 100), (5000, 100, 5001), (5000, 5000, 100)])
def test_seen_values_of_no_weight(rows, cached, p0, p1, value):
    """0 times NaN or infinity is NaN also where the weight is 0 by rounding: a V value that is
    seen spoils its column, in whatever tile, wave or part it lies beside the largest score."""
    t = lifted(rows, cached, 6, p0)
    hit = spoil(t, p1, 1, value, 70)
    t.ready()
    with np.errstate(all="ignore"):
        got, (want, tol) = t.run(), t.want()
    # node j sees the nodes up to itself; before the lifted one is seen the others share the weight
    sees = np.arange(6) >= p1 - cached
    assert not np.isfinite(got[sees][..., hit]).any()
    spoiled = sees[:, None, None] & hit
    got, want, tol = (np.where(spoiled, 0, x) for x in (got, want, tol))
    # the bounds are relative to sum p |v|; beside them a weight (at most 1 after its part's factor) below the
    # least normal number may be 0: (cached + 6) 2^-126 |v|, where nothing of weight has a value but 0
    v = 6.0 if rows == F32 else 127 * 0.03
    assert (np.abs(got - want) <= tol + (cached + 6) * 2.0 ** -126 * v).all()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("rows", [F32, SPINOR])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_seen_k_values_that_are_not_finite(rows, hd, value):
    """In K alone, one column or chunk: no finite value for the nodes that see it, whatever
    the signs of its products sum up to; the others as without it."""
    for cached, p in ((300, 12), (300, 298), (300, 303), (5000, 3000), (5000, 5004)):
        t = Tree(rows, hd, 4, [cached], [6], kind="chain", seed=35)
        spoil(t, p, 0, value, hd - 1)
        t.ready()
        with np.errstate(all="ignore"):
            got, (want, tol) = t.run(), t.want()
        sees = np.arange(6) >= p - cached
        assert not np.isfinite(got[sees]).any(), (cached, p)
        assert (np.abs(got[~sees] - want[~sees]) <= tol[~sees]).all()


@pytest.mark.parametrize("rows", [F32, SPINOR])
def test_seen_v_values_up_to_the_stated_magnitude(rows):
    """Weights reach 2^8 before the running maximum moves, and their sum 2^28 over the longest
    spans: V values below 2^100 stay within f32."""
    for cached, nodes in ((300, 40), (5000, 9)):
        t = Tree(rows, 128, 2, [cached], [nodes], kind="chain", seed=36)
        if rows == F32:
            t.cache.pool[:, 1] *= np.float32(2.0 ** 96)
        else:
            mul = np.ascontiguousarray(t.cache.pool[..., 128:140]).view(np.float32)
            mul[:, 1] *= np.float32(2.0 ** 97)
            t.cache.pool[..., 128:140] = mul.view(np.uint8)
        t.q[:, :256] *= 4                              # scores that rise by several powers of two
        t.dq.put(t.q)
        t.ready()
        with np.errstate(all="ignore"):
            assert 2.0 ** 98 < np.nanmax(np.abs(t.cache.values(0, range(cached + nodes), 1))) < 2.0 ** 100
        t.check()
