"""The operators of drafted token trees on device memory against plain 64-bit
implementations (tests/tree_ref.py, where the tolerances are derived)."""
import ctypes

import numpy as np
import pytest

import orc
import spkv
import tree_ref
from devmem import Dev, Stream, sync

pytestmark = pytest.mark.gpu
F32, EXACT, SPINOR = spkv.ROWS_F32, spkv.ROWS_EXACT, spkv.ROWS_SPINOR


class Tree:
    """One call's inputs on the device; rows past the nodes and columns past the
    heads hold a mark that must survive."""
    MARK = np.float32(-12345.0)

    def __init__(self, rows, hd, G, cached, nodes, window=0, ring=0, kind="tree", seed=0, nkv=2, pad=0, scale=1.0):
        g = np.random.default_rng([seed, hd, G, len(cached)])
        self.cached, self.nodes, self.window, NH = cached, nodes, window, nkv * G
        self.cache = tree_ref.Cache(g, rows, nkv, hd, [c + n for c, n in zip(cached, nodes)], ring, scale)
        self.trees = [tree_ref.masks(g, kind, n) for n in nodes]
        n, self.NH, self.hd = sum(nodes), NH, hd
        self.q = np.full((n, NH * hd + pad), np.nan, np.float32)
        self.q[:, :NH * hd] = g.standard_normal((n, NH * hd))
        w = (max(nodes) + 63) // 64
        vis = np.concatenate([tree_ref.words(see, w) for see, _ in self.trees])
        # bits past a sequence's nodes mean nothing
        for i, k in enumerate(np.repeat(nodes, nodes)):
            for j in range(k, 64 * w):
                vis[i, j // 64] |= np.uint64(1 << (j % 64))
        self.scale = float(np.float32(1) / np.sqrt(np.float32(hd)))
        self.dq, self.dv = Dev(self.q), Dev(vis)
        self.dstart, self.dcached = Dev(np.cumsum([0] + list(nodes)).astype(np.int32)), Dev(np.array(cached, np.int32))
        self.ddepth = Dev(np.concatenate([d for _, d in self.trees]).astype(np.int32))
        self.dout = Dev(np.full((n + 2, NH * hd + pad), self.MARK, np.float32))
        self.args = spkv.TreeArgs(
            n_heads=NH, n_kv_heads=nkv, head_dim=hd, rows=rows, n_seqs=len(cached), n_nodes=n, max_nodes=max(nodes),
            max_positions=max(c + k for c, k in zip(cached, nodes)), window=window, ring_pages=ring, mask_words=w, scale=self.scale,
            node_start=self.dstart.at, cached=self.dcached.at, depth=self.ddepth.at if window else None, visible=self.dv.at,
            q=self.dq.at, q_stride=NH * hd + pad, out=self.dout.at + 4 * (NH * hd + pad), out_stride=NH * hd + pad)

    def ready(self):
        self.cache.upload()
        self.args.tables = self.cache.lists.at
        need = spkv.tree_attention_work(self.args)
        self.work = Dev(np.full(need + 256, 0xA5, np.uint8))
        self.args.work, self.args.work_bytes = self.work.at, need
        return self

    def result(self):
        full = self.dout.get()
        assert (full[0] == self.MARK).all() and (full[-1] == self.MARK).all() and (full[:, self.NH * self.hd:] == self.MARK).all()
        w = self.work.get()
        assert (w[-256:] == 0xA5).all()
        return full[1:-1, :self.NH * self.hd].reshape(-1, self.NH, self.hd)

    def run(self, stream=0):
        spkv.tree_attention(self.args, stream)
        return self.result()

    def want(self):
        head = None
        if self.cache.rows == EXACT:
            head = lambda q, k, v: exact_head(q, k, v, self.scale)   # noqa: E731
        return tree_ref.tree_attention(self.cache, self.cached, self.trees, self.q[:, :self.NH * self.hd].reshape(-1, self.NH, self.hd),
                                       self.window, self.scale, head)

    def check(self, got=None):
        got = self.run() if got is None else got
        want, tol = self.want()
        if self.cache.rows == EXACT:
            assert np.array_equal(got.view(np.uint32), want.astype(np.float32).view(np.uint32))
        else:
            assert np.isfinite(got).all()
            worst = np.abs(got - want) - tol
            assert (worst <= 0).all(), (np.abs(got - want).max(), worst.max())
        return got


def exact_head(q, k, v, scale):
    n, hd = k.shape
    out = np.zeros(hd, np.float32)
    k, v, q = (np.ascontiguousarray(x) for x in (k, v, q))
    orc.lib().orc_attn_head_exact(spkv.ptr(q), spkv.ptr(k), spkv.ptr(v), n - 1, hd, 0, hd, ctypes.c_float(scale), -1, spkv.ptr(out))
    return out


ALL = [F32, SPINOR, EXACT]


@pytest.mark.parametrize("rows", ALL)
@pytest.mark.parametrize("hd,G", [(64, 1), (64, 4), (128, 2), (128, 4), (256, 2), (256, 16), (128, 3)])
def test_head_layouts(rows, hd, G):
    Tree(rows, hd, G, [70], [9], seed=1).ready().check()


@pytest.mark.parametrize("rows", ALL)
@pytest.mark.parametrize("cached,nodes", [([0], [1]), ([0], [5]), ([1], [1]), ([63], [2]), ([64], [1]), ([62], [67]), ([128], [64]),
                                          ([31], [33]), ([1000], [3]), ([515], [130]), ([0, 5, 300, 64], [3, 1, 17, 40])])
def test_lengths(rows, cached, nodes):
    Tree(rows, 128, 2, cached, nodes, seed=2).ready().check()


@pytest.mark.parametrize("rows", ALL)
def test_long_context(rows):
    """Spans cut into parts, and every count of nodes around a tile."""
    for nodes in (1, 8, 9, 33):
        Tree(rows, 128, 2, [5003], [nodes], seed=3, nkv=1).ready().check()


@pytest.mark.parametrize("rows", ALL)
@pytest.mark.parametrize("kind", ["chain", "random", "none"])
def test_masks(rows, kind):
    """Chains, arbitrary masks (a node that does not see itself), nodes without a
    position: zeros for them."""
    t = Tree(rows, 64, 2, [0, 77], [20, 20], kind=kind, seed=4).ready()
    got = t.check()
    if kind == "none":
        assert (got[:20] == 0).all() and np.abs(got[20:]).max() > 0


@pytest.mark.parametrize("rows", ALL)
@pytest.mark.parametrize("cached,ring", [(40, 0), (200, 0), (1000, 0), (1000, 6), (127, 6)])
def test_windows(rows, cached, ring):
    """The window of each node by its depth, in full tables and rings of pages."""
    Tree(rows, 128, 2, [cached, cached + 1], [24, 3], window=100, ring=ring, seed=5).ready().check()
    Tree(rows, 64, 4, [cached], [24], window=1, ring=ring, seed=6).ready().check()


@pytest.mark.parametrize("rows", [F32, SPINOR])
def test_unseen_rows_do_not_reach_a_node(rows):
    """NaN and infinities in rows that some or all nodes do not see: hidden
    nodes' rows for the others, positions before every window, unused places."""
    for bad in (np.nan, np.inf, -np.inf):
        t = Tree(rows, 128, 2, [300], [40], window=64, seed=7)
        for p in range(200):                            # below every window
            t.cache.set(0, p, bad)
        see, depth = t.trees[0]
        leaf = max(range(40), key=lambda j: j)          # nobody else sees the last node
        assert all(leaf not in see[j] for j in range(39))
        t.cache.set(0, 300 + leaf, bad)
        t.ready()
        got, (want, tol) = t.run(), t.want()
        assert np.isfinite(got[:39]).all() and (np.abs(got[:39] - want[:39]) <= tol[:39]).all()


def test_one_sided_rows():
    """Scores far apart (a weight of 1 and zeros) and equal scores."""
    t = Tree(F32, 128, 2, [200], [6], seed=8, scale=30.0).ready()
    t.check()
    t = Tree(F32, 128, 2, [200], [6], seed=8)
    t.q[:, :256] = 0.0
    t.dq.put(t.q)
    t.ready().check()


@pytest.mark.parametrize("rows", [F32, SPINOR])
def test_seen_rows_that_are_not_finite(rows):
    """A node that sees NaN in K or V has no number for an answer, also where it sees
    nothing else; the nodes beside it keep theirs."""
    t = Tree(rows, 128, 2, [0, 500], [6, 20], kind="chain", seed=15)
    t.trees[0] = ([{j} for j in range(6)], list(range(6)))
    vis = t.dv.get()
    vis[:6, 0] = [1 << j for j in range(6)]
    t.dv.put(vis)
    t.cache.set(0, 3, np.nan)                           # node 3 of the first, alone in its sight
    t.cache.set(1, 500 + 12, np.nan)                    # nodes 12.. of the second
    t.ready()
    got, (want, tol) = t.run(), t.want()
    hit = np.array([3] + list(range(6 + 12, 26)))
    rest = np.setdiff1d(np.arange(26), hit)
    assert not np.isfinite(got[hit]).any()
    assert np.isfinite(got[rest]).all() and (np.abs(got[rest] - want[rest]) <= tol[rest]).all()


@pytest.mark.parametrize("rows", ALL)
def test_sequences_without_nodes(rows):
    """Empty places in a batch, and rows behind the last sequence."""
    t = Tree(rows, 128, 2, [40, 300, 0, 9, 1000], [3, 0, 2, 0, 4], seed=16).ready()
    t.check()
    before = t.result()
    t.dstart.put(np.array([0, 3, 3, 5, 5, 5], np.int32))                    # the last sequence's four are nobody's now
    t.dout.put(np.full_like(t.dout.a, t.MARK))
    got = t.run()
    assert np.array_equal(got[:5].view(np.uint32), before[:5].view(np.uint32))
    assert (got[5:] == t.MARK).all()


class Repeated(tree_ref.Cache):
    """A long span whose table names a few pages again and again."""

    def repeat(self, n):
        self.page[0] = np.resize(self.page[0], -(-n // 64))

    def values(self, s, positions, v):
        p = np.asarray(positions)
        return self.pool[self.page[0][p // 64], v, :, p % 64]


@pytest.mark.parametrize("rows,n,hd", [(F32, 1 << 20, 64), (F32, 100003, 256), (EXACT, 1 << 18, 64), (EXACT, 70001, 128)])
def test_longest_spans(rows, n, hd):
    """The largest position counts: more pages than one part of a span holds."""
    t = Tree(rows, hd, 2, [37 * 64 - 3], [3], kind="chain", seed=17, nkv=1)
    t.cache.__class__ = Repeated
    t.cache.repeat(n)
    t.cached = [n - 3]
    t.dcached.put(np.array(t.cached, np.int32))
    t.args.max_positions = n
    t.ready()
    if rows == EXACT:
        t.check()
        return
    # no sum runs over all n: a wave of eight in a part has n / (8 parts) + 32 positions
    # at most, parts are of 256 pages at most; then 8 waves and 64 parts are added
    got, (want, tol) = t.run(), t.want()
    u, terms = 2.0 ** -24, n / (8 * -(-n // 16384)) + 32 + 8 + 64
    tol -= (2 * n - 2 * terms) * u * tree_abs(t)
    assert (tol > 0).all() and tol.max() < 1e-2 and (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


def tree_abs(t):
    """sum p |v| of every node and head."""
    out = np.zeros((3, t.NH, t.hd))
    for j in range(3):
        pos = np.concatenate([np.arange(t.cached[0]), t.cached[0] + np.arange(j + 1)])
        K, V = t.cache.values(0, pos, 0)[:, 0].astype(np.float64), t.cache.values(0, pos, 1)[:, 0].astype(np.float64)
        for h in range(t.NH):
            z = K @ t.q[j, h * t.hd:(h + 1) * t.hd].astype(np.float64) * t.scale
            w = np.exp(z - z.max())
            out[j, h] = w / w.sum() @ np.abs(V)
    return out


@pytest.mark.parametrize("rows", ALL)
def test_strides_and_neighbours(rows):
    Tree(rows, 64, 2, [100, 3], [7, 2], seed=9, pad=12).ready().check()


def test_exact_rows_of_any_size():
    """q and k beyond what three and four 8-bit digits hold take the same integers."""
    for qs, ks in ((1, 40), (1, 200), (1, 3000), (100, 1), (3000, 1)):
        t = Tree(EXACT, 64, 2, [150], [10], seed=10)
        g = np.random.default_rng(ks)
        t.cache.pool[:, 0] = np.rint(g.standard_normal(t.cache.pool[:, 0].shape) * ks * 65536)
        t.q[:, :256] *= qs
        t.dq.put(t.q)
        t.ready().check()


@pytest.mark.parametrize("rows", ALL)
def test_streams_and_graphs(rows):
    """Two calls on two streams at once, each with its own buffers; a captured call
    replayed with new inputs and lengths between eager ones."""
    a, b = Tree(rows, 128, 2, [700], [16], seed=11).ready(), Tree(rows, 128, 2, [900], [30], seed=12).ready()
    s1, s2 = Stream(), Stream()
    for _ in range(3):
        spkv.tree_attention(a.args, s1.h.value)
        spkv.tree_attention(b.args, s2.h.value)
    s1.sync(); s2.sync()
    a.check(a.result()); b.check(b.result())
    first = a.result()
    e = s1.capture(lambda st: spkv.tree_attention(a.args, st))
    for step, cached in enumerate((700, 699, 650, 700)):
        a.cached = [cached]
        a.dcached.put(np.array([cached], np.int32))
        a.dout.put(np.full_like(a.dout.a, a.MARK))
        s1.launch(e); s1.sync()
        got = a.check(a.result())
        spkv.tree_attention(b.args, 0)
        sync()
        b.check(b.result())
    assert np.array_equal(got.view(np.uint32), first.view(np.uint32))


@pytest.mark.parametrize("rows", ALL)
def test_repeats_are_equal(rows):
    t = Tree(rows, 128, 4, [2500], [24], seed=13).ready()
    first = t.run()
    for _ in range(4):
        assert np.array_equal(t.run().view(np.uint32), first.view(np.uint32))


def test_arrays_that_break_their_limits_stay_inside():
    """A node count beyond max_nodes, and positions beyond max_positions, change no
    byte outside the outputs."""
    t = Tree(F32, 64, 2, [100], [8], seed=14).ready()
    t.dstart.put(np.array([0, 1000], np.int32))
    t.run()
    t.dstart.put(np.array([5, 2], np.int32))
    t.run()
    t.dstart.put(np.array([0, 8], np.int32))
    t.dcached.put(np.array([1 << 30], np.int32))
    t.run()
    t.dcached.put(np.array([-5], np.int32))
    t.run()
    t.dcached.put(np.array([100], np.int32))
    t.check()


# ---------------------------------------------------------------- log probabilities
def logprob(x, scale=1.0, given=None, top=0, stride=None, stream=0, want=("entropy", "lse", "top")):
    R, V = x.shape
    stride = stride or V
    buf = np.full((R, stride), np.nan, np.float32)
    buf[:, :V] = x
    given = np.zeros((R, 0), np.int32) if given is None else given
    n = given.shape[1]
    d = dict(logits=Dev(buf), given=Dev(given), lp=Dev(np.full((R + 1, n), 7.0, np.float32)), ent=Dev(np.full(R + 1, 7.0, np.float32)),
             lse=Dev(np.full(R + 1, 7.0, np.float32)), ids=Dev(np.full((R + 1, top), 7, np.int32)), top=Dev(np.full((R + 1, top), 7.0, np.float32)))
    a = spkv.LogprobArgs(n_rows=R, vocab=V, n_given=n, n_top=top, scale=scale, logits=d["logits"].at, stride=stride,
                         given=d["given"].at if n else None, given_logprob=d["lp"].at if n else None,
                         entropy=d["ent"].at if "entropy" in want else None, lse=d["lse"].at if "lse" in want else None,
                         top_ids=d["ids"].at if top else None, top_logprob=d["top"].at if top and "top" in want else None)
    need = spkv.token_logprobs_work(a)
    d["work"] = Dev(np.full(need + 256, 0xA5, np.uint8))
    a.work, a.work_bytes = d["work"].at, need
    d["args"] = a
    spkv.token_logprobs(a, stream)
    assert (d["work"].get()[need:] == 0xA5).all()
    o = {k: d[k].get() for k in ("lp", "ent", "lse", "ids", "top")}
    assert all((v[R] == 7).all() for v in o.values())
    return {k: v[:R] for k, v in o.items()}, d


def check_logprobs(x, scale, given, top, o):
    """u = 2^-24.  d = y - M is off by 2 u (|y| + |M|) (the product, the difference),
    a term by that and 3 u of itself, the sum over V terms by V u more at worst:
    r is relatively off by e = 2 u (largest |y| + |M|) + (V + 8) u, log1p(r) and the
    entropy's second part by about e of r and of sum e^d |d| (+ 8 u).  Weighted, far
    terms count little, so the largest |y| that matters is taken over e^d above 2^-40."""
    lp, ent, lse, ids, tl = tree_ref.logprobs(x, scale, given, top)
    y = x.astype(np.float64) * np.float32(scale)
    m = y.max(1)
    u, V = 2.0 ** -24, x.shape[1]
    near = np.where(y > m[:, None] - 28, np.abs(y), 0).max(1)
    e = 2 * u * (near + np.abs(m)) + (V + 8) * u
    r = np.expm1(lse - m).astype(np.float64)
    dl = e * r / (1 + r) + 4 * u * np.log1p(r)
    assert np.array_equal(o["ids"], ids)
    assert (np.abs(o["lse"] - lse) <= dl + u * np.abs(lse) + 2 * u * np.abs(m)).all()
    for got, want, t in ((o["lp"], lp, given), (o["top"], tl, ids)):
        if got.size:
            yt = np.take_along_axis(y, t.astype(np.int64), 1)
            off = np.where(np.isfinite(yt), np.abs(got - want), 0)
            assert (off <= dl[:, None] + 2 * u * (np.abs(np.where(np.isfinite(yt), yt, 0)) + np.abs(m)[:, None]) + 2 * u * np.abs(np.where(np.isfinite(yt), want, 0))).all()
            assert np.array_equal(np.isfinite(yt), np.isfinite(got)) and (got[~np.isfinite(yt)] == -np.inf).all()
    first = np.log1p(r)
    second = np.maximum(ent.astype(np.float64) - first, 0)
    assert (np.abs(o["ent"] - ent) <= dl + (e + 2 * u * (near + np.abs(m)) + 8 * u) * (second + first) + 4 * u * ent).all()


@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (1, 2, 2), (3, 7, 5), (2, 64, 32), (5, 255, 20), (1, 257, 32), (4, 1000, 0), (2, 4096, 8), (3, 8193, 20),
                                     (2, 32768, 32), (7, 50001, 1), (1, 151936, 5), (2, 262144, 20), (65, 1031, 3)])
def test_logprobs(R, V, top):
    g = np.random.default_rng([R, V])
    x = (g.standard_normal((R, V)) * 3).astype(np.float32)
    given = g.integers(0, V, (R, 3)).astype(np.int32)
    for scale in (1.0, 1 / 0.7):
        o, _ = logprob(x, scale, given, top, stride=V + 5)
        check_logprobs(x, scale, given, top, o)


def test_logprobs_sure_and_masked_rows():
    g = np.random.default_rng(3)
    x = (g.standard_normal((6, 40000)) * 2).astype(np.float32)
    x[0, 77] = 30.0                                     # entropy far below 2^-24
    x[1, 39999] = 14.0
    x[2, 100:] = -np.inf                                # most tokens masked
    x[3, :] = -np.inf; x[3, 5] = -2.0; x[3, 9] = -2.0   # two left, equal
    x[4, :] = np.float32(1.5)                           # all equal
    x[5, :] = np.finfo(np.float32).min; x[5, 6] = 0.0   # masked by the lowest number
    given = np.tile(np.array([[77, 5, 9, 39999]], np.int32), (6, 1))
    o, _ = logprob(x, 1.0, given, 20)
    check_logprobs(x, 1.0, given, 20, o)
    assert abs(o["ent"][3] - np.log(2)) <= 2.0 ** -23 and 0 < o["ent"][0] < 1e-6
    assert list(o["ids"][4]) == list(range(20))


@pytest.mark.parametrize("V,left", [(9001, 3), (262144, 40), (8192, 31), (1024, 19), (8200, 12)])
def test_logprobs_masked_vocabularies(V, left):
    """Few logits above -infinity, some early: the alternatives go on with the
    lowest masked tokens."""
    g = np.random.default_rng([V, left])
    x = np.full((9, V), -np.inf, np.float32)
    for r in range(9):
        at = g.permutation(V if r % 3 else min(V, 200))[:left]
        x[r, at] = g.standard_normal(left)
    o, _ = logprob(x, 1.0, None, 20)
    check_logprobs(x, 1.0, None, 20, o)
    assert np.array_equal(o["ids"], np.argsort(-x, axis=1, kind="stable")[:, :20])


def test_logprobs_ties_go_to_the_lowest_token():
    x = np.zeros((3, 20000), np.float32)
    x[0, 1::2] = -0.0                                   # one zero
    x[1, [19999, 3, 8192, 8191, 12000]] = 4.0
    x[2, ::-1] = np.repeat(np.arange(2500, dtype=np.float32), 8)
    o, _ = logprob(x, 1.0, None, 32)
    assert list(o["ids"][0]) == list(range(32))
    assert list(o["ids"][1][:5]) == [3, 8191, 8192, 12000, 19999] and list(o["ids"][1][5:8]) == [0, 1, 2]
    assert np.array_equal(o["ids"], np.argsort(-x, axis=1, kind="stable")[:, :32])


def test_logprobs_sorted_rows():
    """Ascending and descending rows: every part of a row has its largest at one end."""
    x = np.stack([np.arange(30000), np.arange(30000)[::-1]]).astype(np.float32) * np.float32(1e-3)
    given = np.array([[0, 29999]] * 2, np.int32)
    o, _ = logprob(x, 1.0, given, 32)
    check_logprobs(x, 1.0, given, 32, o)


def test_logprobs_rows_without_a_distribution():
    x = np.zeros((5, 9000), np.float32)
    x[0, 4000] = np.nan
    x[1, 7] = np.inf
    x[2, :] = -np.inf
    x[3, 8] = np.nan; x[3, 3] = np.inf
    x[4, 2] = 1.0
    given = np.array([[4000, -1, 9000]] * 5, np.int32)
    o, _ = logprob(x, 1.0, given, 3)
    assert np.isnan(o["lse"][[0, 3]]).all() and o["lse"][1] == np.inf and o["lse"][2] == -np.inf
    assert np.isnan(o["ent"][:4]).all() and np.isnan(o["lp"][:4]).all() and np.isnan(o["top"][:4]).all()
    assert np.isfinite(o["ent"][4]) and np.isnan(o["lp"][4, 1:]).all() and np.isfinite(o["lp"][4, 0])
    assert list(o["ids"][0]) == [4000, 0, 1] and list(o["ids"][1]) == [7, 0, 1] and list(o["ids"][2]) == [0, 1, 2]
    assert list(o["ids"][3]) == [8, 3, 0] and list(o["ids"][4]) == [2, 0, 1]


def test_logprobs_optional_outputs_and_streams():
    g = np.random.default_rng(5)
    x = (g.standard_normal((3, 20000)) * 3).astype(np.float32)
    o, _ = logprob(x, 1.0, None, 4, want=())
    assert np.array_equal(o["ids"], np.argsort(-x, axis=1, kind="stable")[:, :4]) and (o["ent"] == 7).all() and (o["lse"] == 7).all() and (o["top"] == 7).all()
    given = g.integers(0, 20000, (3, 2)).astype(np.int32)
    ref, _ = logprob(x, 1.0, given, 4)
    s = Stream()
    _, d = logprob(x, 1.0, given, 4, stream=s.h.value)
    e = s.capture(lambda st: spkv.token_logprobs(d["args"], st))
    for k in range(3):
        z = (g.standard_normal(x.shape) * 3).astype(np.float32)
        d["logits"].put(z)
        s.launch(e); s.sync()
        o = {n: d[n].get()[:3] for n in ("lp", "ent", "lse", "ids", "top")}
        check_logprobs(z, 1.0, given, 4, o)
        logprob(x, 1.0, given, 4)


# ---------------------------------------------------------------- kept rows
@pytest.mark.parametrize("rows,hd", [(F32, 64), (F32, 256), (EXACT, 128), (SPINOR, 64), (SPINOR, 256)])
@pytest.mark.parametrize("ring", [0, 4])
def test_kept_rows(rows, hd, ring):
    """Lists of none, one, all and scattered nodes, over page borders and a ring's
    end; nothing else changes."""
    cached = [0, 60, 63, 250, 190]
    keeps = [[0], [0, 1, 5, 6, 30], list(range(20)) + [50], [], [3, 4, 9, 10, 11, 12, 13, 40, 41, 69]]
    nodes = [1, 31, 51, 5, 70]
    g = np.random.default_rng([hd, ring])
    caches = [tree_ref.Cache(g, rows, 3, hd, [c + n for c, n in zip(cached, nodes)], ring).upload() for _ in range(2)]
    lists = Dev(np.concatenate([c.lists.a for c in caches]))
    dc, ds = Dev(np.array(cached, np.int32)), Dev(np.cumsum([0] + [len(k) for k in keeps]).astype(np.int32))
    dk, dr = Dev(np.concatenate(keeps).astype(np.int32)), Dev(np.full(10, ring, np.int32))
    rb = caches[0].pool.strides[3]
    a = spkv.KeepArgs(n_kv_heads=3, row_bytes=rb, n_tables=10, n_seqs=5, max_keep=21, max_positions=400, tables=lists.at,
                      ring_pages=dr.at if ring else None, cached=dc.at, keep_start=ds.at, keep=dk.at)
    spkv.keep_rows(a)
    for c in caches:
        want = c.pool.copy()
        for s, k in enumerate(keeps):
            for i, j in enumerate(k):
                (p0, r0), (p1, r1) = c._at(s, cached[s] + i), c._at(s, cached[s] + j)
                want[p0, :, :, r0] = want[p1, :, :, r1]
        assert np.array_equal(c.dev.get().view(np.uint8), want.view(np.uint8))


def test_kept_rows_leave_out_what_does_not_ascend():
    g = np.random.default_rng(1)
    c = tree_ref.Cache(g, F32, 2, 64, [70]).upload()
    dc, ds = Dev(np.array([40], np.int32)), Dev(np.array([0, 6], np.int32))
    for keep in ([2, 1, 7, 7, 3, 9], [-1, 5, 4, 100000, 20, 30], [0, 0, 0, 1, 1, 2]):
        c.dev.put(c.pool)
        want, last = c.pool.copy(), -1
        for i, j in enumerate(keep):
            if j > last and j >= i and 40 + j < 70:
                last = j
                (p0, r0), (p1, r1) = c._at(0, 40 + i), c._at(0, 40 + j)
                want[p0, :, :, r0] = want[p1, :, :, r1]
        dk = Dev(np.array(keep, np.int32))
        spkv.keep_rows(spkv.KeepArgs(n_kv_heads=2, row_bytes=256, n_tables=1, n_seqs=1, max_keep=6, max_positions=70, tables=c.lists.at,
                                     cached=dc.at, keep_start=ds.at, keep=dk.at))
        assert np.array_equal(c.dev.get().view(np.uint32), want.view(np.uint32))
