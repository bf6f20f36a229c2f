"""Drafted trees and scores on a handle: sp_hipkv_tree_step against decode steps
along every node's path, sp_hipkv_tree_keep, sp_hipkv_score, and the three together
as a speculative decoder runs them.

Exact mode is bit for bit.  Float mode: a tree step and a decode step sum the same
n <= 560 f32 products per score or output in other orders, each sum off by at most
n 2^-24 = 3.3e-5 of its terms' magnitude; later layers and the logits inherit it:
1e-4 of the largest logit."""
import os

import numpy as np
import pytest

import orc
import spkv
from helpers import SMALL, prompt

pytestmark = pytest.mark.gpu


def same_bits(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32))


def close(a, b):
    return np.isfinite(a).all() and np.abs(a.astype(np.float64) - b).max() <= 1e-4 * np.abs(b).max()


class Rig:
    def __init__(self, tmp, shape, pmax=640, max_context=1024, vocab=None):
        # the batched LM head takes whole 64-row tiles of the vocabulary
        self.d = dict(SMALL[shape], vocab=vocab or -(-SMALL[shape]["vocab"] // 64) * 64)
        prefix = os.path.join(str(tmp), f"tree_{shape}_{self.d['vocab']}_{max_context}")
        if not os.path.exists(prefix + ".spt"):
            spkv.write_model(prefix, max_context=max_context, **self.d)
        spm, spt = prefix + ".spm", prefix + ".spt"
        self.spm, self.pmax = spm, pmax
        self.m = spkv.Model(spm, spt)
        self.s = spkv.Session(self.m, max_context)
        self.qm = spkv.l1().sp_session_qwen3_model(self.s.h)
        self.V, self.kvd = self.d["vocab"], self.d["n_kv_heads"] * self.d["head_dim"]

    def backend(self, exact, **kw):
        return spkv.Backend(self.qm, self.pmax, exact=exact, **kw)

    def close(self):
        self.s.close(); self.m.close()


def tree(n, seed, roots=1):
    g = np.random.default_rng(seed)
    return [-1 if i < roots else int(g.integers(max(0, (i - 1) // 3 - 1), max(1, (i + 2) // 2))) for i in range(n)]


def path(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


def log_softmax(x):
    x = x.astype(np.float64)
    z = x - x.max(-1, keepdims=True)
    return z - np.log(np.exp(z).sum(-1, keepdims=True))


SHAPES = ["qwen3-tiny", "gemma3-tiny", "qwen3-hd128", "qwen3-g4", "gemma3-hd256", "gemma3-w200", "gemma3-g4w130", "gemma3-w1", "qwen3-ragged"]


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_tree_step_equals_decode_steps(tmpdir_models, shape, exact):
    r = Rig(tmpdir_models, shape)
    same = same_bits if exact else close
    for ctx, n, roots in ((0, 3, 2), (37, 9, 1), (62, 40, 3), (250, 17, 1)):
        parents, toks = tree(n, ctx, roots), prompt(n, r.V, seed=ctx + 7)
        b = r.backend(exact)
        if ctx:
            b.prefill(prompt(ctx, r.V, seed=3))
        lg, nxt, lp = b.tree_step(toks, parents, r.V)
        assert b.position() == ctx and np.array_equal(nxt, lg.argmax(1))
        leaves = [i for i in range(n) if i not in parents]
        seen, ref = {}, np.zeros(r.V, np.float32)
        for leaf in leaves[:6]:
            f = b.fork()                                # the context alone: forks drop a pending tree
            for i in path(parents, leaf):
                f.decode(int(toks[i]), ref)
                assert same(lg[i], ref), (ctx, n, i)
                seen[i] = ref.copy()
                if parents[i] >= 0:
                    want = log_softmax(seen[parents[i]])[toks[i]]
                    # the f32 logits' spread, V terms each off by 2^-23 of the range at most
                    assert abs(lp[i] - want) <= (1e-5 if exact else 2e-4 * np.abs(ref).max())
                else:
                    assert np.isnan(lp[i])
            f.close()
        b.close()
    r.close()


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("shape", ["qwen3-tiny", "gemma3-tiny", "gemma3-hd256", "qwen3-g4"])
def test_kept_path_is_as_if_decoded(tmpdir_models, shape, exact):
    r = Rig(tmpdir_models, shape)
    same = same_bits if exact else close
    b, one = r.backend(exact), r.backend(exact)
    pr = prompt(57, r.V, seed=5)
    b.prefill(pr); one.prefill(pr)
    lg, ref = np.zeros(r.V, np.float32), np.zeros(r.V, np.float32)
    for step in range(4):
        n = (5, 30, 12, 64)[step]
        parents, toks = tree(n, step), prompt(n, r.V, seed=100 + step)
        b.tree_step(toks, parents)
        keep = path(parents, (0, n - 1, n // 2, n - 2)[step])
        b.tree_keep(keep)
        for i in keep:
            one.decode(int(toks[i]), ref)
        assert b.position() == one.position()
        for l in range(r.d["n_layers"]):
            for x, y in zip(b.read_kv(l, 0, b.position(), r.kvd), one.read_kv(l, 0, one.position(), r.kvd)):
                assert same(x, y), (step, l)
        t = int(ref.argmax())
        b.decode(t, lg); one.decode(t, ref)
        assert same(lg, ref)
    # a dropped tree leaves the context as it was
    b.tree_step([1, 2, 3], [-1, 0, 1])
    b.tree_keep([])
    b.decode(7, lg); one.decode(7, ref)
    assert same(lg, ref)
    b.close(); one.close(); r.close()


@pytest.mark.parametrize("exact", [True, False])
def test_window_rings_and_trees(tmpdir_models, exact):
    """Trees behind a context that has wrapped the window layers' ring."""
    r = Rig(tmpdir_models, "gemma3-hd256")
    same = same_bits if exact else close
    b, one = r.backend(exact), r.backend(exact)
    spkv.check(spkv.kv().sp_hipkv_set_max_rewind(b.h, 64), "max_rewind")
    pr = prompt(400, r.V, seed=8)
    b.prefill(pr); one.prefill(pr)
    ref = np.zeros(r.V, np.float32)
    for step in range(6):
        n = (33, 20, 33, 1, 2, 33)[step]
        parents, toks = tree(n, 40 + step), prompt(n, r.V, seed=200 + step)
        lg, _, _ = b.tree_step(toks, parents, r.V)
        keep = path(parents, n - 1)
        for i in keep:
            one.decode(int(toks[i]), ref)
            assert same(lg[i], ref), step
        b.tree_keep(keep)
    # more nodes than the ring keeps behind the window
    with pytest.raises(RuntimeError, match="window ring"):
        b.tree_step(prompt(128, r.V), tree(128, 1))
    assert b.position() == one.position()
    lg = np.zeros(r.V, np.float32)
    b.decode(3, lg); one.decode(3, ref)
    assert same(lg, ref)
    b.close(); one.close(); r.close()


def test_spinor_sessions(tmpdir_models):
    """Exact: bit for bit.  Float: the oracle attends the rows that the tree step
    stored (its codes may differ from a decode step's by a float's rounding)."""
    r = Rig(tmpdir_models, "gemma3-hd256")
    pr, n = prompt(70, r.V, seed=4), 25
    parents, toks = tree(n, 9), prompt(n, r.V, seed=11)
    b = r.backend(True, kv_codec=spkv.KV_SPINOR)
    b.prefill(pr)
    lg, _, _ = b.tree_step(toks, parents, r.V)
    f, ref = b.fork(), np.zeros(r.V, np.float32)
    keep = path(parents, n - 1)
    for i in keep:
        f.decode(int(toks[i]), ref)
        assert same_bits(lg[i], ref)
    f.close(); b.close()
    b = r.backend(False, kv_codec=spkv.KV_SPINOR)
    b.prefill(pr)
    lg, _, _ = b.tree_step(toks, parents, r.V)
    b.tree_keep(keep)
    o = orc.Oracle(r.spm, r.pmax, orc.FLOAT, kv_flags=orc.KV_SPINOR)
    o.set_kv_forced(True)
    for l in range(r.d["n_layers"]):
        o.set_kv(l, 0, *b.read_kv(l, 0, b.position(), r.kvd))
    o.set_pos(70)
    for i in keep:
        ref = o.step(int(toks[i]))
        assert np.abs(lg[i] - ref).max() <= 1e-3 * np.abs(ref).max()
    o.close(); b.close(); r.close()


def test_forks_do_not_see_a_kept_path(tmpdir_models):
    """A fork taken while the tree is pending shares its pages: keeping a path
    copies what it writes."""
    r = Rig(tmpdir_models, "qwen3-hd128")
    b = r.backend(True)
    b.prefill(prompt(60, r.V, seed=2))
    parents, toks = tree(30, 3), prompt(30, r.V, seed=6)
    b.tree_step(toks, parents)
    f, g = b.fork(), b.fork()
    before = [f.read_kv(l, 0, 60, r.kvd) for l in range(2)]
    with pytest.raises(RuntimeError, match="no tree is pending"):
        f.tree_keep([0])
    keep = path(parents, 29)
    b.tree_keep(keep)
    for l in range(2):
        for x, y in zip(f.read_kv(l, 0, 60, r.kvd), before[l]):
            assert same_bits(x, y)
    lg, ref = np.zeros(r.V, np.float32), np.zeros(r.V, np.float32)
    for i in keep:
        f.decode(int(toks[i]), ref)
    f.decode(9, ref); b.decode(9, lg)
    assert same_bits(lg, ref)
    for h in (b, f, g):
        h.close()
    r.close()


def test_what_ends_a_pending_tree(tmpdir_models):
    r = Rig(tmpdir_models, "qwen3-tiny")
    lg = np.zeros(r.V, np.float32)
    b = r.backend(False)
    b.prefill([1, 2, 3, 4])
    ends = [lambda: b.decode(5, lg), lambda: b.prefill([6, 7]), lambda: b.rewind(1), lambda: b.greedy(3, 2), lambda: b.score([4, 5]),
            lambda: spkv.Backend.decode_batch([b], [3], r.V), lambda: b.tree_keep([]),
            lambda: spkv.check(spkv.kv().sp_hipkv_decode_step_noalloc(b.h, 4, spkv.ptr(lg)), "noalloc")]
    for end in ends:
        b.tree_step([1, 2], [-1, 0])
        end()
        with pytest.raises(RuntimeError, match="no tree is pending"):
            b.tree_keep([0])
    b.rewind(b.position())
    b.tree_step([1, 2], [-1, 0])                        # behind nothing
    spkv.check(spkv.kv().sp_hipkv_set_mode(b.h, 1), "set_mode")
    with pytest.raises(RuntimeError, match="no tree is pending"):
        b.tree_keep([0])
    b.close(); r.close()


def test_tree_refusals(tmpdir_models):
    r = Rig(tmpdir_models, "qwen3-tiny", pmax=100)
    b = r.backend(False)
    b.prefill(prompt(50, r.V))
    for toks, parents, why in (([1, 2], [-1, 1], "parents"), ([1, 2], [-1, -2], "parents"), ([1], [0], "parents"), ([r.V], [-1], "vocabulary"),
                               ([-1], [-1], "vocabulary"), ([], [], "1 to 128"), ([1] * 129, [-1] * 129, "1 to 128"),
                               ([1] * 51, list(range(-1, 50)), "context full"), ([1] * 66, [-1] + [0] * 65, "context full")):
        with pytest.raises(RuntimeError, match=why):
            b.tree_step(toks, parents)
    parents = [-1, 0, 0, 1, 2]
    b.tree_step([1, 2, 3, 4, 5], parents)
    for bad in ([1], [0, 3], [0, 1, 4], [0, 0], [5], [-1], [0, 2, 4, 4]):
        with pytest.raises(RuntimeError, match="no path"):
            b.tree_keep(bad)
    b.tree_keep([0, 2, 4])
    assert b.position() == 53
    kv = spkv.kv()
    assert kv.sp_hipkv_tree_step(None, None, None, 1, None, None, None) != 0 and kv.sp_hipkv_tree_keep(None, None, 0) != 0
    assert kv.sp_hipkv_score(None, None, None, 0, 0, None, None, None, None) != 0
    with pytest.raises(RuntimeError, match="n_top"):
        b.score([1, 2], n_top=33)
    with pytest.raises(RuntimeError, match="given"):
        b.score([1, 2], given=[3, r.V])
    with pytest.raises(RuntimeError, match="context full"):
        b.score([1] * 48)
    assert b.position() == 53
    b.close()
    odd = Rig(tmpdir_models, "qwen3-tiny", vocab=1000)
    w = odd.backend(False)
    w.prefill([1, 2, 3])
    for f in (lambda: w.tree_step([1], [-1]), lambda: w.score([1])):
        with pytest.raises(RuntimeError, match="batched path"):
            f()
    w.close(); odd.close()
    w = r.backend(False)
    w.set_recall(64, 16, 2, 8)
    w.prefill([1, 2, 3])
    with pytest.raises(RuntimeError, match="recall"):
        w.tree_step([1], [-1])
    w.close(); r.close()


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("shape", ["qwen3-hd128", "gemma3-tiny"])
def test_score_equals_decode_steps(tmpdir_models, shape, exact):
    r = Rig(tmpdir_models, shape)
    toks = prompt(300, r.V, seed=21)
    b, one = r.backend(exact), r.backend(exact)
    got = [b.score(toks[:1], n_top=4), b.score(toks[1:130], n_top=4), b.score(toks[130:], n_top=4)]
    lp, ent, ids, tl = (np.concatenate([g[k] for g in got]) for k in range(4))
    assert b.position() == 300 and np.isnan(lp[[0, 129, 299]]).all()
    given = prompt(20, r.V, seed=22)
    given[3] = -1
    b.rewind(20)
    glp = b.score(toks[280:], given=given)[0]
    lg = np.zeros(r.V, np.float32)
    for i in range(300):
        one.decode(int(toks[i]), lg)
        p = log_softmax(lg)
        # the operator on f32 logits: 1e-5 (tests of the operator itself); float mode: the logits' own 1e-4
        t = 1e-5 if exact else 2e-4 * np.abs(lg).max()
        if i not in (0, 129, 299):
            assert abs(lp[i] - p[toks[i + 1]]) <= t
        assert abs(ent[i] + (np.exp(p) * p).sum()) <= (2e-5 if exact else t)
        assert np.abs(tl[i] - p[ids[i]]).max() <= t
        if exact:
            assert np.array_equal(ids[i], np.argsort(-lg, kind="stable")[:4])
        if i >= 280:
            assert np.isnan(glp[i - 280]) if given[i - 280] < 0 else abs(glp[i - 280] - p[given[i - 280]]) <= t
    for l in range(r.d["n_layers"]):
        for x, y in zip(b.read_kv(l, 0, 300, r.kvd), one.read_kv(l, 0, 300, r.kvd)):
            assert (same_bits if exact else close)(x, y)
    b.close(); one.close(); r.close()


def test_score_takes_any_number_of_tokens_in_any_order(tmpdir_models):
    """A vocabulary where 127 rows take more work than 128 do: long, short and long
    calls on one handle, and a handle beside it."""
    r, beside = Rig(tmpdir_models, "qwen3-tiny", vocab=32768), Rig(tmpdir_models, "qwen3-tiny", vocab=32768)
    g = np.random.default_rng(41)
    toks = g.integers(0, r.V, 255).astype(np.int32)
    h, other = r.backend(True), beside.backend(True)
    other.prefill(toks[:40])
    want, again = np.zeros(r.V, np.float32), np.zeros(r.V, np.float32)
    other.decode(int(toks[40]), want)
    other.rewind(1)
    parts = [h.score(toks[a:b], given=toks[a + 1:b + 1], n_top=32) for a, b in ((0, 128), (128, 254))]
    h.rewind(254)
    pieces = [h.score(toks[a:b], given=toks[a + 1:b + 1], n_top=32) for a, b in ((0, 1), (1, 128), (128, 190), (190, 254))]
    for k in range(4):
        x, y = (np.concatenate([p[k] for p in q]) for q in (parts, pieces))
        # the same logits, the operator's sums in another order: 1e-5 each (its own tests)
        assert np.array_equal(x, y) if x.dtype == np.int32 else np.abs(x - y).max() <= 2e-5
    other.decode(int(toks[40]), again)
    assert same_bits(again, want)
    h.close(); other.close(); r.close(); beside.close()


def test_speculative_decoding_gives_the_greedy_tokens(tmpdir_models):
    """Exact mode: drafts from a table of what followed a token before, verified as
    a tree with wrong guesses beside them; the tokens are the greedy loop's."""
    r = Rig(tmpdir_models, "gemma3-w200", pmax=512)
    pr = prompt(40, r.V, seed=31)
    ref = r.backend(True)
    ref.prefill(pr[:-1])
    want, _ = ref.greedy(int(pr[-1]), 120)
    b = r.backend(True)
    b.prefill(pr[:-1])
    g, out, last, steps = np.random.default_rng(1), [], int(pr[-1]), 0
    while len(out) < 120:
        # the true continuation up to a random length, then wrong tokens; siblings everywhere
        good, at = int(g.integers(0, 6)), len(out)
        toks, parents, on = [last], [-1], 0
        for k in range(5):
            true = int(want[at + k]) if k < good and at + k < 120 else int(g.integers(0, r.V))
            for t in (int(g.integers(0, r.V)), true, int(g.integers(0, r.V))):
                toks.append(t); parents.append(on)
            on = len(toks) - 2
        _, nxt, lp = b.tree_step(toks, parents)
        keep, node = [0], 0
        while True:
            kid = [i for i, p in enumerate(parents) if p == node and toks[i] == nxt[node]]
            out.append(int(nxt[node]))
            if not kid:
                break
            node = kid[0]
            keep.append(node)
        b.tree_keep(keep)
        last, steps = out[-1], steps + 1
    assert out[:120] == [int(t) for t in want] and steps < 90
    # the scores of the text agree with what the steps said
    b.rewind(b.position())
    text = list(pr) + out[:119]
    lp, ent, ids, _ = b.score(text, n_top=1)
    assert [int(i) for i in ids[len(pr) - 1:, 0]] == out[:120]
    for h in (ref, b):
        h.close()
    r.close()
