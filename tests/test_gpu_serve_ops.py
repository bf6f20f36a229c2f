"""The operators of serving from a paged cache on device memory against plain 64-bit
implementations (tests/serve_ref.py, where the tolerances are derived)."""
import ctypes

import numpy as np
import pytest

import spkv
import tree_ref
from devmem import Dev, Stream, hip, sync
from serve_ref import B, BLOCK, PAGE, U, Append, Cache8, Cached, Packed, Prompt, cache_attention, close, packed_start, prepared, prompt_attention

pytestmark = pytest.mark.gpu
F32, BF16, BLOCK8, ROWS = spkv.F32, spkv.BF16, spkv.ROWS_BLOCK8, spkv.ROWS_F32
TYPES = [F32, BF16]
HEADS = [(64, 1), (64, 4), (128, 2), (128, 4), (256, 2), (256, 16), (128, 3), (64, 7)]


def rng(*seed):
    return np.random.default_rng(list(seed))


def f32_cache(g, nkv, hd, lens, ring=0):
    c = tree_ref.Cache(g, ROWS, nkv, hd, lens, ring)
    c.pool[:] = g.standard_normal(c.pool.shape)
    return c.upload()


# ---------------------------------------------------------------- append
def appended(g, rows, typ, hd, G, cached, counts, ring=0, nkv=2, room=None, **kw):
    if rows == BLOCK8:
        c = Cache8(g, nkv, hd, cached, ring, room or [a + b for a, b in zip(cached, counts)]).upload()
    else:
        c = f32_cache(g, nkv, hd, room or [a + b for a, b in zip(cached, counts)], ring)
    return Append(g, c, rows, typ, hd, G, cached, counts, **kw)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("rows", [BLOCK8, ROWS])
@pytest.mark.parametrize("hd,G", HEADS)
def test_append_heads(rows, typ, hd, G):
    appended(rng(1, hd, G), rows, typ, hd, G, [70, 0], [9, 100]).check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("rows", [BLOCK8, ROWS])
@pytest.mark.parametrize("cached,counts", [([0], [1]), ([0], [16]), ([15], [1]), ([15], [2]), ([63], [2]), ([64], [1]), ([17], [130]), ([1], [63]),
                                           ([0, 5, 300, 64, 7], [3, 0, 17, 64, 0]), ([0] * 70, [1] * 70), ([100] * 3, [0, 0, 5]), ([3, 90], [200, 1])])
def test_append_lengths(rows, typ, cached, counts):
    appended(rng(2, len(cached)), rows, typ, 128, 2, cached, counts).check()


@pytest.mark.parametrize("rows", [BLOCK8, ROWS])
@pytest.mark.parametrize("kw", [dict(norm=False), dict(freq=False), dict(norm=False, freq=False), dict(q_out=False), dict(k_out=None), dict(q_out="same", k_out="same"),
                                dict(pad=8), dict(q_out=False, k_out=None, pad=16), dict(more_tokens=5)])
def test_append_forms(rows, kw):
    for typ in TYPES:
        appended(rng(3), rows, typ, 64, 2, [20, 50], [30, 5], **kw).check()


@pytest.mark.parametrize("typ", TYPES)
def test_append_far_positions(typ):
    """The angle of a position near 2^20: off by 0.06 in 32 bits."""
    g = rng(4)
    c = Cache8(g, 1, 128, [PAGE], 1, [PAGE])                 # a ring of one page holds any position
    c.upload()
    Append(g, c, BLOCK8, typ, 128, 2, [(1 << 20) - 20], [20], base=1e6).check()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_append_step_by_step(hd):
    """Tokens one by one, each against what it should leave: scales grow, earlier codes are
    rounded again; and the values stay within a step and a half of the block's last scale."""
    for typ in TYPES:
        g = rng(5)
        n, nkv = 40, 2
        c = Cache8(g, nkv, hd, [0], 0, [n]).upload()
        grow = (2.0 ** (np.arange(n) % BLOCK / 2))[:, None, None]
        k, v = g.standard_normal((n, nkv, hd)) * grow, g.standard_normal((n, nkv, hd)) * grow[::-1]
        for t in range(n):
            c.lens = [t]
            Append(g, c, BLOCK8, typ, hd, 1, [t], [1], norm=False, freq=False, k=k[t:t + 1], v=v[t:t + 1]).check()
        for which, x in ((0, k), (1, v)):
            codes, sc = c.values(0, range(n), which)
            x = Packed(x, typ).values()
            assert (np.abs(codes * sc[..., None] - x) <= 1.5 * sc[..., None]).all()


def test_append_extremes():
    """Zeros, the smallest and largest numbers, and values around 127 of a power of two."""
    g = rng(6)
    vals = [0.0, -0.0, 1e-45, 1.1754944e-38, 2.0 ** -119, 127 * 2.0 ** -126, 127.0, np.nextafter(np.float32(127), np.float32(200)), 63.5, 64.0, 3.4028235e38, -3e38]
    n = len(vals)
    x = np.zeros((n * BLOCK, 1, 64))
    for i, a in enumerate(vals):
        x[i * BLOCK:(i + 1) * BLOCK, 0] = a * (g.random((BLOCK, 64)) < 0.5)
    c = Cache8(g, 1, 64, [0], 0, [n * BLOCK]).upload()
    a = Append(g, c, BLOCK8, F32, 64, 1, [0], [n * BLOCK], norm=False, freq=False, k=x, v=x)
    a.check()
    assert np.isfinite(c.s[c.page[0]][:, 0, 0].reshape(-1)[:n]).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd", [64, 256])
def test_append_values_that_are_not_finite(hd, bad):
    """Their block gets a scale of NaN, keeps it, and is started anew at its first position."""
    g = rng(7)
    x = g.standard_normal((40, 2, hd))
    x[5, 0, 3], x[33, 1, 60] = bad, bad
    for typ in TYPES:
        c = Cache8(g, 2, hd, [0], 0, [48]).upload()
        a = Append(g, c, BLOCK8, typ, hd, 1, [0], [40], norm=False, freq=False, k_out=None, k=x, v=x)
        a.check()
        assert np.isnan(c.s).sum() >= 4
        one = g.standard_normal((1, 2, hd))
        Append(g, c, BLOCK8, typ, hd, 1, [40], [1], norm=False, freq=False, k=one, v=one).check()
        again = g.standard_normal((8, 2, hd))
        Append(g, c, BLOCK8, typ, hd, 1, [32], [8], norm=False, freq=False, k=again, v=again).check()
        pg, i = c.block(0, 2)
        assert np.isfinite(c.s[pg, :, :, i]).all()


@pytest.mark.parametrize("rows", [BLOCK8, ROWS])
@pytest.mark.parametrize("cached,counts,ring", [([100, 640], [40, 3], 3), ([0], [1000], 3), ([70], [64 * 3], 3), ([5000], [200], 1), ([130], [1], 2)])
@pytest.mark.parametrize("hd", [64, 256])
def test_append_rings(hd, rows, cached, counts, ring):
    g = rng(8, ring)
    if rows == BLOCK8:
        c = Cache8(g, 2, hd, cached, ring).upload()
    else:
        c = f32_cache(g, 2, hd, [64 * ring] * len(cached), ring)
    Append(g, c, rows, F32, hd, 2, cached, counts).check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("cached,counts", [([0], [1]), ([15], [2]), ([7], [3]), ([8], [8]), ([62], [3]), ([17], [130]), ([0, 5, 300, 9, 7], [3, 0, 17, 64, 0]), ([100] * 3, [0, 0, 5])])
def test_append_wide_heads(typ, cached, counts):
    appended(rng(10, len(cached)), BLOCK8, typ, 256, 2, cached, counts).check()


def test_append_more_heads_than_a_wave():
    appended(rng(9), BLOCK8, BF16, 64, 1, [3], [20], nkv=70).check()


# ---------------------------------------------------------------- prompts
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd,G", HEADS)
def test_prompt_heads(typ, hd, G):
    Prompt(rng(11, hd, G), typ, hd, G, [70, 9]).check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("counts", [[1], [2], [31], [32], [33], [63], [64], [65], [129], [200], [1, 1, 1], [0, 5, 0, 0, 70, 1, 0], [40] * 20, [3] * 70])
def test_prompt_lengths(typ, counts):
    Prompt(rng(12, len(counts)), typ, 128, 2, counts).check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_long(typ, hd):
    Prompt(rng(13, hd), typ, hd, 2, [700], nkv=1).check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
def test_prompt_windows(typ, window):
    Prompt(rng(14, window), typ, 64, 2, [300, 17], window=window, nkv=1).check()
    Prompt(rng(15, window), typ, 128, 3, [130], window=window, nkv=1).check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0, 1e-30])
def test_prompt_scales(typ, scale):
    Prompt(rng(16), typ, 64, 2, [100, 3], scale=scale).check()


@pytest.mark.parametrize("typ", TYPES)
def test_prompt_strides_and_rows_behind(typ):
    Prompt(rng(17), typ, 128, 2, [50, 20], pad=8, more_tokens=6).check()


@pytest.mark.parametrize("typ", TYPES)
def test_prompt_peaked_weights(typ):
    """Scores in the hundreds: the running maximum moves far, weights vanish."""
    Prompt(rng(18), typ, 64, 2, [300], wide=60.0).check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_prompt_values_that_are_not_attended(typ, hd, bad):
    """K and V rows of later tokens, of tokens before the window and of other sequences hold
    values that are not finite: tokens that do not attend them are as without, the others
    are not finite (from K everywhere, from V in its column)."""
    g = rng(19, hd)
    counts, window, G = [90, 80], 40, 2
    p = Prompt(g, typ, hd, G, counts, window=window, nkv=1)
    clean, tol = p.want()
    k, v = p.k.values().copy(), p.v.values().copy()
    k[20, 0, 5] = bad                                       # attended by tokens 20 .. 59 of sequence 0
    v[70, 0, 7] = bad                                       # by 70 .. 89
    v[100, 0, :] = bad                                      # token 10 of sequence 1: 10 .. 49
    p.k, p.v = Packed(k, typ), Packed(v, typ)
    p.args.k, p.args.k_stride, p.args.v, p.args.v_stride = p.k.at, p.k.stride, p.v.at, p.v.stride
    got = p.run()
    hit = np.zeros(got.shape, bool)
    hit[70:90, :, 7] = True
    hit[100:140] = True
    gone = np.zeros(got.shape, bool)
    gone[20:60] = True
    if np.isinf(bad) and typ == BF16:                       # scores of -inf have weight 0
        assert 0 < np.isfinite(got[20:60]).all(-1).sum() < 40 * G
    else:
        assert not np.isfinite(got[gone]).any()
    assert not np.isfinite(got[hit & ~gone]).any()
    rest = ~(hit | gone)
    assert (np.abs(got - clean)[rest] <= tol[rest]).all()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd,counts", [(64, [90, 40]), (128, [90, 40]), (256, [90, 40]), (64, [300]), (128, [300])])
@pytest.mark.parametrize("big", [1e10, 1e25, 3e38])
def test_prompt_large_values_that_are_not_attended(typ, hd, counts, big):
    """Finite, and far above what the tokens before them, behind their window and of other
    sequences attend, whose bounds do not know of them."""
    g = rng(23, hd)
    T = sum(counts)
    k, v = g.standard_normal((T, 2, hd)), g.standard_normal((T, 2, hd))
    v[33, 0] *= big / 10
    v[60, 1, 3] = -big
    k[75, 1] = big * 0.9
    p = Prompt(g, typ, hd, 2, counts, window=20, k=k, v=v)
    got, (want, tol) = p.run(), p.want()
    fine = np.ones(T, bool)
    fine[33:min(53, counts[0])] = fine[60:80] = fine[75:95] = False    # those that attend them (some of 1e25 and more are not finite)
    assert fine.sum() > 60 and (np.abs(got - want)[fine] <= tol[fine]).all()
    if big == 1e10:
        few = ~fine
        few[75:95] = False
        assert (np.abs(got - want)[few] <= tol[few]).all()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("low", [1, 40, 200])
def test_prompt_large_values_of_small_weight(typ, hd, low):
    """V of 1e20 where the weights are e^-80, first or for long the only ones: what is left of them
    is 1e-15 beside the others' 1."""
    g = rng(24, hd, low)
    q, k, v = g.standard_normal((300, 2, hd)), g.standard_normal((300, 1, hd)), g.standard_normal((300, 1, hd))
    q[..., 0], k[..., 0], k[:low, 0, 0] = 30, 0, -80 / 30 * hd ** 0.5
    v[:low] *= 1e20
    Prompt(g, typ, hd, 2, [300], nkv=1, q=q, k=k, v=v).check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd,n,nkv", [(64, 400, 48), (128, 300, 64), (128, 250, 160), (128, 900, 12), (256, 230, 150)])
def test_prompt_long_with_many_heads(typ, hd, n, nkv):
    """Too many rows for a workgroup a unit."""
    Prompt(rng(25, hd), typ, hd, 1, [n], nkv=nkv).check()


@pytest.mark.parametrize("hd,window", [(128, 0), (128, 300)])
def test_prompt_of_many_workgroups(hd, window):
    """One sequence whose rows fill the device more than once; a few of its heads and tokens are compared."""
    g = rng(27, window)
    n, nkv = 2000, 60
    p = Prompt(g, BF16, hd, 1, [n], nkv=nkv, window=window)
    got, few = p.run(), [0, 7, nkv - 1]
    q, k, v = (x.values()[:, few] for x in (p.q, p.k, p.v))
    for t in (0, 1, 63, 64, 255, 256, 257, 300, 1023, 1500, n - 1):
        lo = max(0, t - window + 1) if window else 0
        want, tol = prompt_attention(q[lo:t + 1], k[lo:t + 1], v[lo:t + 1], [t + 1 - lo], 0, p.scale, BF16) if t < 300 else (None, None)
        if want is None:                                    # the last token alone: the others' rows cost most of the time
            for h in range(len(few)):
                K, V, x = (a.astype(np.float64) for a in (k[lo:t + 1, h], v[lo:t + 1, h], q[t, h]))
                z = K @ x * p.scale
                w = np.exp(z - z.max())
                w /= w.sum()
                o, r = w @ V, w @ np.abs(V)
                d = (6 * hd + 20) * U * p.scale * (np.abs(K) @ np.abs(x)).max() + 4 * U * np.abs(z - z.max()).max()
                bound = ((4 * d + (12 * len(z) + 64) * U) * r + U * np.abs(o) + B * r) * (1 + B) + B * np.abs(o)
                assert (np.abs(got[t, few[h]] - o) <= bound).all()
        else:
            assert (np.abs(got[t, few] - want[-1]) <= tol[-1]).all()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n,nkv", [(200, 40), (200, 100)])
def test_prompt_wide_heads_in_a_window(typ, n, nkv):
    Prompt(rng(26, nkv), typ, 256, 1, [n, 3], window=70, nkv=nkv).check()


@pytest.mark.parametrize("typ", TYPES)
def test_prompt_nothing_read_behind_the_last_row(typ):
    """k and v that end with the last sequence: what lies behind is not a row of theirs."""
    g = rng(20)
    p = Prompt(g, typ, 64, 1, [33], nkv=1)
    p.k, p.v = Packed(p.k.values(), typ, 0, 0), Packed(p.v.values(), typ, 0, 0)
    p.args.k, p.args.k_stride, p.args.v, p.args.v_stride = p.k.at, p.k.stride, p.v.at, p.v.stride
    p.check()


# ---------------------------------------------------------------- cache
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd,G", HEADS)
def test_cache_heads(typ, hd, G):
    Cached(rng(21, hd, G), typ, hd, G, [70, 5], [9, 1]).ready().check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("cached,counts", [([0], [1]), ([0], [5]), ([1], [1]), ([15], [1]), ([63], [2]), ([64], [1]), ([62], [67]), ([128], [64]),
                                           ([1000], [3]), ([515], [130]), ([0, 5, 300, 64, 9], [3, 0, 17, 40, 0]), ([33] * 40, [1] * 40)])
def test_cache_lengths(typ, cached, counts):
    Cached(rng(22, len(cached)), typ, 128, 2, cached, counts).ready().check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_cache_long(typ, hd):
    """Spans cut into parts, and every count of tokens around a tile."""
    for n in (1, 8, 9, 33):
        Cached(rng(23, n), typ, hd, 2, [5003], [n], nkv=1).ready().check()


@pytest.mark.parametrize("typ", TYPES)
def test_cache_ragged_parts(typ):
    Cached(rng(24), typ, 64, 2, [9000, 10, 700, 0, 2500], [2, 1, 3, 1, 0], nkv=1).ready().check()


def test_cache_longest():
    """Positions up to 2^17: page tables of 2048 entries."""
    Cached(rng(25), F32, 64, 1, [(1 << 17) - 1], [1], nkv=1).ready().check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("cached,ring", [(40, 0), (200, 0), (1000, 0), (1000, 4), (127, 4), (2000, 3)])
def test_cache_windows(typ, cached, ring):
    Cached(rng(26, cached), typ, 128, 2, [cached, cached + 1], [24, 3], window=100, ring=ring).ready().check()
    Cached(rng(27, cached), typ, 64, 4, [cached], [24], window=1, ring=ring).ready().check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_cache_scales(typ, scale):
    Cached(rng(28), typ, 64, 2, [100, 3], [2, 2], scale=scale, wide=3.0).ready().check()


@pytest.mark.parametrize("typ", TYPES)
def test_cache_strides_and_rows_behind(typ):
    for cached in ([70, 9], [6000, 9]):                     # one part, and several
        Cached(rng(29), typ, 128, 2, cached, [5, 2], pad=8, more_tokens=6).ready().check()


def test_cache_scales_far_apart():
    """Blocks whose scales differ by 2^60, in K and in V, zero scales among them."""
    g = rng(30)
    t = Cached(g, F32, 64, 2, [500], [2], nkv=1)
    for pg in t.cache.page[0]:
        t.cache.s[pg, 1] *= 2.0 ** g.choice([-30, 0, 30], 4)
        t.cache.s[pg, 0] *= 2.0 ** g.choice([-30, 0], 4)
    t.cache.s[t.cache.page[0][2], :, 0, 1] = 0
    t.ready().check()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_cache_scales_that_are_not_finite(bad):
    """A block's scale of NaN or infinity reaches the tokens that attend one of its positions, all
    of their values; tokens before it and those whose window is past it are as without."""
    for which in (0, 1):
        for typ in TYPES:
            g = rng(31, which)
            t = Cached(g, typ, 64, 2, [100], [40], window=30, nkv=1)
            want, tol = t.want()
            pg, i = t.cache.block(0, 7)                      # positions 112 .. 127, from token 12 on
            t.cache.s[pg, which, 0, i] = bad
            t.ready()
            got = t.run()
            assert not np.isfinite(got[12:]).any()
            assert (np.abs(got - want)[:12] <= tol[:12]).all()
            late = Cached(g, typ, 64, 2, [157], [3], window=30, nkv=1)    # windows from 128 on
            pg, i = late.cache.block(0, 7)
            late.cache.s[pg, which, 0, i] = bad
            late.ready().check()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_cache_q_that_is_not_finite(bad):
    t = Cached(rng(33), F32, 64, 2, [100], [3], nkv=1)
    want, tol = t.want()
    q = t.q.values().copy()
    q[1, 0, 9] = bad
    t.q = Packed(q, F32)
    t.args.q = t.q.at
    got = t.ready().run()
    assert not np.isfinite(got[1, 0]).any()
    rest = np.ones(got.shape, bool)
    rest[1, 0] = False
    assert (np.abs(got - want)[rest] <= tol[rest]).all()


@pytest.mark.parametrize("value", [0.0, 1e-42, 3e38])
def test_cache_extreme_q(value):
    g = rng(34)
    q = g.standard_normal((2, 2, 64))
    q[1] = value
    t = Cached(g, F32, 64, 2, [100], [2], nkv=1, q=q, scale=1e-38 if value > 1 else 0.125)
    t.ready().check()


# ---------------------------------------------------------------- as they would be used
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd,G,window", [(128, 2, 0), (64, 4, 40), (256, 2, 100)])
def test_prompts_then_tokens(typ, hd, G, window):
    """A packed batch of prompts is appended and attended, then tokens one at a time and a piece of
    five: the cache's values are those of append, outputs those of the cache that it left."""
    g = rng(41, hd)
    counts, nkv = [70, 1, 130], 2
    ring = -(-(window + 5) // PAGE) + 1 if window else 0
    room = [c + 20 for c in counts]
    c = Cache8(g, nkv, hd, [0] * 3, ring, room).upload()
    a = Append(g, c, BLOCK8, typ, hd, G, [0] * 3, counts)
    p = Prompt(g, typ, hd, G, counts, window=window, nkv=nkv, q=a.q0, k=a.k0, v=a.v0)
    p.args.q, p.args.q_stride, p.args.k, p.args.k_stride = a.q_out.at, a.q_out.stride, a.k_out.at, a.k_out.stride
    s = Stream()
    spkv.append(a.args, s.h.value)
    spkv.prompt_attention(p.args, s.h.value)
    s.sync()
    a.check(run=False)
    p.q, p.k = a.q_out, a.k_out
    a.q_out.dev.a, a.k_out.dev.a = a.q_out.dev.get(), a.k_out.dev.get()
    close(p.got(), *p.want())
    at = list(counts)
    for step in (1, 1, 5, 1):
        n = [step] * 3
        a = Append(g, c, BLOCK8, typ, hd, G, at, n)
        t = Cached(g, typ, hd, G, at, n, window=window, nkv=nkv, cache=c, q=a.q0).ready()
        t.args.q, t.args.q_stride = a.q_out.at, a.q_out.stride
        spkv.append(a.args, s.h.value)
        spkv.cache_attention(t.args, s.h.value)
        s.sync()
        a.check(run=False)
        a.q_out.dev.a = a.q_out.dev.get()
        t.q = a.q_out
        close(t.got(), *t.want())
        at = [x + step for x in at]


def test_appended_f32_rows_are_tree_attentions():
    """f32 rows that append writes, read by tree attention as a chain."""
    g = rng(42)
    cached, n, hd, G, nkv = 100, 5, 128, 2, 2
    c = f32_cache(g, nkv, hd, [cached + n])
    a = Append(g, c, ROWS, F32, hd, G, [cached], [n])
    spkv.append(a.args)
    a.check(run=False)
    see, depth = tree_ref.masks(g, "chain", n)
    vis, out = Dev(tree_ref.words(see, 1)), Dev(np.zeros((n, nkv * G, hd), np.float32))
    t = spkv.TreeArgs(n_heads=nkv * G, n_kv_heads=nkv, head_dim=hd, rows=ROWS, n_seqs=1, n_nodes=n, max_nodes=n, max_positions=cached + n, window=0, ring_pages=0,
                      mask_words=1, scale=0.1, node_start=a.hold["start"].at, cached=a.hold["cached"].at, visible=vis.at, tables=c.lists.at, q=a.q_out.at,
                      q_stride=a.q_out.stride, out=out.at, out_stride=nkv * G * hd)
    need = spkv.tree_attention_work(t)
    work = Dev(np.zeros(need + 16, np.uint8))
    t.work, t.work_bytes = work.at, need
    spkv.tree_attention(t)
    q = a.q_out.get()[:n]
    c.pool = c.dev.get()
    want, tol = tree_ref.tree_attention(c, [cached], [(see, depth)], q, 0, float(np.float32(0.1)))
    assert (np.abs(out.get() - want) <= tol).all()


@pytest.mark.parametrize("typ", TYPES)
def test_calls_in_a_graph(typ):
    """A decode step captured and replayed on new inputs, with the program's own work between the
    replays: each replay is the call on those inputs."""
    g = rng(43)
    hd, G, nkv, cached = 128, 2, 2, [3000, 40]
    c = Cache8(g, nkv, hd, cached, 0, [x + 16 for x in cached]).upload()
    a = Append(g, c, BLOCK8, typ, hd, G, cached, [1, 1])
    t = Cached(g, typ, hd, G, cached, [1, 1], nkv=nkv, cache=c, q=a.q0).ready()
    p = Prompt(g, typ, hd, G, [60, 70], nkv=nkv)
    t.args.q, t.args.q_stride = a.q_out.at, a.q_out.stride
    s = Stream()

    def record(stream):
        spkv.append(a.args, stream)
        spkv.cache_attention(t.args, stream)
        spkv.prompt_attention(p.args, stream)

    e = s.capture(record)
    for k in range(4):
        x = rng(44, k)
        q, kk, v = (Packed(x.standard_normal(z.shape), typ) for z in (a.q, a.k, a.v))
        for dst, src in ((a.q, q), (a.k, kk), (a.v, v)):
            dst.dev.put(src.dev.a[:, :dst.stride] if dst.stride == src.stride else src.dev.a)
        c.dev.put(c.pool)
        a.q0, a.k0, a.v0 = q.values()[:2], kk.values()[:2], v.values()[:2]
        pq = Packed(x.standard_normal(p.q.shape), typ)
        p.q.dev.put(pq.dev.a)
        p.q.dev.a = pq.dev.a
        s.launch(e)
        s.sync()
        before = c.pool.copy()
        a.check(run=False)
        q_out = a.q_out.get()
        want, tol = cache_attention(c, q_out[:2], cached, [1, 1], 0, t.scale, typ)
        close(t.got(), want, tol)
        close(p.got(), *p.want())
        Dev(np.zeros(1 << 20, np.uint8)).get()
        c.pool[:] = before


def test_graph_of_other_lengths():
    """What a graph was captured with bounds the lengths; where sequences lie and end, the device
    memory says at each replay."""
    g = rng(48)
    hd, G, nkv = 128, 2, 2
    most = [5000, 300, 2000]
    c = Cache8(g, nkv, hd, [x + 8 for x in most]).upload()
    t = Cached(g, F32, hd, G, most, [8, 8, 8], nkv=nkv, cache=c).ready()
    p = Prompt(g, BF16, hd, G, [90, 300, 10], nkv=nkv)
    s = Stream()

    def record(stream):
        spkv.cache_attention(t.args, stream)
        spkv.prompt_attention(p.args, stream)

    e = s.capture(record)
    for cached, counts, prompts in ((most, [8, 8, 8], [90, 300, 10]), ([0, 299, 64], [1, 8, 0], [300, 0, 100]), ([4999, 1, 130], [1, 1, 1], [1, 1, 1]), ([64, 63, 1999], [3, 1, 5], [150, 100, 150])):
        t.cached, t.counts, p.counts = cached, counts, prompts
        t.dcached.put(np.array(cached, np.int32)); t.dstart.put(packed_start(counts)); p.dstart.put(packed_start(prompts))
        for out in (t.out, p.out):
            out.dev.put(np.full(out.dev.a.shape, out.one, out.dev.a.dtype))
        s.launch(e)
        s.sync()
        close(t.got(), *t.want())
        close(p.got(), *p.want())


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("cached", [[100, 30], [9000, 30]])
def test_rows_before_the_first_sequence(typ, cached):
    """start need not begin with 0: rows before it stay as they are, too."""
    g = rng(49)
    n, off = [40, 21], 7
    p = Prompt(g, typ, 64, 2, n, more_tokens=off)
    t = Cached(g, typ, 64, 2, cached, n, more_tokens=off).ready()
    for x, run in ((p, spkv.prompt_attention), (t, spkv.cache_attention)):
        x.dstart.put(packed_start(n) + off)
        run(x.args)
        raw = x.out.dev.get()
        assert (raw[:off] == x.out.one).all() and (raw[sum(n) + off:] == x.out.one).all()
        got = x.out.values(raw)[off:off + sum(n)]
        q = x.q.values()[off:]
        if x is p:
            close(got, *prompt_attention(q, p.k.values()[off:], p.v.values()[off:], n, 0, p.scale, typ))
        else:
            close(got, *cache_attention(t.cache, q, cached, n, 0, t.scale, typ))


def test_two_streams_at_once():
    """Calls on two streams with workspaces of their own."""
    g = rng(45)
    a, b = Cached(g, F32, 128, 2, [4000], [3], nkv=1).ready(), Cached(g, BF16, 64, 4, [3000, 20], [1, 2], nkv=1).ready()
    s, r = Stream(), Stream()
    for _ in range(5):
        spkv.cache_attention(a.args, s.h.value)
        spkv.cache_attention(b.args, r.h.value)
    s.sync(); r.sync()
    a.check(a.got())
    b.check(b.got())


def test_same_bits_again():
    """No order of arrival decides a sum: the same call gives the same bits."""
    g = rng(46)
    for typ in TYPES:
        t, p = Cached(g, typ, 128, 2, [5000, 900], [2, 7], nkv=1).ready(), Prompt(g, typ, 128, 2, [500], nkv=1)
        x, y = t.run().copy(), p.run().copy()
        for _ in range(3):
            assert np.array_equal(t.run().view(np.uint32), x.view(np.uint32)) and np.array_equal(p.run().view(np.uint32), y.view(np.uint32))


def test_beside_a_pending_error():
    """An error that an earlier call of the program left neither fails these calls nor is taken by them."""
    g = rng(47)
    t, p = Cached(g, F32, 64, 2, [5000], [3], nkv=1).ready(), Prompt(g, F32, 64, 2, [40], nkv=1)
    a = appended(g, BLOCK8, F32, 64, 2, [20], [5])
    hip().hipGetLastError()
    code = hip().hipMalloc(None, ctypes.c_size_t(16))
    assert code != 0
    spkv.cache_attention(t.args)
    spkv.prompt_attention(p.args)
    spkv.append(a.args)
    assert hip().hipGetLastError() == code
    sync()
    t.check(t.got())
    p.check(p.got())
    a.check(run=False)
