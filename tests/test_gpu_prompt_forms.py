"""Attention of packed prompts in the forms that longer calls take, against whole matrices
in 64 bits; bounds as serve_ref.prompt_attention derives them."""
import numpy as np
import pytest

import spkv
from serve_ref import B, U, Prompt, packed_start

pytestmark = pytest.mark.gpu
F32, BF16 = spkv.F32, spkv.BF16


def reference(p, heads=None):
    """[tokens][the given q heads][hd] and the bound.  Values that are not finite are taken as 0: rows that
    attend them are not compared."""
    q, k, v = (np.where(np.isfinite(x), x, 0).astype(np.float64) for x in (p.q.values(), p.k.values(), p.v.values()))
    NH, hd = q.shape[1:]
    G, heads, scale = NH // k.shape[1], list(range(NH)) if heads is None else heads, p.scale
    out, tol = np.zeros((sum(p.counts), len(heads), hd)), np.zeros((sum(p.counts), len(heads), hd))
    for a, n in zip(packed_start(p.counts), p.counts):
        t = np.arange(n)
        seen = t <= t[:, None]
        if p.window:
            seen &= t > t[:, None] - p.window
        for i, h in enumerate(heads):
            x, K, V = q[a:a + n, h], k[a:a + n, h // G], v[a:a + n, h // G]
            if not n:
                continue
            z = np.where(seen, x @ K.T * scale, -np.inf)
            off = z.max(1, keepdims=True) - z
            w = np.exp(-off)
            w /= w.sum(1, keepdims=True)
            d = (6 * hd + 20) * U * abs(scale) * np.where(seen, np.abs(x) @ np.abs(K).T, 0).max(1) + 4 * U * np.where(seen, off, 0).max(1)
            if p.typ == F32:
                d += 2.0 ** -39 * abs(scale) * np.where(seen, np.abs(x).max(1)[:, None] * np.abs(K).sum(1) + np.abs(x).sum(1)[:, None] * np.abs(K).max(1), 0).max(1)
            o, r, m = w @ V, w @ np.abs(V), seen.sum(1)
            e = (4 * d + (12 * m + 64) * U)[:, None] * r + U * np.abs(o)
            if p.typ == F32:
                big = w * np.abs(V).max(1)
                e += (2.0 ** -31 * m * big.max(1) + 2.0 ** -39 * big.sum(1))[:, None]
            else:
                e = (e + B * r) * (1 + B) + B * np.abs(o)
            out[a:a + n, i], tol[a:a + n, i] = o, e
    return out, tol


def check(p, heads=None, rows=None):
    """The given rows [token][head] (all) are within the bound."""
    got, (want, tol) = p.run(), reference(p, heads)
    got = got if heads is None else got[:, heads]
    ok = np.isfinite(got) & (np.abs(got - want) <= tol)
    assert (ok if rows is None else ok[rows]).all()
    return got


# Keys of 128 rows shared by two waves each: the parts' outputs are joined in LDS
TWO_PARTS = [(1, 24, [900], 0), (1, 24, [900], 700), (2, 8, [1300], 0), (2, 8, [1700], 555), (4, 8, [1000], 0), (2, 8, [901, 0, 1700], 0), (2, 8, [3000], 0)]


@pytest.mark.parametrize("G,nkv,counts,window", TWO_PARTS)
def test_two_parts(G, nkv, counts, window):
    p = Prompt(np.random.default_rng([61, G, sum(counts)]), BF16, 128, G, counts, window=window, nkv=nkv)
    check(p, None if sum(counts) < 1500 else [0, 5, G * nkv - 1])


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n", [100, 300])
def test_zero_q(typ, hd, n):
    """A head whose q is zero, padding tokens with zeros, and rows of the smallest numbers: the mean of the V that they attend."""
    g = np.random.default_rng([62, hd, n])
    q = g.standard_normal((n, 4, hd))
    q[:, 1], q[40:90], q[:, 3] = 0, 0, q[:, 3] * 1e-38
    check(Prompt(g, typ, hd, 1, [n], nkv=4, q=q))
    check(Prompt(g, typ, hd, 4, [n - 20, 20], nkv=1, q=q, window=70))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [1e-38, -1e-39, 2e-45])
def test_tiny_scales(hd, scale):
    """Keys shared by the waves of a workgroup, and a difference of scores that weighs anything beyond f32."""
    for counts, nkv in ([300], 4), ([1300], 16):
        p = Prompt(np.random.default_rng([63, hd]), BF16, hd, 1, counts, nkv=nkv, scale=scale)
        check(p, None if nkv == 4 else [0, 15])


@pytest.mark.parametrize("hd,n", [(64, 100), (64, 300), (128, 100), (128, 300), (256, 100), (256, 700)])
@pytest.mark.parametrize("scale", [1e-8, -1e-20, 1e-38, 2e-45])
def test_zero_q_and_tiny_scales(hd, n, scale):
    """f32: what a difference of scores weighs, beside a q of zeros, is below f32's smallest number."""
    g = np.random.default_rng([64, hd, n])
    q = g.standard_normal((n, 2, hd))
    q[:, 1], q[30:80], q[80:90] = 0, 0, q[80:90] * 1e-38
    check(Prompt(g, F32, hd, 1, [n], nkv=2, q=q, scale=scale))
    check(Prompt(g, F32, hd, 2, [n], nkv=1, q=q, scale=scale, window=50))


# type, head_dim, q heads for each kv head, kv heads, tokens, window: every form that is built (test_prompt_plans.py)
FORMS = [
    (F32, 64, 2, 2, [100, 27], 0), (F32, 64, 8, 16, [300], 0), (F32, 64, 8, 16, [300], 70), (F32, 64, 2, 2, [300, 9, 150], 0), (F32, 64, 3, 2, [700], 0),
    (F32, 64, 2, 2, [500], 130), (F32, 128, 2, 2, [100, 27], 0), (F32, 128, 16, 16, [300], 0), (F32, 128, 16, 16, [300], 70), (F32, 128, 2, 2, [300, 9, 150], 0),
    (F32, 128, 3, 2, [700], 0), (F32, 128, 2, 2, [500], 130), (F32, 256, 2, 2, [300, 9], 0), (F32, 256, 2, 2, [300, 9], 70), (F32, 256, 16, 7, [300], 0),
    (F32, 256, 16, 4, [300], 70),
    (BF16, 64, 2, 2, [100, 27], 0), (BF16, 64, 4, 8, [700], 0), (BF16, 64, 4, 8, [700], 130), (BF16, 64, 2, 2, [300, 9, 250], 0), (BF16, 64, 3, 2, [900], 200),
    (BF16, 128, 2, 2, [100, 27], 0), (BF16, 128, 4, 8, [700], 0), (BF16, 128, 4, 8, [700], 130), (BF16, 128, 2, 2, [300, 9, 250], 0), (BF16, 128, 3, 2, [900], 200),
    (BF16, 128, 1, 24, [900], 0), (BF16, 128, 4, 8, [1000], 900), (BF16, 128, 16, 4, [2000], 0), (BF16, 128, 16, 4, [2000], 300), (BF16, 128, 16, 4, [2000], 1400),
    (BF16, 128, 1, 24, [900], 333), (BF16, 128, 2, 8, [1300], 64), (F32, 64, 4, 8, [700], 130),
    (BF16, 256, 2, 2, [300, 9], 0), (BF16, 256, 3, 2, [500], 70),
]


def form(case, **kw):
    typ, hd, G, nkv, counts, window = case
    return Prompt(np.random.default_rng([65, hd, G, nkv, sum(counts)]), typ, hd, G, counts, window=window, nkv=nkv, **kw)


def few(p):
    NH, G = p.q.shape[1], p.q.shape[1] // p.k.shape[1]
    return sorted({0, G - 1, G % NH, NH // 2, NH - 1})


@pytest.mark.parametrize("case", FORMS, ids=str)
def test_forms(case):
    p = form(case, pad=8, more_tokens=3)
    check(p, few(p))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("case", FORMS, ids=str)
def test_forms_beside_values_that_are_not_finite(case, bad):
    """In V at one column of a token of the first kv head, in K at another token, in all of V at a third: rows that do
    not attend them are as without, those that do are not finite (from K everywhere)."""
    p = form(case)
    n, W = p.counts[0], p.window or 1 << 30
    k, v = p.k.values().copy(), p.v.values().copy()
    one, key, all_of = n // 2 + 3, 3 * n // 4, 7 * n // 8
    v[one, 0, 7], k[key, 0, 5], v[all_of, -1] = bad, np.nan, bad
    p.k, p.v = type(p.k)(k, p.typ), type(p.v)(v, p.typ)
    p.args.k, p.args.k_stride, p.args.v, p.args.v_stride = p.k.at, p.k.stride, p.v.at, p.v.stride
    heads = few(p)
    G, t = p.q.shape[1] // p.k.shape[1], np.arange(sum(p.counts))

    def attends(token, kv):
        return ((t >= token) & (t < min(token + W, n)))[:, None] & (np.array(heads) // G == kv)

    gone = np.repeat(attends(key, 0)[..., None], p.q.shape[2], 2) | attends(all_of, p.k.shape[1] - 1)[..., None]
    gone[..., 7] |= attends(one, 0)
    got, (want, tol) = p.run()[:, heads], reference(p, heads)
    assert not np.isfinite(got[gone]).any()
    assert np.isfinite(got[~gone]).all() and (np.abs(got - want) <= tol)[~gone].all()
