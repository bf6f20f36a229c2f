"""Token log probabilities within the errors of the sums they make, whatever the vocabulary.

u = 2^-24, y = scale x, d = y - M.  A term's exponent is off by
  a = u (|y| + |M|)   (the products with scale) + u |d| (the difference) + 2 u |d| (log2 e, the product with it),
and the term by a factor of e^a and 3 u (the exponential, a step or two).  No f32 sum is longer
than 32 terms of a thread, 6 steps over lanes, 4 waves and the term of equals: 43 roundings,
all of terms of one sign; segments are joined in 64 bits.  So with t = e^d over the tokens
below the largest
  r = sum t        is off by  Er = sum t (a + 3 u) + 44 u r + V 2^-126   (the last: terms below normal numbers)
  s = sum t |d|    is off by  Es = sum t ((a + 3 u) |d| + a + u |d|) + 44 u s + V 2^-126 200,
  l = log1p(r)     by  dl = Er / (1 + r),
and lse = M + l, log p = (y - M) - l, H = l + s / (1 + r) by these and one rounding for each of
their steps."""
import numpy as np
import pytest

from test_gpu_tree_ops import logprob

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def check(x, scale, given, o):
    y = x.astype(np.float64) * np.float64(np.float32(scale))
    R, V = y.shape
    M = y.max(1, keepdims=True)
    d = (y - M).astype(np.longdouble)
    below = (x < x.max(1, keepdims=True)) & np.isfinite(y)
    with np.errstate(invalid="ignore", under="ignore"):
        t = np.where(below, np.exp(d), 0)
        ad = np.where(below, -d, 0).astype(np.float64)
        a = np.where(below, U * (np.abs(y) + np.abs(M)) + 3 * U * ad, 0)
    more = (x == x.max(1, keepdims=True)).sum(1) - 1
    r, s = t.sum(1) + more, (t * ad).sum(1)
    Er = (t * (a + 3 * U)).sum(1) + 44 * U * r + V * 2.0 ** -126
    Es = (t * ((a + 3 * U) * ad + a + U * ad)).sum(1) + 44 * U * s + V * 2.0 ** -126 * 200
    l, dl = np.log1p(r), Er / (1 + r)
    M = M[:, 0]
    lse, H = M + l, l + s / (1 + r)
    assert (np.abs(o["lse"] - lse) <= dl + U * (np.abs(M) + np.abs(lse))).all()
    assert (np.abs(o["ent"] - H) <= dl + Es / (1 + r) + s * Er / (1 + r) ** 2 + U * H).all()
    order = np.argsort(-x, axis=1, kind="stable")[:, :o["ids"].shape[1]]
    assert np.array_equal(o["ids"], order)
    for got, tok in ((o["lp"], given), (o["top"], order)):
        yt = np.take_along_axis(y, tok.astype(np.int64), 1)
        want = (yt - M[:, None]) - l[:, None]
        lim = dl[:, None] + U * (np.abs(yt) + np.abs(M)[:, None] + np.abs(yt - M[:, None]) + l[:, None] + np.abs(want))
        assert (np.abs(got - want) <= lim).all(), float((np.abs(got - want) / lim).max())
    return float(dl.max())


@pytest.mark.parametrize("R,V", [(1, 2048), (3, 8193), (1, 151936), (5, 151936), (33, 151936), (2, 262144), (20, 262144), (1, 1 << 20)])
@pytest.mark.parametrize("scale", [1.0, 1 / 0.8, 0.01])
def test_within_the_sums_errors(R, V, scale):
    g = np.random.default_rng([R, V, 9])
    x = (g.standard_normal((R, V)) * 2.5).astype(np.float32)
    for i in range(R):
        x[i, g.integers(0, V, 24)] += (6 + 2 * g.standard_normal(24)).astype(np.float32)      # a few likely tokens
    x[0, :] += 3.0                                     # a largest logit away from 0
    given = g.integers(0, V, (R, 4)).astype(np.int32)
    o, _ = logprob(x, scale, given, 20)
    assert check(x, scale, given, o) < 2e-5


def test_sure_rows_and_flat_rows():
    """A remainder far below 1, equal logits, and logits of one small step."""
    g = np.random.default_rng(4)
    x = (g.standard_normal((5, 151936)) * 2).astype(np.float32)
    x[0, 5000] = 40.0
    x[1, 77] = 25.0; x[1, 151935] = 25.0
    x[2, :] = -7.25
    x[3, :] = 0.0; x[3, 9] = 2.0 ** -20
    x[4, :] = -100.0 - np.arange(151936, dtype=np.float32) / 4096
    given = np.array([[5000, 77, 151935, 9]] * 5, np.int32)
    o, _ = logprob(x, 1.0, given, 20)
    check(x, 1.0, given, o)


def test_logits_that_scaling_takes_out_of_range():
    """y beyond f32 is infinite: the lowest number as a mask has p = 0 at any temperature, and a
    row whose largest y is +inf, or that has none above -inf, has no distribution."""
    lowest, largest = np.finfo(np.float32).min, np.finfo(np.float32).max
    g = np.random.default_rng(6)
    x = np.full((4, 9000), lowest, np.float32)
    x[0, :50] = g.standard_normal(50)
    x[1, 8999] = -3.0
    x[3, :] = 0.0; x[3, 70] = largest
    given = np.array([[3, 8000]] * 4, np.int32)
    o, _ = logprob(x, 1.25, given, 3)
    check(x[:1, :50], 1.25, given[:1, :1], {k: v[:1, :1] if k == "lp" else v[:1] for k, v in o.items()})
    assert o["lp"][0, 1] == -np.inf and o["ent"][1] == 0 and o["lse"][1] == -3.75 and o["ids"][1, 0] == 8999 and o["top"][1, 0] == 0
    assert np.isnan(o["lp"][2:]).all() and np.isnan(o["ent"][2:]).all() and o["lse"][2] == -np.inf and o["lse"][3] == np.inf
    assert list(o["ids"][3]) == [70, 0, 1] and list(o["ids"][2]) == [0, 1, 2]
