"""Attention over the 8-bit cache at the ends of its numbers' range."""
import numpy as np
import pytest

import spkv
from serve_ref import BLOCK, Cached, close

pytestmark = pytest.mark.gpu
TYPES = [spkv.F32, spkv.BF16]


def climbing(typ, hd, n, scale_v, top):
    """n positions whose scores climb, by `top` in base 2 in all, V blocks of the scale given."""
    g = np.random.default_rng([71, hd, n])
    q = np.zeros((1, 2, hd))
    q[..., 0] = 1
    t = Cached(g, typ, hd, 2, [n - 1], [1], nkv=1, q=q, scale=top / 127 / np.log2(np.e))
    for p in range(n):
        pg, i = t.cache.block(0, p // BLOCK)
        t.cache.k[pg, 0, p % 64] = 0
        t.cache.k[pg, 0, p % 64, 0] = 127 * p // n
        t.cache.s[pg, 0, 0, i], t.cache.s[pg, 1, 0, i] = 1, scale_v
    return t.ready()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n", [400, 9000])
def test_values_below_the_limit(typ, hd, n):
    """V below 2^90, weights that grow to 2^15.9 before the running maximum moves."""
    climbing(typ, hd, n, 2.0 ** 83, 15.9).check()
    climbing(typ, hd, n, 2.0 ** 83, 40.0).check()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n", [400, 9000])
@pytest.mark.parametrize("e", [100, 112, 118, 121])
def test_values_above_the_limit(typ, n, e):
    """They are right, or not finite."""
    t = climbing(typ, 64, n, 2.0 ** e, 15.9)
    with np.errstate(over="ignore"):
        got, (want, tol) = t.run(), t.want()
    fine = np.isfinite(got)
    assert (np.abs(got - want) <= tol)[fine].all()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n", [1, 60, 9000])
def test_scores_below_every_number(typ, n):
    """A token all of whose scores are below f32's range has no finite value; its neighbours do."""
    g = np.random.default_rng([72, n])
    q = g.standard_normal((2, 2, 64))
    q[0, 1] = -3e38
    t = Cached(g, typ, 64, 2, [n - 1], [2], nkv=1, q=q, scale=1.0)
    t.cache.k[:] = np.abs(t.cache.k.astype(np.int16)).clip(1, 127)
    t.cache.s[:, 0] = 8
    t.ready()
    got, (want, tol) = t.run(), t.want()
    assert not np.isfinite(got[0, 1]).any()
    got[0, 1], want[0, 1], tol[0, 1] = 0, 0, 0
    close(got, want, tol)
