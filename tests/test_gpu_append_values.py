"""Appending rows with values that are not finite: what the formula makes of each value."""
import numpy as np
import pytest

import spkv
import tree_ref
from serve_ref import Append, Cache8, Packed, prepared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", [spkv.F32, spkv.BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("rotated", [False, True])
def test_norm_of_a_row_with_an_infinity(typ, hd, n, rotated):
    """The root is infinite: the row's other values are 0 (their partners in the rotation aside), as infinity
    over infinity they have none; other rows are as without."""
    g = np.random.default_rng([81, hd, n])
    k = g.standard_normal((n, 2, hd))
    k[1, 1, 5], k[2, 0, 9] = np.inf, np.nan
    c = tree_ref.Cache(g, spkv.ROWS_F32, 2, hd, [n], 0).upload()
    a = Append(g, c, spkv.ROWS_F32, typ, hd, 2, [0], [n], freq=rotated, k=k, eps=0.0 if n == 3 else 1e-6)
    q = a.q.values()
    q[0, 3, 8] = -np.inf
    a.q.dev.put(Packed(q, typ).dev.a)
    spkv.append(a.args)
    for out, x, w in ((a.q_out, q, a.nq), (a.k_out, a.k0, a.nk)):
        want, got = prepared(x, a.pos, a.freq, w, a.eps), out.get(n)
        zero, none = want == 0, np.isnan(want)
        assert np.isnan(got[none]).all() and (got[zero] == 0).all() and zero.sum() >= hd - 2
        assert np.isfinite(got[~none]).all() and (np.abs(got - want) <= 2.0 ** -7 * np.abs(want) + 1e-30)[~none].all()


@pytest.mark.parametrize("hd", [64, 256])
def test_block_of_a_row_with_an_infinity(hd):
    g = np.random.default_rng([82, hd])
    k = g.standard_normal((40, 2, hd))
    k[20, 1, 5] = np.inf
    c = Cache8(g, 2, hd, [0], 0, [40]).upload()
    a = Append(g, c, spkv.ROWS_BLOCK8, spkv.F32, hd, 1, [0], [40], k_out=None, k=k)
    a.check()
    pg, i = c.block(0, 1)
    assert np.isnan(c.s[pg, 0, 1, i]) and np.isfinite(c.s[pg, 0, 0, i])
