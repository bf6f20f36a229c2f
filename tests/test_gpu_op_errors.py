"""Errors of a call of an operator on device memory are its own: one that an earlier
call of the program left behind neither fails it nor is taken by it."""
import ctypes

import numpy as np
import pytest

import spkv
import tree_ref
from devmem import Dev, hip
from helpers import prompt
from test_gpu_tree_ops import ALL, F32, Tree, check_logprobs, logprob
from test_gpu_tree_step import Rig, path, same_bits, tree

pytestmark = pytest.mark.gpu


class Pending:
    """An error of a refused argument, left by the program; still there afterwards."""

    def __enter__(self):
        hip().hipGetLastError()
        self.code = hip().hipMalloc(None, ctypes.c_size_t(16))
        assert self.code != 0 and hip().hipPeekAtLastError() == self.code

    def __exit__(self, kind, value, trace):
        left = hip().hipGetLastError()
        assert kind or left == self.code


@pytest.mark.parametrize("rows", ALL)
def test_tree_attention_beside_a_pending_error(rows):
    for cached in (100, 5000):
        t = Tree(rows, 128, 2, [cached], [9], seed=41, nkv=1).ready()
        with Pending():
            spkv.tree_attention(t.args)
        t.check(t.result())


def test_token_logprobs_beside_a_pending_error():
    x = np.random.default_rng(2).standard_normal((3, 20000)).astype(np.float32)
    given = np.array([[1], [2], [3]], np.int32)
    o, d = logprob(x, 1.0, given, 4)
    with Pending():
        spkv.token_logprobs(d["args"])
    check_logprobs(x, 1.0, given, 4, {k: d[k].get()[:3] for k in o})


def test_keep_rows_beside_a_pending_error():
    """A call that failed after its rows had moved would be made again, and move others."""
    c = tree_ref.Cache(np.random.default_rng(1), F32, 2, 64, [70]).upload()
    dc, ds, dk = Dev(np.array([40], np.int32)), Dev(np.array([0, 3], np.int32)), Dev(np.array([1, 4, 9], np.int32))
    a = spkv.KeepArgs(n_kv_heads=2, row_bytes=256, n_tables=1, n_seqs=1, max_keep=3, max_positions=70, tables=c.lists.at,
                      cached=dc.at, keep_start=ds.at, keep=dk.at)
    want = c.pool.copy()
    for i, j in enumerate((1, 4, 9)):
        (p0, r0), (p1, r1) = c._at(0, 40 + i), c._at(0, 40 + j)
        want[p0, :, :, r0] = want[p1, :, :, r1]
    with Pending():
        spkv.keep_rows(a)
    assert np.array_equal(c.dev.get().view(np.uint32), want.view(np.uint32))


def test_tree_keep_beside_a_pending_error(tmpdir_models):
    r = Rig(tmpdir_models, "qwen3-hd128")
    b, one = r.backend(True), r.backend(True)
    for x in (b, one):
        x.prefill(prompt(57, r.V, seed=5))
    parents, toks = tree(12, 1), prompt(12, r.V, seed=100)
    b.tree_step(toks, parents)
    keep = path(parents, 11)
    assert keep != list(range(len(keep)))
    with Pending():
        b.tree_keep(keep)
    lg, ref = np.zeros(r.V, np.float32), np.zeros(r.V, np.float32)
    for i in keep:
        one.decode(int(toks[i]), ref)
    assert b.position() == one.position()
    for l in range(r.d["n_layers"]):
        for x, y in zip(b.read_kv(l, 0, b.position(), r.kvd), one.read_kv(l, 0, one.position(), r.kvd)):
            assert same_bits(x, y)
    b.decode(7, lg); one.decode(7, ref)
    assert same_bits(lg, ref)
    b.close(); one.close(); r.close()
