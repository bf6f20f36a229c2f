"""Nodes with many children: log probabilities are of at most 64 of them, the step itself
of any number."""
import numpy as np
import pytest

from helpers import prompt
from test_gpu_tree_step import Rig, log_softmax, same_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("children", [64, 65, 127])
def test_children_of_one_node(tmpdir_models, children):
    r = Rig(tmpdir_models, "qwen3-hd128")
    b = r.backend(True)
    b.prefill(prompt(40, r.V, seed=5))
    parents, toks = [-1] + [0] * children, prompt(1 + children, r.V, seed=6)
    if children > 64:
        with pytest.raises(RuntimeError, match="at most 64 children"):
            b.tree_step(toks, parents)
        with pytest.raises(RuntimeError, match="no tree is pending"):
            b.tree_keep([0])
        lg, nxt, lp = b.tree_step(toks, parents, r.V, logprob=False)
        assert lp is None
    else:
        lg, nxt, lp = b.tree_step(toks, parents, r.V)
        want = log_softmax(lg[0])[toks[1:]]
        # f32 logits' spread, as for other trees: 1e-5
        assert np.isnan(lp[0]) and np.abs(lp[1:] - want).max() <= 1e-5
    assert np.array_equal(nxt, lg.argmax(1))
    ref = np.zeros(r.V, np.float32)
    for i in (1, children // 2, children):
        f = b.fork()
        for j in (0, i):
            f.decode(int(toks[j]), ref)
            assert same_bits(lg[j], ref)
        f.close()
    b.tree_keep([0, children])
    assert b.position() == 42
    b.close(); r.close()
