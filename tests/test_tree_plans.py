"""The GPU tests' tree attention sizes reach every form that is built (no GPU needed)."""
import pytest

import spkv
from test_gpu_tree_forms import FLOAT, INTEGER


def plan(rows, hd, G, nkv, S, cached, nodes, window):
    return spkv.tree_attention_plan(spkv.TreeArgs(
        n_heads=G * nkv, n_kv_heads=nkv, head_dim=hd, rows=rows, n_seqs=S, n_nodes=S * nodes, max_nodes=nodes, max_positions=cached + nodes,
        window=window, mask_words=(nodes + 63) // 64, scale=0.1))


def test_every_float_form_is_reached():
    """(rows, head_dim, row tiles), each with one part and with several."""
    built = {(spkv.ROWS_F32, 64): 4, (spkv.ROWS_F32, 128): 3, (spkv.ROWS_F32, 256): 2,
             (spkv.ROWS_SPINOR, 64): 3, (spkv.ROWS_SPINOR, 128): 2, (spkv.ROWS_SPINOR, 256): 1}
    want = {(*k, rt, parts) for k, n in built.items() for rt in range(1, n + 1) for parts in (False, True)}
    reached, windows = set(), set()
    for case in FLOAT:
        rt, parts, *rest = plan(*case)
        assert rest == [0, 0]
        reached.add((*case[:2], rt, parts > 1))
        if case[7]:
            windows.add((*case[:2], rt))
    assert reached == want
    assert windows == {k[:3] for k in want}


def test_every_exact_form_is_reached():
    """Row tiles of the scores (5 take the kernel for 6) and of the V sums, one part and several."""
    plans = [(case[1], plan(*case)) for case in INTEGER]
    for hd in (64, 128, 256):
        mine = [p for h, p in plans if h == hd]
        assert {min(p[0], 6) if p[0] != 5 else 6 for p in mine} == {1, 2, 3, 4, 6} and 5 in {p[0] for p in mine}
        assert {p[2] for p in mine} == ({1, 2} if hd == 64 else {1, 2, 3})
        assert {p[1] > 1 for p in mine} == {False, True} and {p[3] > 1 for p in mine} == {False, True}


def test_plan_refusals():
    with pytest.raises(RuntimeError, match="tree_attention_plan"):
        plan(spkv.ROWS_F32, 96, 1, 1, 1, 10, 1, 0)
    assert spkv.kv().sp_hipkv_tree_attention_plan(None, None) != 0
