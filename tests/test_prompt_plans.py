"""The GPU tests' prompt sizes reach every form that is built (no GPU needed)."""
import pytest

import spkv
from test_gpu_prompt_forms import BF16, F32, FORMS, TWO_PARTS


def plan(typ, hd, G, nkv, counts, window):
    return spkv.prompt_attention_plan(spkv.PromptArgs(n_heads=G * nkv, n_kv_heads=nkv, head_dim=hd, type=typ, n_seqs=len(counts), n_tokens=sum(counts),
                                                      max_tokens=max(counts), window=window, scale=0.1))


def test_every_form_is_reached():
    """(rows of a workgroup, keys of a tile, parts, waves), each with and without a window."""
    built = {(F32, 64): {(128, 32, 1, 4), (64, 128, 4, 8)}, (F32, 128): {(128, 32, 1, 4), (128, 64, 2, 8)}, (F32, 256): {(64, 32, 1, 4), (128, 32, 1, 8)},
             (BF16, 64): {(128, 64, 1, 4), (64, 128, 4, 8)}, (BF16, 128): {(128, 64, 1, 4), (64, 128, 4, 8), (128, 64, 2, 8), (256, 64, 1, 8)},
             (BF16, 256): {(64, 32, 1, 4)}}
    for windowed in (False, True):
        reached = {k: set() for k in built}
        for case in FORMS:
            if bool(case[5]) == windowed:
                reached[case[:2]].add(plan(*case))
        assert reached == built


def test_two_parts_are_reached():
    assert {plan(BF16, 128, *case) for case in TWO_PARTS} == {(128, 64, 2, 8)}


GOOD = dict(n_heads=1, n_kv_heads=1, head_dim=64, type=F32, scale=0.1)


def test_plan_refusals():
    for bad in (dict(head_dim=96), dict(window=-1), dict(n_tokens=-1), dict(scale=float("nan"))):
        with pytest.raises(RuntimeError, match="prompt_attention_plan"):
            spkv.prompt_attention_plan(spkv.PromptArgs(**{**GOOD, **bad}))
    assert spkv.kv().sp_hipkv_prompt_attention_plan(None, None) != 0
    a = spkv.PromptArgs(**GOOD)
    assert spkv.prompt_attention_plan(a)[0] and spkv.kv().sp_hipkv_prompt_attention_plan(a, None) != 0


@pytest.mark.parametrize("typ,hd,G,nkv,n", [(BF16, 128, 2, 8, 1200), (BF16, 128, 2, 8, 2800), (BF16, 128, 4, 8, 4000), (BF16, 64, 2, 8, 1200), (F32, 64, 4, 8, 1000),
                                            (F32, 128, 4, 8, 1900)])
def test_keys_are_not_shared_in_short_windows_of_many_rows(typ, hd, G, nkv, n):
    """Forms for few rows and long spans, and for very many rows: a window makes spans short, and workgroups are
    more than the device runs at once."""
    assert plan(typ, hd, G, nkv, [n], 0) != plan(typ, hd, G, nkv, [n], 128)
    assert plan(typ, hd, G, nkv, [n], 128)[2] == 1 and plan(typ, hd, G, nkv, [n], 128)[0] == 128
    assert plan(typ, hd, G, nkv, [n], n) == plan(typ, hd, G, nkv, [n], 0)
