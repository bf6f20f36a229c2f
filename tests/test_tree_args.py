"""What the operators on device memory refuse: checked on the host, before any
device is touched, so no GPU is needed and no address is looked at."""
import ctypes

import pytest

import spkv

P = 1 << 20                                             # a 16-byte aligned address nobody reads


def tree(**kw):
    d = dict(n_heads=16, n_kv_heads=8, head_dim=128, rows=spkv.ROWS_F32, n_seqs=2, n_nodes=20, max_nodes=16, max_positions=1000,
             window=0, ring_pages=0, mask_words=1, scale=0.1, node_start=P, cached=P, depth=P, visible=P, tables=P, q=P,
             q_stride=2048, out=P, out_stride=2048, work=P, work_bytes=1 << 40)
    d.update(kw)
    return spkv.TreeArgs(**d)


@pytest.mark.parametrize("bad", [
    dict(head_dim=96), dict(head_dim=0), dict(n_kv_heads=0), dict(n_heads=12), dict(n_heads=0), dict(n_heads=136, n_kv_heads=8),
    dict(rows=3), dict(rows=-1), dict(n_seqs=-1), dict(n_seqs=4097), dict(n_heads=4104, n_kv_heads=1026), dict(n_nodes=-1), dict(n_nodes=33), dict(max_nodes=513, mask_words=9),
    dict(n_seqs=4096, n_nodes=(1 << 18) + 1, max_nodes=512, mask_words=8), dict(max_positions=(1 << 20) + 1), dict(rows=spkv.ROWS_EXACT, max_positions=(1 << 18) + 1), dict(max_positions=-1),
    dict(window=-1), dict(ring_pages=-1), dict(max_nodes=65, mask_words=1), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(node_start=None), dict(cached=None), dict(visible=None), dict(tables=None), dict(q=None), dict(out=None),
    dict(window=5, depth=None), dict(q_stride=2047), dict(q_stride=2050), dict(out_stride=100), dict(q=P + 4), dict(out=P + 8),
    dict(visible=P + 4),
])
def test_tree_refusals(bad):
    with pytest.raises(RuntimeError, match="sp_hipkv_tree_attention"):
        spkv.tree_attention(tree(**bad))


def test_tree_work_is_required():
    need = spkv.tree_attention_work(tree(n_seqs=1, n_nodes=16, max_positions=100000))
    if need:
        for kw in (dict(work=None), dict(work_bytes=need - 1), dict(work=P + 8)):
            with pytest.raises(RuntimeError, match="work"):
                spkv.tree_attention(tree(n_seqs=1, n_nodes=16, max_positions=100000, **kw))
    with pytest.raises(RuntimeError):
        spkv.tree_attention_work(tree(head_dim=32))
    assert spkv.kv().sp_hipkv_tree_attention(None, None) != 0
    assert spkv.kv().sp_hipkv_tree_attention_work(ctypes.byref(tree()), None) != 0


@pytest.mark.parametrize("vocab", [1, 2048, 2049, 8192, 20000, 32768, 100000, 151936, 262144, 262145, 1 << 20])
def test_logprob_work_of_a_call_is_enough_for_a_smaller_one(vocab):
    for top in (0, 1, min(vocab, 32)):
        need = [spkv.token_logprobs_work(logprob(n_rows=r, vocab=vocab, stride=vocab, n_top=top)) for r in range(1, 600)]
        assert need == sorted(need)
    assert spkv.token_logprobs_work(logprob(n_rows=7, vocab=vocab, stride=vocab, n_top=0)) <= \
        spkv.token_logprobs_work(logprob(n_rows=7, vocab=vocab, stride=vocab, n_top=1))


def test_nothing_to_do_touches_no_device():
    spkv.tree_attention(tree(n_nodes=0, q=None))
    spkv.tree_attention(tree(n_nodes=0, n_seqs=0))
    spkv.token_logprobs(logprob(n_rows=0))
    spkv.keep_rows(keep(n_tables=0, n_seqs=0))
    spkv.keep_rows(keep(max_keep=0, keep=None))


def logprob(**kw):
    d = dict(n_rows=4, vocab=1000, n_given=2, n_top=5, scale=1.0, logits=P, stride=1000, given=P, given_logprob=P, entropy=P, lse=P,
             top_ids=P, top_logprob=P, work=P, work_bytes=1 << 40)
    d.update(kw)
    return spkv.LogprobArgs(**d)


@pytest.mark.parametrize("bad", [
    dict(n_rows=-1), dict(n_rows=65536), dict(vocab=0), dict(vocab=(1 << 20) + 1, stride=1 << 21), dict(n_given=-1), dict(n_given=65), dict(n_top=-1),
    dict(n_top=33), dict(vocab=4, stride=4), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(stride=999), dict(logits=None), dict(logits=P + 2), dict(given=None), dict(given_logprob=None), dict(top_ids=None),
])
def test_logprob_refusals(bad):
    with pytest.raises(RuntimeError, match="sp_hipkv_token_logprobs"):
        spkv.token_logprobs(logprob(**bad))


def keep(**kw):
    d = dict(n_kv_heads=8, row_bytes=512, n_tables=4, n_seqs=2, max_keep=5, max_positions=100, tables=P, seq=None, ring_pages=None,
             cached=P, keep_start=P, keep=P)
    d.update(kw)
    return spkv.KeepArgs(**d)


@pytest.mark.parametrize("bad", [
    dict(n_kv_heads=0), dict(row_bytes=0), dict(row_bytes=140), dict(n_tables=-1), dict(n_seqs=-1), dict(n_seqs=0), dict(max_keep=-1),
    dict(max_keep=513), dict(max_positions=-1), dict(tables=None), dict(cached=None), dict(keep_start=None), dict(keep=None),
])
def test_keep_refusals(bad):
    with pytest.raises(RuntimeError, match="sp_hipkv_keep_rows"):
        spkv.keep_rows(keep(**bad))
