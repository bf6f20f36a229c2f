"""What the operators of serving from a paged cache refuse: checked on the host, before any
device is touched, so no GPU is needed and no address is looked at."""
import ctypes

import pytest

import spkv

P = 1 << 20                                             # a 16-byte aligned address nobody reads
HEADS = dict(n_heads=16, n_kv_heads=8, head_dim=128, type=spkv.F32, n_seqs=2, n_tokens=20, max_tokens=16, start=P, q=P, q_stride=2048)
BAD_HEADS = [dict(head_dim=96), dict(head_dim=0), dict(n_kv_heads=0), dict(n_heads=12), dict(n_heads=0), dict(n_heads=136), dict(n_heads=4104, n_kv_heads=1026),
             dict(type=2), dict(type=-1), dict(n_seqs=-1), dict(n_seqs=4097), dict(n_tokens=-1), dict(n_tokens=33), dict(max_tokens=-1),
             dict(n_seqs=4096, max_tokens=512, n_tokens=(1 << 20) + 1), dict(start=None), dict(q_stride=2047), dict(q_stride=2050), dict(q_stride=1024),
             dict(q=P + 4), dict(q=P + 8), dict(type=spkv.BF16, q_stride=2052), dict(q_stride=(1 << 22) + 8)]


def append(**kw):
    return spkv.AppendArgs(**{**HEADS, **dict(rows=spkv.ROWS_BLOCK8, max_positions=1000, ring_pages=0, eps=1e-6, cached=P, tables=P, freq=P, q_norm=P,
                                              k_norm=P, k=P, k_stride=1024, v=P, v_stride=1024, q_out=P, q_out_stride=2048, k_out=P, k_out_stride=1024), **kw})


def prompt(**kw):
    return spkv.PromptArgs(**{**HEADS, **dict(window=0, scale=0.1, k=P, k_stride=1024, v=P, v_stride=1024, out=P, out_stride=2048), **kw})


def cached(**kw):
    return spkv.CacheArgs(**{**HEADS, **dict(max_positions=1000, window=0, ring_pages=0, scale=0.1, cached=P, tables=P, out=P, out_stride=2048,
                                             work=P, work_bytes=1 << 40), **kw})


@pytest.mark.parametrize("bad", BAD_HEADS + [
    dict(rows=spkv.ROWS_EXACT), dict(rows=spkv.ROWS_SPINOR), dict(rows=4), dict(max_positions=-1), dict(max_positions=(1 << 20) + 1), dict(ring_pages=-1),
    dict(max_tokens=(1 << 20) + 1), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(cached=None), dict(tables=None), dict(tables=P + 4),
    dict(freq=P + 4), dict(q=None), dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 4), dict(k_stride=1020), dict(v_stride=1025), dict(q_out=P + 8),
    dict(q_out_stride=2044), dict(k_out=P + 8), dict(k_out_stride=1000), dict(q_out_stride=2052), dict(k_out_stride=1028),
    dict(v_stride=(1 << 22) + 8), dict(k_out_stride=(1 << 22) + 8)])
def test_append_refusals(bad):
    with pytest.raises(RuntimeError, match="sp_hipkv_append"):
        spkv.append(append(**bad))


@pytest.mark.parametrize("bad", BAD_HEADS + [
    dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(k=P + 4), dict(v=P + 8),
    dict(out=P + 4), dict(k_stride=1020), dict(v_stride=1026), dict(out_stride=2044), dict(k_stride=(1 << 22) + 8), dict(out_stride=1 << 23),
    dict(n_seqs=4096, n_tokens=4096, n_heads=4096, n_kv_heads=4096, head_dim=64, **{x + "_stride": 1 << 18 for x in ("q", "k", "v", "out")})])
def test_prompt_refusals(bad):
    with pytest.raises(RuntimeError, match="sp_hipkv_prompt_attention"):
        spkv.prompt_attention(prompt(**bad))


@pytest.mark.parametrize("bad", BAD_HEADS + [
    dict(max_positions=-1), dict(max_positions=(1 << 20) + 1), dict(max_tokens=513), dict(window=-1), dict(ring_pages=-1), dict(scale=float("nan")),
    dict(scale=float("-inf")), dict(cached=None), dict(tables=None), dict(tables=P + 4), dict(q=None), dict(out=None), dict(out=P + 8), dict(out_stride=2046), dict(out_stride=(1 << 22) + 8),
    dict(n_seqs=4096, max_tokens=512, n_tokens=(1 << 18) + 1)])
def test_cache_refusals(bad):
    with pytest.raises(RuntimeError, match="sp_hipkv_cache_attention"):
        spkv.cache_attention(cached(**bad))


def test_cache_work_is_required():
    big = dict(n_seqs=1, n_tokens=1, max_positions=100000)
    need = spkv.cache_attention_work(cached(**big))
    assert need > 0
    for kw in (dict(work=None), dict(work_bytes=need - 1), dict(work=P + 8)):
        with pytest.raises(RuntimeError, match="work"):
            spkv.cache_attention(cached(**big, **kw))
    with pytest.raises(RuntimeError):
        spkv.cache_attention_work(cached(head_dim=32))
    assert spkv.kv().sp_hipkv_cache_attention_work(ctypes.byref(cached()), None) != 0


def test_null_blocks():
    for f in ("append", "prompt_attention", "cache_attention"):
        assert getattr(spkv.kv(), "sp_hipkv_" + f)(None, None) != 0


def test_nothing_to_do_touches_no_device():
    spkv.append(append(n_tokens=0, k=None, v=None, q=None, tables=None))
    spkv.prompt_attention(prompt(n_tokens=0, n_seqs=0, q=None))
    spkv.cache_attention(cached(n_tokens=0, q=None, out=None))


def test_page_bytes():
    assert spkv.block8_page_bytes(8, 128) == 2 * 8 * (64 * 128 + 16)
    for bad in ((0, 128), (8, 96), (4097, 64), (-1, 64)):
        assert spkv.block8_page_bytes(*bad) == 0
