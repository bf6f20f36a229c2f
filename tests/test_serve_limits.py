"""Sizes that attention over the 8-bit cache refuses or takes: checked on the host, no GPU needed."""
import pytest

import spkv
from test_serve_args import cached


@pytest.mark.parametrize("ring,window,max_tokens,max_positions", [
    (4, 0, 1, 257), (1, 64, 1, 65), (2, 66, 1, 200), (2, 64, 3, 200), (19, 1024, 131, 5000), (16383, 0, 1, 1 << 20), (4, 1 << 30, 1, 300), (1, 2, 1, 100),
    (2, 2147483647, 16, 1000)])
def test_rings_that_do_not_hold_what_is_attended(ring, window, max_tokens, max_positions):
    kw = dict(ring_pages=ring, window=window, max_tokens=max_tokens, max_positions=max_positions, n_seqs=1, n_tokens=1)
    for call in (spkv.cache_attention, spkv.cache_attention_work):
        with pytest.raises(RuntimeError, match="ring_pages"):
            call(cached(**kw))


@pytest.mark.parametrize("ring,window,max_tokens,max_positions", [
    (4, 0, 1, 256), (1, 1, 1, 5000), (2, 65, 1, 200), (2, 64, 2, 200), (19, 1024, 130, 5000), (16384, 0, 512, 1 << 20), (5, 1 << 30, 1, 300), (2147483647, 0, 1, 1 << 20)])
def test_rings_that_do(ring, window, max_tokens, max_positions):
    spkv.cache_attention_work(cached(ring_pages=ring, window=window, max_tokens=max_tokens, max_positions=max_positions, n_seqs=1, n_tokens=1))


def test_any_span_of_a_ring_is_in_pages_of_its_own():
    """The bound by counting: where the largest span that is taken begins at each place of a page."""
    for ring in (1, 2, 3, 7):
        most = max(n for n in range(1, 64 * ring + 1) if ok(ring, n))
        assert all((at + most - 1) // 64 - at // 64 < ring for at in range(64))
        assert any((at + most) // 64 - at // 64 >= ring for at in range(64))


def ok(ring, span):
    try:
        spkv.cache_attention_work(cached(ring_pages=ring, window=span, max_tokens=1, max_positions=5000, n_seqs=1, n_tokens=1))
    except RuntimeError:
        return False
    return True


@pytest.mark.parametrize("seqs,G,max_tokens,positions,fits", [(2048, 8, 512, 2000, True), (4096, 8, 512, 2000, False), (4096, 4, 512, 2000, True), (2049, 8, 512, 2000, False),
                                                              (4096, 16, 1, 1 << 20, True), (4096, 16, 2, 1 << 20, True), (4096, 16, 3, 1 << 20, False)])
def test_workgroups_of_a_call(seqs, G, max_tokens, positions, fits):
    """n_seqs n_kv_heads for every 16 rows of a sequence and every part of its span: 2^22 of them at most."""
    kw = dict(n_seqs=seqs, n_tokens=seqs, n_kv_heads=8, n_heads=8 * G, head_dim=64, max_tokens=max_tokens, max_positions=positions, q_stride=512 * G, out_stride=512 * G)
    if fits:
        spkv.cache_attention_work(cached(**kw))
    else:
        for call in (spkv.cache_attention, spkv.cache_attention_work):
            with pytest.raises(RuntimeError, match="too many"):
                call(cached(**kw))
