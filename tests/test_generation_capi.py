"""Host-side checks of the entry points of generation over the paged cache:
invalid arguments are refused before any launch (runs without a GPU)."""

import ctypes

import pytest

from glorcq_amd import _lib

P = 1 << 20  # a pointer that no call may follow


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _numbers(x):
    return None if x is None else ctypes.cast((ctypes.c_int32 * max(len(x), 1))(*x), ctypes.c_void_p)


def _copy(lib, src=(0,), dst=(1,), tokens=None, frm={}, to={}, pairs=None, **kw):
    """One cache of 8 pages a layer, 2 layers of 2 heads (128 KB of k and of v)."""
    pools = dict(k_pages=P, v_pages=2 * P, k_scales=3 * P, v_scales=4 * P, pages=8)
    a = dict(layers=2, kv_heads=2, head_dim=128, page_size=64,
             pairs=len(src) if pairs is None else pairs)
    keep = [_numbers(x) for x in (src, dst, tokens)]
    p = _lib.PagedCopyParams(from_=_lib.PagedPools(**{**pools, **frm}),
                             to=_lib.PagedPools(**{**pools, **to}),
                             src=keep[0], dst=keep[1], tokens=keep[2], **{**a, **kw})
    return lib.glq_paged_copy(ctypes.byref(p), None), lib.glq_last_error()


@pytest.mark.parametrize("kw,what", [
    (dict(head_dim=96), b"head_dim"), (dict(page_size=48), b"page_size"),
    (dict(page_size=8), b"page_size"), (dict(page_size=2048), b"page_size"),
    (dict(kv_heads=0), b"kv_heads"), (dict(kv_heads=1025), b"kv_heads"),
    (dict(layers=-1), b"layers"), (dict(layers=65536), b"layers"),
    (dict(pairs=-1), b"pairs"), (dict(pairs=(1 << 24) + 1), b"pairs"),
    (dict(frm=dict(pages=-1)), b"pages"), (dict(to=dict(pages=1 << 31)), b"pages"),
    (dict(frm=dict(k_pages=None)), b"null"), (dict(to=dict(v_pages=None)), b"null"),
    (dict(to=dict(k_scales=None)), b"come together"),
    (dict(frm=dict(v_scales=None)), b"come together"),
    (dict(frm=dict(k_pages=P + 8)), b"aligned"),
    (dict(to=dict(v_pages=P * 9)), b"must be one"), (dict(to=dict(pages=7)), b"must be one"),
    (dict(to=dict(k_pages=P + 4096)), b"must be one"),
    (dict(to=dict(k_pages=P * 9, v_pages=P * 10, k_scales=P * 11)), b"must be one"),
    (dict(to=dict(k_pages=P * 9, v_pages=P + 4096, k_scales=P * 11, v_scales=P * 12)),
     b"must be one"),
    (dict(src=[8]), b"out of range"), (dict(src=[-1]), b"out of range"),
    (dict(dst=[8]), b"out of range"), (dict(dst=[-1]), b"out of range"),
    (dict(tokens=[65]), b"tokens"), (dict(tokens=[-1]), b"tokens"),
    (dict(src=[0, 1], dst=[2, 2]), b"pair 1: a page is written twice"),
    (dict(src=[0, 2], dst=[2, 3]), b"pair 1: a page that is read is written"),
    (dict(src=[3], dst=[3]), b"read is written"),
    (dict(src=[0, 1, 2], dst=[4, 5, 8]), b"pair 2: page out of range"),
])
def test_copy_checks(lib, kw, what):
    rc, msg = _copy(lib, **kw)
    assert rc == 1 and what in msg


def test_copy_of_nothing(lib):
    assert lib.glq_paged_copy(None, None) == 1
    assert _copy(lib, src=(), dst=())[0] == 0
    assert _copy(lib, layers=0)[0] == 0
    assert _copy(lib, tokens=[0])[0] == 0  # no launch


def _beam(lib, **kw):
    a = dict(logits=P, scores=2 * P, prompts=2, beams=4, vocab=1000, row_stride=1000, num=8,
             out_scores=3 * P, out_parents=4 * P, out_tokens=5 * P, counters=6 * P, scratch=7 * P,
             counter_bytes=1 << 20, scratch_bytes=1 << 20)
    p = _lib.BeamSelectParams(**{**a, **kw})
    return lib.glq_beam_select(ctypes.byref(p), None), lib.glq_last_error()


@pytest.mark.parametrize("kw,what", [
    (dict(prompts=-1), b"prompts"), (dict(prompts=1 << 21), b"prompts"),
    (dict(prompts=1 << 14), b"65535"), (dict(beams=0), b"beams"), (dict(beams=65), b"beams"),
    (dict(vocab=0), b"vocab"), (dict(vocab=(1 << 24) + 1), b"vocab"), (dict(num=0), b"num"),
    (dict(num=129), b"num"), (dict(vocab=1, num=5), b"num"), (dict(dtype=3), b"dtype"),
    (dict(dtype=-1), b"dtype"), (dict(row_stride=999), b"row_stride"),
    (dict(logits=None), b"null"), (dict(scores=None), b"null"), (dict(out_tokens=None), b"null"),
    (dict(logits=P + 1), b"aligned"), (dict(logits=P + 2, dtype=2), b"aligned"),
    (dict(scores=P + 2), b"aligned"), (dict(out_parents=P + 4), b"aligned"),
    (dict(counters=None), b"workspace"), (dict(scratch=None), b"workspace"),
    (dict(counter_bytes=4), b"workspace"), (dict(scratch_bytes=100), b"workspace"),
    (dict(scratch=P + 8), b"workspace"), (dict(counters=P + 2), b"workspace"),
    (dict(out_scores=P + 8000), b"overlap"), (dict(out_scores=2 * P), b"overlap"),
    (dict(out_tokens=2 * P + 24), b"overlap"), (dict(out_parents=2 * P - 120), b"overlap"),
])
def test_beam_checks(lib, kw, what):
    rc, msg = _beam(lib, **kw)
    assert rc == 1 and what in msg


def test_attention_refuses_negative_sinks(lib):
    cache = _lib.PagedCache(k_pages=P, v_pages=P, page_table=P, lengths=P, seqs=2, max_pages=4,
                            table_stride=4, pages=8, kv_heads=2, head_dim=128, page_size=64)
    p = _lib.PagedAttentionParams(cache=cache, tokens=2, q=P, out=2 * P, q_heads=8, window=4,
                                  sinks=-1, scale=1.0, counters=P, scratch=P,
                                  counter_bytes=1 << 30, scratch_bytes=1 << 30)
    assert lib.glq_paged_attention(ctypes.byref(p), None) == 1
    assert b"sinks" in lib.glq_last_error()


def test_beam_of_nothing_and_workspace(lib):
    assert lib.glq_beam_select(None, None) == 1
    assert _beam(lib, prompts=0, logits=None)[0] == 0
    assert lib.glq_beam_select_counter_bytes(-1, 4) == lib.glq_beam_select_counter_bytes(1, 0) == -1
    assert lib.glq_beam_select_counter_bytes(3, 4) >= 60
    size = lib.glq_beam_select_scratch_bytes
    assert size(0, 4, 1000, 8) == 0 and 0 < size(1, 4, 1000, 8) <= size(8, 4, 1000, 8)
    for bad in ((-1, 4, 1000, 8), (1, 0, 1000, 8), (1, 65, 1000, 8), (1, 4, 0, 8), (1, 4, 1000, 0),
                (1, 4, 1000, 129), (1, 4, 1 << 25, 8)):
        assert size(*bad) == -1


def test_copy_pairs_of_no_tokens(lib):
    """They neither write nor read: the same page twice, or another pair's."""
    assert _copy(lib, src=[0, 1], dst=[2, 2], tokens=[0, 0])[0] == 0  # (no launch)
    assert _copy(lib, src=[0, 2, 3], dst=[2, 3, 3], tokens=[0, 0, 0])[0] == 0
    for src, dst, tokens, what in (([8, 0], [1, 2], [0, 0], b"pair 0: page out of range"),
                                   ([0, 1], [8, 2], [0, 0], b"pair 0: page out of range"),
                                   ([0, 1, 3], [2, 2, 2], [0, 4, 4], b"pair 2: a page is written twice"),
                                   ([0, 2], [2, 3], [1, 1], b"pair 1: a page that is read is written")):
        rc, msg = _copy(lib, src=src, dst=dst, tokens=tokens)
        assert rc == 1 and what in msg


def test_version_tells_the_sinks_apart(lib):
    """glq_paged_attention_params has sinks where a library before 0.2.0 had a
    field that it did not read."""
    assert lib.glq_version() >= 200
