"""The paged cache's bookkeeping (host side, on the CPU): which pages belong to
which sequence."""

import pytest
import torch

from glorcq_amd.paged_cache import PagedKVCache


def _cache(**kw):
    a = dict(layers=2, kv_heads=2, head_dim=64, max_seqs=3, max_seq_len=100, page_size=16,
             device="cpu")
    return PagedKVCache(**{**a, **kw})


def _pages(c, b):
    n = -(-c.length(b) // c.page_size)
    row = c.page_table[b]
    assert (row[n:] == -1).all()
    return row[:n].tolist()


def _check(c):
    own = [p for b in range(c.max_seqs) for p in _pages(c, b)]
    assert len(set(own)) == len(own) and all(0 <= p < c.pages for p in own)
    assert len(own) + c.free_pages == c.pages
    assert c.lengths.tolist() == [c.length(b) for b in range(c.max_seqs)]


def test_extend_and_release():
    c = _cache()
    assert c.pages == 21 and tuple(c.page_table.shape) == (3, 7)
    c.extend([16, 0, 33])
    _check(c)
    assert [len(_pages(c, b)) for b in range(3)] == [1, 0, 3]
    before = _pages(c, 2)
    c.extend(1)
    _check(c)
    assert [c.length(b) for b in range(3)] == [17, 1, 34]
    assert _pages(c, 2) == before  # there was room in its last page
    c.release(2)
    _check(c)
    assert c.length(2) == 0
    c.extend([0, 0, 100])
    _check(c)
    c.reset()
    _check(c)
    assert c.free_pages == 21


def test_extend_refuses_whole_steps():
    c = _cache(pages=4)
    c.extend([16, 16, 16])
    for bad, what in (([0, 17, 0], "pages needed"), ([0, 0, 85], "max_seq_len"), ([1, 1], "counts"),
                      ([0, -1, 0], "counts"), (1, "pages needed")):
        with pytest.raises(RuntimeError, match=what):
            c.extend(bad)
        _check(c)
        assert [c.length(b) for b in range(3)] == [16, 16, 16]
    c.extend([0, 16, 0])
    _check(c)


def test_formats():
    c = _cache(dtype=torch.float16)
    k, v, ks, vs = c.layers[1]
    assert k.dtype == torch.float16 and tuple(k.shape) == (21, 2, 16, 64) and ks is None
    assert tuple(v.shape) == (21, 2, 1, 64, 16) and vs is None
    k, v, ks, vs = _cache().layers[0]
    assert k.dtype == torch.float8_e4m3fn and tuple(ks.shape) == (21, 2, 1)
    for kw in (dict(page_size=24), dict(dtype=torch.float32), dict(max_seqs=0), dict(pages=0)):
        with pytest.raises(RuntimeError):
            _cache(**kw)
