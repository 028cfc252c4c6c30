"""Copies of pages in all layers at once (kernels.paged_copy): every byte of the
pools afterwards, and what is refused."""

import random

import pytest
import torch

from glorcq_amd import kernels

pytestmark = pytest.mark.gpu

FP8, FP16 = torch.float8_e4m3fn, torch.float16


def pools(gpu, layers, pages, Hk, D, page, dtype, seed):
    """Pools of any bits."""
    g = torch.Generator().manual_seed(seed)
    t = kernels.paged_cache_tensors(pages, Hk, D, page, dtype, gpu, layers=layers)
    for x in t:
        if x is not None:
            raw = x.view(torch.uint8)
            raw.copy_(torch.randint(0, 256, raw.shape, generator=g, dtype=torch.uint8))
    return t


def raw(t):
    return [None if x is None else x.view(torch.uint8).cpu().clone() for x in t]


def expected(frm, to, layers, page, src, dst, tokens):
    """The target's bytes: blocks of 16 tokens, page by page and head by head."""
    out = [None if x is None else x.clone() for x in to]
    for x, y in zip(frm, out):
        if x is None:
            continue
        shape = (x.shape[:2], y.shape[:2]) if layers is not None else ((1, *x.shape[:1]),
                                                                      (1, *y.shape[:1]))
        Hk = x.shape[2 if layers is not None else 1]
        x = x.view(*shape[0], Hk, page // 16, -1)
        y = y.view(*shape[1], Hk, page // 16, -1)
        for i, (s, d) in enumerate(zip(src, dst)):
            n = page // 16 if tokens is None else -(-tokens[i] // 16)
            y[:, d, :, :n] = x[:, s, :, :n]
    return out


def check(gpu, layers, pages, Hk, D, page, dtype, src, dst, tokens=None, other=None, seed=1):
    t = pools(gpu, layers, pages, Hk, D, page, dtype, seed)
    to = None if other is None else pools(gpu, layers, other, Hk, D, page, dtype, seed + 1)
    before, into = raw(t), raw(t if to is None else to)
    k, v, ks, vs = t
    kernels.paged_copy(k, v, src, dst, k_scales=ks, v_scales=vs, tokens=tokens, to=to)
    torch.cuda.synchronize()
    want = expected(before, into, layers, page, src, dst, tokens)
    for x, y in zip(raw(t if to is None else to), want):
        assert (x is None) == (y is None) and (x is None or torch.equal(x, y))
    if to is not None:
        for x, y in zip(raw(t), before):
            assert x is None or torch.equal(x, y)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("layers,Hk,D,page", [
    (None, 1, 64, 16), (1, 3, 128, 32), (5, 4, 128, 64), (2, 16, 64, 16), (3, 2, 64, 1024),
    (2, 1, 128, 1024), (70, 2, 64, 32)])
@pytest.mark.parametrize("other", [None, 11])
def test_whole_pages(gpu, dtype, layers, Hk, D, page, other):
    check(gpu, layers, 9, Hk, D, page, dtype, [2, 8, 2, 0], [1, 3, 6, 5], other=other)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("layers,Hk,D,page", [
    (None, 1, 64, 16), (1, 3, 128, 32), (5, 4, 128, 64), (2, 16, 64, 16), (3, 2, 64, 1024),
    (2, 1, 128, 1024), (3, 5, 64, 128)])
@pytest.mark.parametrize("other", [None, 12])
def test_parts_of_pages(gpu, dtype, layers, Hk, D, page, other):
    """0, 1, 15, 16, 17 tokens, all but one, all."""
    tokens = [0, 1, 15, 16, min(17, page), page - 1, page]
    check(gpu, layers, 12, Hk, D, page, dtype, [0, 1, 0, 3, 4, 4, 3], [5, 6, 7, 8, 9, 10, 11],
          tokens=tokens, other=other)


def test_many_pages(gpu):
    """More pairs than one launch takes, in any order; some of no tokens."""
    r = random.Random(5)
    order = list(range(1300))
    r.shuffle(order)
    src = [order[r.randrange(600)] for _ in range(700)]
    tokens = [r.choice((0, 5, 16, 32)) for _ in range(700)]
    check(gpu, 2, 1300, 2, 64, 32, FP8, src, order[600:], tokens=tokens)
    check(gpu, 2, 1300, 2, 64, 32, FP16, src, order[600:])


def test_nothing(gpu):
    check(gpu, 2, 3, 1, 64, 16, FP8, [], [])
    check(gpu, 2, 3, 1, 64, 16, FP8, [1, 1], [0, 2], tokens=[0, 0])


def test_a_layer_onto_another(gpu):
    """Layers of one cache are caches of their own."""
    t = pools(gpu, 3, 4, 2, 64, 16, FP8, 3)
    before = raw(t)
    one, two = ([x[i] for x in t] for i in (0, 2))
    kernels.paged_copy(one[0], one[1], [3, 1], [1, 2], k_scales=one[2], v_scales=one[3], to=two)
    for x, was in zip(raw(t), before):
        was[2, 1], was[2, 2] = was[0, 3].clone(), was[0, 1].clone()
        assert torch.equal(x, was)


def test_offsets_past_32_bits(gpu):
    """A pool of more than 4 GB."""
    L, P = 3, 9000
    t = kernels.paged_cache_tensors(P, 8, 128, 128, FP16, gpu, layers=L)
    assert t[0].numel() * 2 > 1 << 32
    rows = torch.randn(L, 8, 128, 128, device=gpu).half()
    t[0][:, P - 1], t[1][:, P - 2] = rows, rows.view(L, 8, 8, 128, 16)
    kernels.paged_copy(t[0], t[1], [P - 1, P - 2], [0, P - 3])
    assert torch.equal(t[0][:, 0], rows) and torch.equal(t[1][:, P - 3], rows.view(L, 8, 8, 128, 16))
    assert not t[0][:, 1].any() and not t[1][:, 0].any()


def test_numbers_as_tensors_and_on_a_stream(gpu):
    t = pools(gpu, 2, 6, 1, 64, 16, FP16, 4)
    before = raw(t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kernels.paged_copy(t[0], t[1], torch.tensor([5, 0]), torch.tensor([1, 2]),
                           tokens=torch.tensor([3, 16]))
    s.synchronize()
    for x, y in zip(raw(t), expected(before, before, 2, 16, [5, 0], [1, 2], None)):
        assert x is None or torch.equal(x, y)


def test_captured(gpu):
    """A captured copy copies what the pages hold at its replays."""
    t = pools(gpu, 2, 6, 2, 64, 32, FP8, 6)
    k, v, ks, vs = t
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kernels.paged_copy(k, v, [0, 1], [2, 3], k_scales=ks, v_scales=vs, tokens=[17, 9])
    for seed in (7, 8, 9):
        for x, y in zip(t, pools(gpu, 2, 6, 2, 64, 32, FP8, seed)):
            x.view(torch.uint8).copy_(y.view(torch.uint8))
        before = raw(t)
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(raw(t), expected(before, before, 2, 32, [0, 1], [2, 3], [17, 9])):
            assert torch.equal(x, y)


def test_refusals(gpu):
    t = pools(gpu, 2, 6, 2, 64, 32, FP8, 6)
    before = raw(t)
    k, v, ks, vs = t
    half = kernels.paged_cache_tensors(6, 2, 64, 32, FP16, gpu, layers=2)
    kw = dict(k_scales=ks, v_scales=vs)
    bad = [
        (([0], [6]), kw, "out of range"), (([-1], [1]), kw, "out of range"),
        (([0, 1], [2, 2]), kw, "written twice"), (([0, 2], [2, 3]), kw, "read is written"),
        (([3], [3]), kw, "read is written"), (([0], [1]), dict(kw, tokens=[33]), "tokens"),
        (([0], [1]), dict(kw, tokens=[-1]), "tokens"), (([0], [1, 2]), kw, "one length"),
        (([0], [1]), dict(kw, tokens=[]), "one length"), (([0.5], [1]), kw, "numbers"),
        (([1 << 40], [1]), kw, "numbers"), (([0], [1]), {}, "need k_scales"),
        ((torch.tensor([0]).to(gpu), [1]), kw, "host memory"),
        (([0], [1]), dict(kw, to=half), "type"), (([0], [1]), dict(kw, to=t[:2]), "to must be"),
        (([0], [1]), dict(kw, to=[x[:1] for x in t]), "layers"),
        # another cache that shares some of this one's memory
        (([0], [1]), dict(kw, to=(k, v.clone(), ks, vs)), "share"),
        (([0], [1]), dict(kw, to=(k.clone(), v, ks.clone(), vs.clone())), "share"),
    ]
    for args, more, what in bad:
        with pytest.raises(RuntimeError, match=what):
            kernels.paged_copy(k, v, *args, **more)
    for x in ((k[:, ::2], v), (k, v[:, :3]), (k.cpu(), v), (k[0, 0], v)):
        with pytest.raises(RuntimeError):
            kernels.paged_copy(*x, [0], [1], **kw)
    for x, y in zip(raw(t), before):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [FP8, FP16])
def test_pairs_of_no_tokens_beside_others(gpu, dtype):
    """A page that one pair writes may be another's that copies nothing."""
    check(gpu, 3, 9, 2, 64, 64, dtype, [0, 1, 5, 2, 6], [5, 5, 7, 0, 6], tokens=[20, 0, 0, 0, 0])
    check(gpu, 3, 9, 2, 64, 64, dtype, [0, 1, 2], [5, 5, 6], tokens=[64, 0, 64], other=8)
