"""Attention over the paged cache with a window and sinks (kernels.
paged_attention(window=, sinks=)) against its formula in 64 bits, with the pages
that no new token sees taken out of the cache.

The bounds are paged_ref.attend's, term by term, over the positions that a row
sees: nothing else than the set of positions differs."""

import math

import pytest
import torch

from glorcq_amd import kernels
from test_paged_gpu import FP8, FP16, Cache, batch

pytestmark = pytest.mark.gpu


def seen(pos, window, sinks):
    lo = max(0, pos - window + 1) if window else 0
    return torch.cat([torch.arange(min(sinks, lo)), torch.arange(lo, pos + 1)])


def attend(q, k, v, ev, first, scale, window, sinks, fp8):
    """q (n, Hq, D) fp16 at positions first .. -> (out, bound) (n, Hq, D) float64."""
    n, Hq, D = q.shape
    Hk = k.shape[1]
    rep, u = Hq // Hk, 2.0 ** -24
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(n):
        if first + i < 0:
            continue
        at = seen(first + i, window, sinks)
        L = k.shape[0]
        for h in range(Hk):
            kk, vv = k[at, h], v[at, h]
            qq = q[i, h * rep:(h + 1) * rep].double()
            t = qq @ kk.T * scale
            p = torch.softmax(t, -1)
            r = p @ vv
            mag = qq.abs() @ kk.abs().T * abs(scale)
            d = (2 * D * u * mag + 8 * u * (t.abs() + 33)).amax(-1, keepdim=True)
            e = ev[h][at // 16].double() if fp8 else torch.zeros(len(at), dtype=torch.float64)
            t2 = t * math.log2(math.e)
            M = (t2 + e).amax(-1, keepdim=True)
            total = torch.exp2(t2 - M).sum(-1, keepdim=True)
            codes = (vv * torch.exp2(-e)[:, None]).abs().sum(0)
            sub = (4 if n * rep > 32 else 1) * 2.0 ** -25 * codes / total
            out[i, h * rep:(h + 1) * rep] = r
            tol[i, h * rep:(h + 1) * rep] = (
                2.0 ** -11 * r.abs() + 2.0 ** -25
                + (2.0 ** -11 + 2 * d + 2 * L * u + 4 * u) * (p @ vv.abs()) * 1.001 + sub)
    return out, tol


def free_unseen(c, news, window, sinks):
    """Takes the pages out of the table that no new token sees, and gives them
    to somebody whose values are NaN; returns how many."""
    freed = 0
    for b, n in enumerate(news):
        L = c.model.k[b].shape[0]
        lo = max(0, L - n + 1 - window) if window else 0
        for i in range(-(-sinks // c.page), lo // c.page):
            pg = int(c.cpu_table[b, i])
            for x in c.t:
                if x is not None:
                    x.view(torch.uint8)[pg] = 255
            c.table[b, i] = -1
            freed += 1
    return freed


def check(c, q, news, window, sinks, scale=None, **kw):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    s, kp, vp = c.pages()
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, scale, starts=batch(news, c.dev),
                                window=window, sinks=sinks, **s, **kw)
    torch.cuda.synchronize()
    got = y.cpu().double().view(q.shape)
    lo = 0
    for b, n in enumerate(news):
        k, v = c.model.k[b], c.model.v[b]
        ref, tol = attend(q[lo:lo + n].cpu(), k, v, c.model.ev[b], k.shape[0] - n, scale, window,
                          sinks, c.fp8)
        d = (got[lo:lo + n] - ref).abs()
        bad = ~(d <= tol)
        assert not bad.any(), (b, int(bad.sum()), float((d / tol)[bad].max()))
        lo += n
    return y


def make(gpu, dtype, D, page, Hq, Hk, news, past, seed, window, sinks, free=True):
    c = Cache(gpu, len(news), Hk, D, page, dtype, max(map(sum, zip(news, past))) + page, seed)
    c.fill([n + p for n, p in zip(news, past)])
    q = (torch.randn(sum(news), Hq, D, generator=c.g) * 2).half().to(gpu)
    return c, q, free_unseen(c, news, window, sinks) if free else 0


# (new tokens, tokens behind, window, sinks): decode steps, prompts, both; a window
# not yet full, one that reaches into the sinks, sinks that end inside a block, at
# a page's end, past a tile; one position of each
CASES = [
    ([1], [0], 16, 4), ([1], [15], 16, 4), ([1], [19], 16, 4), ([1], [900], 1, 1),
    ([1, 1, 1], [700, 3, 164], 100, 5), ([3, 3], [200, 61], 50, 70),
    ([1, 40, 0, 7, 150], [300, 0, 5, 463, 270], 33, 17), ([200], [0], 40, 4), ([300], [130], 64, 64),
    ([2, 70], [1000, 800], 129, 130), ([1, 90], [500, 10], 1000, 8),
]


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D,page,Hq,Hk", [(128, 64, 8, 1), (64, 16, 4, 4), (128, 32, 6, 2),
                                          (64, 128, 20, 1)])
@pytest.mark.parametrize("news,past,window,sinks", CASES)
def test_sinks(gpu, dtype, D, page, Hq, Hk, news, past, window, sinks):
    c, q, _ = make(gpu, dtype, D, page, Hq, Hk, news, past, 41, window, sinks)
    check(c, q, news, window, sinks)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D,page,Hq,Hk,news,past,window,sinks", [
    (128, 64, 8, 1, [1], [9000], 5000, 300),              # one unit over many workgroups
    (64, 16, 2, 2, [1] * 3, [6000, 17, 4100], 2000, 100),  # units that share workgroups
    (128, 32, 4, 2, [2, 3, 1], [5000, 0, 2300], 1500, 9),
    (64, 64, 3, 3, [1] * 130, [5 * i for i in range(130)], 200, 64),  # more units than workgroups
    (128, 64, 8, 1, [40], [4000], 3000, 500),             # a prompt's positions split
    (64, 32, 8, 2, [130, 70], [2600, 1500], 1200, 33),
    (64, 64, 64, 64, [640], [100], 100, 50),              # 320 units
])
def test_sinks_split(gpu, dtype, D, page, Hq, Hk, news, past, window, sinks):
    """The units' pieces over waves and workgroups; twice, since a call leaves
    its counters zero."""
    c, q, freed = make(gpu, dtype, D, page, Hq, Hk, news, past, 42, window, sinks)
    assert freed > 0 or past == [100]
    y = check(c, q, news, window, sinks)
    assert torch.equal(y, check(c, q, news, window, sinks))


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("news,past", [([1, 1], [500, 40]), ([60, 2], [400, 300])])
def test_sinks_that_change_nothing(gpu, dtype, news, past):
    """Without a window, with one that sees all, and with no sinks, the results
    are those of the call without them, bit for bit."""
    c, q, _ = make(gpu, dtype, 128, 32, 8, 2, news, past, 43, 0, 0, free=False)
    for window, sinks in ((0, 7), (100000, 7), (0, 1 << 40), (64, 0)):
        y = check(c, q, news, window, sinks)
        s, kp, vp = c.pages()
        assert torch.equal(y, kernels.paged_attention(
            q, kp, vp, c.table, c.lengths, 128 ** -0.5, starts=batch(news, gpu), window=window, **s))
    # sinks that reach every window: all positions
    y = check(c, q, news, 64, 100000)
    assert torch.allclose(y.float(), check(c, q, news, 0, 0).float(), atol=2e-3, rtol=2e-3)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("news,past,window,sinks", [
    ([1, 1], [270, 105], 60, 20), ([20, 3], [250, 100], 33, 7), ([200, 90], [0, 90], 40, 50)])
def test_sinks_unseen_nan(gpu, dtype, news, past, window, sinks):
    """A position behind the sinks and before the windows of some rows may hold
    NaN: the rows that see it have it, the others nothing of it.  So may one of
    the sinks."""
    at = [sinks + 3, sinks - 2]
    c = Cache(gpu, 2, 2, 128, 64, dtype, 384, 44, nan=True)
    c.fill([n + p for n, p in zip(news, past)])
    for b in range(2):
        c.model.v[b][at[b], 1, 9] = float("nan")
        c.model.k[b][at[b], 0, 7] = float("nan")
    c.upload()
    q = torch.randn(sum(news), 8, 128, generator=c.g).half().to(gpu)
    s, kp, vp = c.pages()
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.1, starts=batch(news, gpu),
                                window=window, sinks=sinks, **s).cpu().double().view(q.shape)
    lo = 0
    for b, (n, p) in enumerate(zip(news, past)):
        k, v = (torch.nan_to_num(x, nan=0.0) for x in (c.model.k[b], c.model.v[b]))
        ref, tol = attend(q[lo:lo + n].cpu(), k, v, c.model.ev[b], p, 0.1, window, sinks, c.fp8)
        other = torch.ones(128, dtype=torch.bool)
        other[9] = False
        for i in range(n):
            row, ok = y[lo + i], (y[lo + i] - ref[i]).abs() <= tol[i]
            if at[b] in seen(p + i, window, sinks):
                assert row[:4].isnan().all() and row[4:, 9].isnan().all() and ok[4:, other].all()
            else:
                assert ok.all(), (b, i)
        lo += n


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("n", [5, 50])
def test_rows_that_see_nothing(gpu, dtype, n):
    """Tokens before position 0 are 0, one that sees a sink's page out of range
    or that lies past the page table NaN; rows behind the last sequence are left."""
    c = Cache(gpu, 3, 1, 64, 16, dtype, 112, 45)
    c.fill([2, 100, 100])
    c.lengths[0] = 2
    c.lengths[2] = 114  # two tokens past the page table's 112 positions
    c.table[1, 1] = -1  # of the sinks
    st = torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32, device=gpu)
    q = torch.randn(3 * n + 2, 2, 64, generator=c.g).half().to(gpu)
    out = torch.full((3 * n + 2, 128), 7.0).half().to(gpu)
    s, kp, vp = c.pages()
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.1, starts=st, window=10, sinks=20,
                                out=out, **s).cpu()
    assert y is not None and (y[:n - 2] == 0).all() and (y[3 * n:] == 7).all()
    ref, tol = attend(q[n - 2:n].cpu(), c.model.k[0], c.model.v[0], c.model.ev[0], 0, 0.1, 10, 20,
                      c.fp8)
    assert ((y[n - 2:n].double().view(2, 2, 64) - ref).abs() <= tol).all()
    assert y[n:2 * n].isnan().all() and y[3 * n - 2:3 * n].isnan().all()


def test_graph_replays_follow_lengths(gpu):
    """A captured step replayed while its sequences grow past their windows and
    pages are freed, with eager work between."""
    news, window, sinks = [1, 1, 1], 40, 6
    c, q, _ = make(gpu, FP8, 128, 16, 8, 2, news, [150, 20, 77], 46, window, sinks, free=False)
    s, kp, vp = c.pages()
    ws = kernels.paged_attention_workspace(q, kp, c.table)
    args = (q, kp, vp, c.table, c.lengths, 0.09)
    kw = dict(window=window, sinks=sinks, workspace=ws, **s)
    kernels.paged_attention(*args, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = kernels.paged_attention(*args, **kw)
    full = c.lengths.clone()
    for back in (0, 3, 17, 0):
        c.lengths.copy_((full - back).clamp(min=1))
        free_unseen_now = [max(0, int(L) - window) // 16 for L in c.lengths]
        if back == 0:
            for b, hi in enumerate(free_unseen_now):
                c.table[b, 1:max(1, hi)] = -1
        else:
            c.table.copy_(c.cpu_table.int())
        want = kernels.paged_attention(*args, **kw).clone()
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and bool(torch.isfinite(y).all())


def test_refusals(gpu):
    c, q, _ = make(gpu, FP16, 64, 16, 2, 1, [1], [30], 47, 0, 0)
    s, kp, vp = c.pages()
    for kw in (dict(sinks=-1), dict(window=4, sinks=-3)):
        with pytest.raises(RuntimeError, match="sinks"):
            kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.1, **s, **kw)
