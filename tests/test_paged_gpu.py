"""The paged key/value cache (kernels.paged_append, kernels.paged_attention)
against its formulas in 64 bits (paged_ref), over formats, head layouts, page
sizes, lengths and masks; the bounds are paged_ref's, derived there."""

import math

import pytest
import torch

import paged_ref as R
from glorcq_amd import kernels

pytestmark = pytest.mark.gpu

FP8, FP16 = torch.float8_e4m3fn, torch.float16


class Cache:
    """A layer's pool on the GPU, filled with garbage, and its model."""

    def __init__(self, dev, B, Hk, D, page, dtype, max_len, seed, pool=None, nan=False):
        self.g = torch.Generator().manual_seed(seed)
        self.dev, self.fp8, self.page, self.D, self.Hk = dev, dtype == FP8, page, D, Hk
        P = -(-max_len // page)
        self.pool = pool or B * P + 2
        self.model = R.Model(B, Hk, D, page, self.fp8, self.pool, self.g)
        self.t = kernels.paged_cache_tensors(self.pool, Hk, D, page, dtype, dev)
        for x in self.t:
            if x is not None:  # any bits: what no token has written counts for nothing
                raw = x.view(torch.uint8)
                raw.copy_(torch.randint(0, 256, raw.shape, generator=self.g, dtype=torch.uint8))
                if nan:
                    raw.fill_(255)
        order = torch.randperm(B * P, generator=self.g)[:B * P].to(torch.int32) + 1
        self.table = order.view(B, P).to(dev)
        self.lengths = torch.zeros(B, dtype=torch.int32, device=dev)
        self.cpu_table = self.table.cpu().long()

    def pages(self):
        k, v, ks, vs = self.t
        return dict(k_scales=ks, v_scales=vs), k, v

    def fill(self, news, wide=True):
        """Puts random tokens into the model and the pages (host side)."""
        for b, n in enumerate(news):
            for which in "kv":
                x = torch.randn(n, self.Hk, self.D, generator=self.g, dtype=torch.float64)
                if wide:  # blocks of different scales, wide channels
                    x = x * torch.exp2(torch.randint(-3, 4, (n, 1, 1), generator=self.g))
                    x[..., ::17] *= 6
                self.model.put(which, b, x.half().double())
        self.upload()

    def upload(self):
        """The model's tokens into the pages."""
        for b in range(self.model.B):
            for which, pages, scales in (("k", self.t[0], self.t[2]), ("v", self.t[1], self.t[3])):
                x = getattr(self.model, which)[b]
                e = getattr(self.model, "e" + which)[b]
                L = x.shape[0]
                self.lengths[b] = L
                pos = torch.arange(L)
                pg, at = self.cpu_table[b, pos // self.page], pos % self.page
                if self.fp8:
                    x = x * torch.exp2(-e.T[pos // 16].double())[..., None]
                val = x.float().to(pages.dtype)
                host = pages.cpu()
                raw = host.view(torch.uint8) if self.fp8 else host
                val = val.view(torch.uint8) if self.fp8 else val
                if which == "k":
                    raw[pg, :, at] = val
                else:
                    raw[pg, :, at // 16, :, at % 16] = val
                pages.view(torch.uint8).copy_(host.view(torch.uint8))
                if self.fp8:
                    host = scales.cpu().view(torch.uint8)
                    host[pg, :, at // 16] = (e.T[pos // 16] + 127).to(torch.uint8)
                    scales.view(torch.uint8).copy_(host)

    def tokens(self, b, L):
        """(k, v, ek, ev) that the pages hold of sequence b: (L, Hk, D) values,
        (Hk, blocks) exponents."""
        kp, vp = (x.cpu() for x in self.t[:2])
        pos = torch.arange(L)
        pg, at = self.cpu_table[b, pos // self.page], pos % self.page
        if not self.fp8:
            return kp[pg, :, at].double(), vp[pg, :, at // 16, :, at % 16].double(), None, None
        ks, vs = (x.cpu().view(torch.uint8).long() - 127 for x in self.t[2:])
        k = kp.view(torch.uint8)[pg, :, at].view(FP8).double()
        v = vp.view(torch.uint8)[pg, :, at // 16, :, at % 16].contiguous().view(FP8).double()
        bk, bv = ks[pg, :, at // 16], vs[pg, :, at // 16]
        return (k * torch.exp2(bk.double())[..., None], v * torch.exp2(bv.double())[..., None],
                bk[::16].T, bv[::16].T)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=1e30), torch.nan_to_num(b, nan=1e30))


def batch(news, dev):
    st = torch.tensor([0] + list(news)).cumsum(0).to(torch.int32).to(dev)
    return None if len(set(news)) == 1 else st


def new_tokens(T, Hq, Hk, D, dev, gen, amp=1.0):
    """q, k, v as slices of one matrix, as a fused projection makes them."""
    qkv = (torch.randn(T, (Hq + 2 * Hk) * D, generator=gen) * amp).half()
    cut = [Hq * D, Hk * D, Hk * D]
    return qkv.split(cut, 1), qkv.to(dev).split(cut, 1)


def rope_rows(pos, D):
    ang = pos.double()[:, None] * 1e4 ** (-torch.arange(0, D, 2).double() / D)
    ang = torch.cat([ang, ang], 1)
    return torch.cos(ang).half(), torch.sin(ang).half()


def check_append(c, news, Hq, norm, rope, seed, amp=1.0, item=False):
    """One append on cache `c` (its model's tokens behind), checked; the model
    then holds what the pages hold."""
    gen = torch.Generator().manual_seed(seed)
    Hk, D, dev = c.Hk, c.D, c.dev
    T, B = sum(news), len(news)
    past = [c.model.k[b].shape[0] for b in range(B)]
    (q, k, v), (gq, gk, gv) = new_tokens(T, Hq, Hk, D, dev, gen, amp)
    qw = kw = cos = sin = None
    if norm:
        qw, kw = ((0.5 + torch.rand(D, generator=gen)).half() for _ in range(2))
    if rope:
        pos = torch.cat([torch.arange(p, p + n) for p, n in zip(past, news)])
        cos, sin = rope_rows(pos, D)
    up = lambda x: None if x is None else x.to(dev)  # noqa: E731
    before = [None if x is None else x.view(torch.uint8).cpu().clone() for x in c.t]
    c.lengths.copy_(torch.tensor([p + n for p, n in zip(past, news)]))
    gq_in = gq
    if item:  # a batched GEMV's output
        R_ = Hk * D
        gq_in = gq.reshape(T, -1, R_).transpose(0, 1).contiguous()
    kw_, kp, vp = c.pages()
    out = kernels.paged_append(gk, gv, kp, vp, c.table, c.lengths, starts=batch(news, dev), **kw_,
                               cos=up(cos), sin=up(sin), q=gq_in, q_norm_w=up(qw), k_norm_w=up(kw),
                               eps=1e-6)
    torch.cuda.synchronize()
    # q: the fp16 rounding of a value within the bound
    val, err = R.head_norm_rope(q.reshape(T, Hq, D), qw, cos, sin, 1e-6)
    got = out.cpu().double()
    assert (got >= (val - err).half().double()).all() and (got <= (val + err).half().double()).all()
    kval, kerr = R.head_norm_rope(k.reshape(T, Hk, D), kw, cos, sin, 1e-6)
    vval = v.reshape(T, Hk, D).double()
    lo = 0
    touched = [None if x is None else torch.zeros_like(x, dtype=torch.bool) for x in before]
    for b, n in enumerate(news):
        L, old_k, old_ek = past[b] + n, c.model.k[b], c.model.ek[b]
        gk_, gv_, gek, gev = c.tokens(b, L)
        # v: no arithmetic, so exactly the model's
        c.model.put("v", b, vval[lo:lo + n])
        assert same(gv_, c.model.v[b])
        kv, ke = kval[lo:lo + n], kerr[lo:lo + n]
        if not c.fp8:
            assert same(gk_[:past[b]], old_k)
            new = gk_[past[b]:]
            assert (new >= (kv - ke).half().double()).all()
            assert (new <= (kv + ke).half().double()).all()
        elif n:
            assert torch.equal(gev, c.model.ev[b])
            for i in range(past[b] // 16, -(-L // 16)):
                s, t = max(i * 16, past[b]), min(i * 16 + 16, L)
                for h in range(Hk):
                    x, dx = kv[s - past[b]:t - past[b], h], ke[s - past[b]:t - past[b], h]
                    was = int(old_ek[h, i]) if i * 16 < past[b] else R.MIN_EXP
                    e = int(gek[h, i])
                    assert max(was, R.scale_exp(float((x.abs() - dx).max()))) <= e \
                        <= max(was, R.scale_exp(float((x.abs() + dx).max())))
                    f = 2.0 ** -e
                    assert (gk_[s:t, h] * f >= R.e4m3_of((x - dx) * f)).all()
                    assert (gk_[s:t, h] * f <= R.e4m3_of((x + dx) * f)).all()
                    # tokens that the block had: scaled along
                    kept = R.e4m3_of(old_k[i * 16:s, h] * f)
                    assert same(gk_[i * 16:s, h] * f, kept)
            assert same(gk_[:past[b] // 16 * 16], old_k[:past[b] // 16 * 16])
        # what may have changed: the blocks with new tokens (fp16: the tokens)
        for i in range(past[b] // 16, -(-L // 16) if n else 0):
            pg, blk = int(c.cpu_table[b, i * 16 // c.page]), i * 16 % c.page // 16
            s = max(past[b] - i * 16, 0) if not c.fp8 else 0
            t = min(L - i * 16, 16) if not c.fp8 else 16
            touched[0][pg, :, blk * 16 + s:blk * 16 + t] = True
            if c.fp8:
                touched[1][pg, :, blk] = True
                touched[2][pg, :, blk] = touched[3][pg, :, blk] = True
                # zero behind the last token
                end = min(L - i * 16, 16)
                assert not c.t[0].view(torch.uint8)[pg, :, blk * 16 + end:blk * 16 + 16].any()
                assert not c.t[1].view(torch.uint8)[pg, :, blk, :, end:].any()
            else:
                touched[1][pg, :, blk, :, 2 * s:2 * t] = True
        lo += n
        c.model.k[b] = gk_
        if c.fp8:
            c.model.ek[b] = gek
    for x, was, tch in zip(c.t, before, touched):
        if x is not None:
            now = x.view(torch.uint8).cpu()
            assert torch.equal(now[~tch], was[~tch])
    return out


def check_attend(c, q, news, scale, window=0, out=None, **kw):
    """paged_attention of q (T, Hq, D) on the model's last tokens, checked."""
    s, kp, vp = c.pages()
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, scale, starts=batch(news, c.dev),
                                window=window, out=out, **s, **kw)
    torch.cuda.synchronize()
    got = y.cpu().double().view(q.shape)
    lo = 0
    for b, n in enumerate(news):
        k, v = c.model.k[b], c.model.v[b]
        ref, tol = R.attend(q[lo:lo + n].cpu(), k, v, c.model.ev[b], k.shape[0] - n, scale, window,
                            c.fp8)
        d = (got[lo:lo + n] - ref).abs()
        bad = ~(d <= tol)
        assert not bad.any(), (b, int(bad.sum()), float((d / tol)[bad].max()))
        lo += n
    return y


# (new tokens, tokens behind) a sequence
APPENDS = [
    ([1], [0]), ([1], [15]), ([1, 1, 1], [7, 16, 100]), ([5, 0, 33, 1], [0, 9, 31, 47]),
    ([130], [3]), ([2, 2], [63, 64]), ([16, 16], [16, 8]),
]


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D,page,Hq,Hk", [(128, 64, 8, 2), (64, 16, 3, 3), (128, 128, 7, 1)])
@pytest.mark.parametrize("news,past", APPENDS)
def test_append(gpu, dtype, D, page, Hq, Hk, news, past):
    c = Cache(gpu, len(news), Hk, D, page, dtype, max(map(sum, zip(news, past))) + page, 3)
    c.fill(past)
    check_append(c, news, Hq, True, True, 11)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("norm,rope,item", [(False, True, True), (True, False, False),
                                            (False, False, False)])
def test_append_without(gpu, dtype, norm, rope, item):
    c = Cache(gpu, 3, 2, 128, 32, dtype, 100, 5)
    c.fill([0, 20, 40])
    check_append(c, [9, 1, 30], 8, norm, rope, 12, item=item)


@pytest.mark.parametrize("dtype", [FP8, FP16])
def test_append_token_by_token(gpu, dtype):
    """Blocks whose scale grows with later tokens, up to the next block."""
    c = Cache(gpu, 2, 2, 64, 16, dtype, 64, 6)
    amps = [1e-6, 1e-3, 1e-3, 0.5, 0.25, 3.0, 40.0, 41.0, 900.0, 1.0] + [2.0] * 12
    for i, amp in enumerate(amps):
        check_append(c, [1, 1], 4, False, True, 100 + i, amp=amp)


def test_append_nothing_finite(gpu):
    """Infinities and NaN become NaN and set no scale; all-zero blocks too."""
    c = Cache(gpu, 1, 1, 64, 16, FP8, 64, 7)
    T = 20
    k = torch.randn(T, 64, generator=c.g).half()
    v = torch.randn(T, 64, generator=c.g).half()
    k[3, 5], k[4, 6], v[7, 8] = float("inf"), float("nan"), float("-inf")
    k[16:], v[16:] = 0, 0
    c.lengths.fill_(T)
    s, kp, vp = c.pages()
    kernels.paged_append(k.to(gpu), v.to(gpu), kp, vp, c.table, c.lengths, **s)
    for which, x in (("k", k), ("v", v)):
        c.model.put(which, 0, x.double().view(T, 1, 64))
    gk, gv, gek, gev = c.tokens(0, T)
    assert same(gk, c.model.k[0]) and same(gv, c.model.v[0])
    assert torch.equal(gek, c.model.ek[0]) and torch.equal(gev, c.model.ev[0])
    assert int(gk.isnan().sum()) == 2 and int(gv.isnan().sum()) == 1
    assert int(gek[0, 1]) == R.MIN_EXP


# (new tokens, tokens behind) a sequence
ATTENDS = [
    ([1], [0]), ([1], [16]), ([1, 1, 1], [700, 3, 64]), ([3, 3], [0, 61]),
    ([1, 40, 0, 7, 150], [300, 0, 5, 63, 70]), ([200], [0]), ([65], [130]),
]


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D,page,Hq,Hk", [(128, 64, 8, 1), (64, 16, 4, 4), (128, 32, 6, 2),
                                          (64, 128, 20, 1)])
@pytest.mark.parametrize("news,past", ATTENDS)
def test_attention(gpu, dtype, D, page, Hq, Hk, news, past):
    c = Cache(gpu, len(news), Hk, D, page, dtype, max(map(sum, zip(news, past))) + page, 21)
    c.fill([n + p for n, p in zip(news, past)])
    q = (torch.randn(sum(news), Hq, D, generator=c.g) * 2).half().to(gpu)
    check_attend(c, q, news, D ** -0.5)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D,page,Hq,Hk,news,past,window", [
    (128, 64, 8, 1, [1], [9000], 0),                    # one unit over many workgroups
    (64, 16, 2, 2, [1] * 3, [6000, 17, 4100], 0),       # units that share workgroups
    (128, 32, 4, 2, [2, 3, 1], [5000, 0, 2300], 1500),
    (64, 64, 3, 3, [1] * 130, list(range(130)), 0),     # more units than workgroups
    (128, 128, 40, 2, [1, 1], [2500, 100], 0),          # more rows than a unit holds
    (64, 32, 1, 1, [1] * 600, [i % 70 for i in range(600)], 0),  # more sequences than threads
])
def test_attention_split(gpu, dtype, D, page, Hq, Hk, news, past, window):
    """The units' pieces over waves and workgroups, and their merging; twice,
    since a call leaves its counters zero."""
    c = Cache(gpu, len(news), Hk, D, page, dtype, max(past) + page, 28)
    c.fill([n + p for n, p in zip(news, past)])
    q = (torch.randn(sum(news), Hq, D, generator=c.g) * 2).half().to(gpu)
    y = check_attend(c, q, news, D ** -0.5, window=window)
    assert torch.equal(y, check_attend(c, q, news, D ** -0.5, window=window))


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D,page,Hq,Hk,news,past,window", [
    (128, 64, 8, 1, [4, 4], [70, 1000], 0),        # 32 rows a sequence
    (128, 64, 8, 1, [5, 5], [70, 1000], 0),        # 40
    (64, 16, 4, 2, [16, 17, 1], [40, 700, 90], 0),  # 32, 34 and 2 in a batch
    (128, 64, 8, 1, [8, 8], [70, 1000], 0),        # 64 rows a sequence
    (128, 64, 8, 1, [9, 9], [70, 1000], 0),        # 72
    (64, 16, 4, 2, [32, 33, 1], [40, 700, 90], 0),  # 64, 66 and 2 in a batch
    (128, 64, 8, 1, [40], [3000], 0),              # few units over a long context
    (128, 32, 4, 2, [130, 70], [2600, 1500], 0),
    (64, 128, 8, 1, [33, 20], [4100, 33], 2000),
    (64, 16, 2, 2, [100] * 3, [900, 0, 2500], 0),
    (64, 64, 64, 64, [640], [0], 0),               # 320 units, two a CU in turn
    (64, 64, 64, 64, [300, 340], [0, 20], 0),
])
def test_attention_prompt_split(gpu, dtype, D, page, Hq, Hk, news, past, window):
    """Rows about the limit between the two forms, and prompts whose positions
    are split over workgroups."""
    c = Cache(gpu, len(news), Hk, D, page, dtype, max(map(sum, zip(news, past))) + page, 31)
    c.fill([n + p for n, p in zip(news, past)])
    q = (torch.randn(sum(news), Hq, D, generator=c.g) * 2).half().to(gpu)
    y = check_attend(c, q, news, D ** -0.5, window=window)
    assert torch.equal(y, check_attend(c, q, news, D ** -0.5, window=window))


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("window", [1, 16, 50, 200, 100000])
def test_attention_window(gpu, dtype, window):
    news, past = [1, 40, 7, 90], [300, 0, 150, 60]
    c = Cache(gpu, 4, 2, 128, 32, dtype, 340, 22)
    c.fill([n + p for n, p in zip(news, past)])
    q = torch.randn(sum(news), 8, 128, generator=c.g).half().to(gpu)
    check_attend(c, q, news, 0.1, window=window)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("news,past,window", [([1, 1], [70, 5], 0), ([20, 3], [50, 0], 0),
                                              ([20, 1], [90, 80], 33), ([200], [0], 40)])
def test_attention_unseen_nan(gpu, dtype, news, past, window):
    """What a row does not see -- the rest of a page, positions before the
    window, the later tokens of its own batch -- may be NaN or infinite."""
    c = Cache(gpu, len(news), 2, 128, 64, dtype, 256, 23, nan=True)
    c.fill([n + p for n, p in zip(news, past)])
    # a token in the middle of each sequence's new ones
    hit = [p + n // 2 for n, p in zip(news, past)]
    for b, p in enumerate(hit):
        c.model.k[b][p, 0, 7] = float("nan")
        c.model.v[b][p, 1, 9] = float("nan")
    c.upload()
    q = torch.randn(sum(news), 8, 128, generator=c.g).half().to(gpu)
    s, kp, vp = c.pages()
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.1, starts=batch(news, gpu),
                                window=window, **s).cpu().double().view(q.shape)
    lo = 0
    for b, (n, p) in enumerate(zip(news, past)):
        k, v = (torch.nan_to_num(x, nan=0.0) for x in (c.model.k[b], c.model.v[b]))
        ref, tol = R.attend(q[lo:lo + n].cpu(), k, v, c.model.ev[b], p, 0.1, window, c.fp8)
        for i in range(n):
            pos = p + i
            sees = pos >= hit[b] and (window == 0 or pos - window < hit[b])
            row = y[lo + i]
            if sees:
                assert row[:4].isnan().all() and row[4:, 9].isnan().all()
                other = torch.ones(128, dtype=torch.bool)
                other[9] = False
                assert ((row - ref[i]).abs() <= tol[i])[4:, other].all()
            else:
                assert ((row - ref[i]).abs() <= tol[i]).all(), (b, i)
        lo += n


@pytest.mark.parametrize("dtype", [FP8, FP16])
def test_attention_wide_scales(gpu, dtype):
    """V blocks of scales from 2^-24 to 2^8, and weights that follow them."""
    c = Cache(gpu, 1, 1, 64, 32, dtype, 400, 24)
    n = 300
    for which in "kv":
        x = torch.randn(n, 1, 64, generator=c.g, dtype=torch.float64)
        if which == "v":
            x *= torch.exp2((torch.arange(n) // 16 * 7 % 28 - 14).double())[:, None, None]
        c.model.put(which, 0, x.half().double())
    c.upload()
    q = (torch.randn(1, 4, 64, generator=c.g) * 6).half().to(gpu)
    check_attend(c, q, [1], 0.125)


def test_attention_extreme_scores(gpu):
    """Scores of +-60000: one position takes all of the weight."""
    c = Cache(gpu, 1, 1, 128, 64, FP16, 200, 25)
    c.fill([150])
    q = torch.full((1, 2, 128), 300.0).half().to(gpu)
    q[0, 1] = -300.0
    check_attend(c, q, [1], 0.2)


@pytest.mark.parametrize("dtype", [FP8, FP16])
def test_rows_that_see_nothing(gpu, dtype):
    """Tokens before position 0 are 0; one past the page table, or that sees a
    page out of range, NaN; rows behind the last sequence keep what they held."""
    c = Cache(gpu, 4, 1, 64, 16, dtype, 48, 26)
    c.fill([2, 40, 48, 30])
    st = torch.tensor([0, 5, 7, 9, 12], dtype=torch.int32, device=gpu)  # 5 new of 2 tokens
    T = 15
    q = torch.randn(T, 2, 64, generator=c.g).half().to(gpu)
    c.lengths[2] = 49                       # its last position is past the table
    c.table[1, 1] = c.pool                  # positions 16 .. 31 of sequence 1
    c.table[3, 0] = -1
    out = torch.full((T, 128), 7.0, dtype=torch.float16, device=gpu)
    s, kp, vp = c.pages()
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.125, starts=st, out=out, **s)
    torch.cuda.synchronize()
    assert y.data_ptr() == out.data_ptr()
    y = y.cpu()
    assert not y[:3].any()
    ref, tol = R.attend(q[3:5].cpu(), c.model.k[0], c.model.v[0], c.model.ev[0], 0, 0.125, 0, c.fp8)
    assert ((y[3:5].double().view(2, 2, 64) - ref).abs() <= tol).all()
    assert y[5:7].isnan().all() and y[8].isnan().all() and y[9:12].isnan().all()
    assert not y[7].isnan().any()
    assert (y[12:] == 7.0).all()
    # a window that the bad page lies outside of
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.125, starts=st, window=7, **s)
    assert not y[5:7].isnan().any() and not y[9:12].isnan().any()


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_rows_that_see_nothing(gpu, dtype, D):
    """The same for prompts."""
    c = Cache(gpu, 4, 1, D, 16, dtype, 800, 32)
    c.fill([40, 700, 784, 100])
    news = [90, 80, 75, 0]
    st = batch(news, gpu)
    q = torch.randn(250, 2, D, generator=c.g).half().to(gpu)
    c.lengths[2] = c.table.shape[1] * 16 + 1  # its last position is past the table
    c.table[1, 10] = c.pool                   # positions 160 .. 175 of sequence 1
    out = torch.full((250, 2 * D), 7.0, dtype=torch.float16, device=gpu)
    s, kp, vp = c.pages()
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.125, starts=st, out=out, **s).cpu()
    assert not y[:50].any()
    ref, tol = R.attend(q[50:90].cpu(), c.model.k[0], c.model.v[0], c.model.ev[0], 0, 0.125, 0,
                        c.fp8)
    assert ((y[50:90].double().view(ref.shape) - ref).abs() <= tol).all()
    assert y[90:170].isnan().all() and y[244].isnan().all()
    # (positions 726 .. 783 of sequence 2; 784 .. 799 hold any bits)
    assert not y[170:228].isnan().any() and (y[245:] == 7.0).all()
    # a window that the bad page lies outside of
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.125, starts=st, window=440, **s)
    assert not y[90:170].isnan().any()


@pytest.mark.parametrize("dtype", [FP8, FP16])
def test_prompt_split_with_infinities(gpu, dtype):
    """Infinities (NaN in 8 bits) of V inside the splits of a prompt's context,
    seen by all rows or by some."""
    c = Cache(gpu, 1, 1, 128, 64, dtype, 2200, 33)
    c.fill([2100])
    n, first = 60, 2040
    for p, d, x in ((3, 5, "inf"), (1500, 5, "inf"), (700, 9, "-inf"), (1999, 11, "nan"),
                    (2070, 20, "inf")):
        c.model.v[0][p, 0, d] = float(x if dtype == FP16 else "nan")
    c.upload()
    q = torch.randn(n, 4, 128, generator=c.g).half().to(gpu)
    s, kp, vp = c.pages()
    y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.1, **s).cpu().double().view(n, 4, 128)
    v = c.model.v[0]
    ref, tol = R.attend(q.cpu(), c.model.k[0], torch.nan_to_num(v, nan=0., posinf=0., neginf=0.),
                        c.model.ev[0], first, 0.1, 0, c.fp8)
    odd = {5: range(n), 9: range(n), 11: range(n), 20: range(30, n)}
    for d in range(128):
        rows = torch.tensor([i in odd.get(d, ()) for i in range(n)])
        assert not y[rows, :, d].isfinite().any()
        assert ((y[~rows, :, d] - ref[~rows, :, d]).abs() <= tol[~rows, :, d]).all()
    if dtype == FP16:
        assert (y[:, :, 5] == float("inf")).all() and (y[:, :, 9] == float("-inf")).all()
        assert y[:, :, 11].isnan().all() and (y[30:, :, 20] == float("inf")).all()


@pytest.mark.parametrize("dtype", [FP8, FP16])
def test_append_out_of_range(gpu, dtype):
    """Nothing is written for positions below 0, past the table, or of pages
    out of range; rows behind the last sequence are not read."""
    c = Cache(gpu, 3, 1, 64, 16, dtype, 48, 27)
    c.fill([0, 0, 0])
    c.table[1, 0] = c.pool + 5
    st = torch.tensor([0, 4, 20, 40], dtype=torch.int32, device=gpu)
    c.lengths.copy_(torch.tensor([2, 16, 60]))
    k = torch.randn(44, 64, generator=c.g).half()
    v = torch.randn(44, 64, generator=c.g).half()
    k[40:] = float("nan")
    q = k.clone()
    before = [None if x is None else x.view(torch.uint8).clone() for x in c.t]
    out = torch.full((44, 1, 64), 7.0, dtype=torch.float16, device=gpu)
    s, kp, vp = c.pages()
    kernels.paged_append(k.to(gpu), v.to(gpu), kp, vp, c.table, c.lengths, starts=st,
                         q=q.to(gpu), q_out=out, **s)
    torch.cuda.synchronize()
    assert torch.equal(out[:40, 0].cpu(), q[:40]) and (out[40:] == 7.0).all()
    # sequence 0: tokens 2, 3 at positions 0, 1; sequence 2: 40 .. 47 of 40 .. 59
    c.model.put("k", 0, k[2:4].double().view(2, 1, 64))
    c.model.put("v", 0, v[2:4].double().view(2, 1, 64))
    gk, gv = c.tokens(0, 2)[:2]
    assert same(gk, c.model.k[0]) and same(gv, c.model.v[0])
    pos = torch.arange(40, 48)
    pg = c.cpu_table[2, pos // 16]
    m = R.Model(1, 1, 64, 16, c.fp8, 1, None)
    m.put("k", 0, k[20:28].double().view(8, 1, 64))
    m.put("v", 0, v[20:28].double().view(8, 1, 64))
    if not c.fp8:
        assert same(c.t[0].cpu()[pg, :, pos % 16].double(), m.k[0])
    else:  # the block had tokens (garbage) before: its scale counts
        e = int(c.t[3].view(torch.uint8)[int(pg[0]), 0, 0])
        assert e >= max(int(m.ev[0][0, 0]) + 127, int(before[3][int(pg[0]), 0, 0]))
    written = {int(c.cpu_table[0, 0]), int(c.cpu_table[2, 2])}
    for x, was in zip(c.t, before):
        if x is not None:
            now = x.view(torch.uint8)
            for p in range(c.pool):
                assert p in written or torch.equal(now[p], was[p]), p


def test_pool_past_32_bits(gpu):
    """Pages that lie past 4 GB of their pool."""
    page, Hk, D = 64, 8, 128
    pool = (1 << 32) // (page * Hk * D) + 300
    k = torch.zeros(pool, Hk, page, D, dtype=torch.uint8, device=gpu).view(FP8)
    v = torch.zeros(pool, Hk, page // 16, D, 16, dtype=torch.uint8, device=gpu).view(FP8)
    ks, vs = (torch.zeros(pool, Hk, page // 16, dtype=torch.uint8, device=gpu)
              .view(torch.float8_e8m0fnu) for _ in range(2))
    small = kernels.paged_cache_tensors(300, Hk, D, page, FP8, gpu)
    L = 200
    g = torch.Generator().manual_seed(1)
    x = [torch.randn(L, Hk * D, generator=g).half().to(gpu) for _ in range(3)]
    table = torch.tensor([[pool - 1, pool - 7, 3, pool - 100]], dtype=torch.int32, device=gpu)
    low = torch.tensor([[299, 293, 3, 200]], dtype=torch.int32, device=gpu)
    n = torch.tensor([L], dtype=torch.int32, device=gpu)
    out = []
    for pages, t in (((k, v, ks, vs), table), (small, low)):
        q = kernels.paged_append(x[1], x[2], pages[0], pages[1], t, n, k_scales=pages[2],
                                 v_scales=pages[3], q=x[0])
        out.append(kernels.paged_attention(q, pages[0], pages[1], t, n, 0.1, k_scales=pages[2],
                                           v_scales=pages[3]))
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1]) and bool(out[0].any())
    assert torch.equal(k.view(torch.uint8)[pool - 1], small[0].view(torch.uint8)[299])


@pytest.mark.parametrize("dtype", [FP8, FP16])
def test_prompt_then_tokens(gpu, dtype):
    """The two together, as a model's layer uses them: ragged prompts, then
    decode steps in a captured graph replayed with other lengths, each step
    checked; a repeated step gives the same bits."""
    B, Hq, Hk, D, page = 3, 8, 2, 128, 32
    c = Cache(gpu, B, Hk, D, page, dtype, 160, 31)
    c.fill([0, 0, 0])
    news = [70, 1, 33]
    q = check_append(c, news, Hq, True, True, 41)
    check_attend(c, q, news, D ** -0.5)
    gen = torch.Generator().manual_seed(9)
    s, kp, vp = c.pages()
    buf = [torch.zeros(B, (Hq + 2 * Hk) * D, dtype=torch.float16, device=gpu),
           torch.zeros(B, D, dtype=torch.float16, device=gpu),
           torch.zeros(B, D, dtype=torch.float16, device=gpu)]
    w = (0.5 + torch.rand(D, generator=gen)).half().to(gpu)

    def step():
        q, k, v = buf[0].split([Hq * D, Hk * D, Hk * D], 1)
        q = kernels.paged_append(k, v, kp, vp, c.table, c.lengths, **s, cos=buf[1], sin=buf[2],
                                 q=q, q_norm_w=w, k_norm_w=w)
        return q, kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.09, **s)

    graph = None
    for i in range(20):
        past = [c.model.k[b].shape[0] for b in range(B)]
        c.lengths.copy_(torch.tensor([p + 1 for p in past]))
        buf[0].copy_(torch.randn(buf[0].shape, generator=gen))
        cos, sin = rope_rows(torch.tensor(past), D)
        buf[1].copy_(cos)
        buf[2].copy_(sin)
        q, y = step()
        if graph is None:
            eager = (q, y)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                gq, gy = step()
        torch.cuda.synchronize()
        want = y.clone()
        gy.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gy, want) and torch.equal(gq, q)
        for b in range(B):
            k, v, ek, ev = c.tokens(b, past[b] + 1)
            c.model.k[b], c.model.v[b] = k, v
            if c.fp8:
                c.model.ek[b], c.model.ev[b] = ek, ev
            ref, tol = R.attend(q[b:b + 1].cpu(), k, v, ev, past[b], 0.09, 0, c.fp8)
            assert ((y[b].cpu().double().view(ref[0].shape) - ref[0]).abs() <= tol[0]).all()
    del eager


def test_other_stream_and_views(gpu):
    """On a stream of the caller's; a page table that is part of a wider one;
    a given workspace."""
    c = Cache(gpu, 2, 2, 64, 16, FP8, 64, 33)
    c.fill([40, 61])
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=gpu)
    wide[:, 2:2 + c.table.shape[1]] = c.table
    t = wide[:, 2:2 + c.table.shape[1]]
    q = torch.randn(2, 4, 64, generator=c.g).half().to(gpu)
    s, kp, vp = c.pages()
    ref = check_attend(c, q, [1, 1], 0.125)
    ws = kernels.paged_attention_workspace(q, kp, t)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = kernels.paged_attention(q, kp, vp, t, c.lengths, 0.125, workspace=ws, **s)
    torch.cuda.synchronize()
    assert torch.equal(y, ref)


def test_graphs_at_once(gpu):
    """Captured calls have workspaces of their own: three graphs replayed on
    streams of their own at once, with eager calls beside them, give the eager
    results every time."""
    c = Cache(gpu, 2, 2, 128, 32, FP8, 5100, 34)
    c.fill([5000, 4000])
    s, kp, vp = c.pages()
    calls = []
    for n in (1, 3, 40):  # merged over workgroups; more rows; a split prompt
        q = torch.randn(2 * n, 8, 128, generator=c.g).half().to(gpu)
        calls.append(lambda q=q: kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.1, **s))
    want = [f().clone() for f in calls]
    graphs = []
    for f in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = f()
        graphs.append((g, y, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(6):
        for _, y, _ in graphs:
            y.zero_()
        torch.cuda.synchronize()
        for g, _, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
        eager = [f() for f in calls]
        torch.cuda.synchronize()
        for (_, y, _), e, w in zip(graphs, eager, want):
            assert torch.equal(y, w) and torch.equal(e, w)
    # a workspace made for more tokens and sequences serves these calls
    ws = kernels.paged_attention_workspace(torch.empty(3000, 8, 128, dtype=FP16, device=gpu), kp,
                                           torch.empty(70, 160, dtype=torch.int32, device=gpu))
    for n, w in zip((1, 3, 40), want):
        q = calls[(1, 3, 40).index(n)].__defaults__[0]
        y = kernels.paged_attention(q, kp, vp, c.table, c.lengths, 0.1, workspace=ws, **s)
        assert torch.equal(y, w)


@pytest.mark.parametrize("dtype", [FP8, FP16])
def test_captured_ragged_batch(gpu, dtype):
    """One captured step of 200 rows replayed for batches that divide them
    otherwise, padded ones among them: pages and results are the eager ones,
    rows behind the last sequence keep what they held."""
    B, T, Hq, Hk, D, page = 4, 200, 8, 2, 64, 32
    c = Cache(gpu, B, Hk, D, page, dtype, 700, 36)
    c.fill([300, 0, 17, 64])
    gen = torch.Generator().manual_seed(37)
    mine = [None if x is None else x.clone() for x in c.t]  # the graph's pages
    st = torch.zeros(B + 1, dtype=torch.int32, device=gpu)
    x = torch.zeros(T, (Hq + 2 * Hk) * D, dtype=torch.float16, device=gpu)
    cos, sin = (t.to(gpu) for t in rope_rows(torch.arange(T), D))
    outs = [torch.zeros(T, Hq * D, dtype=torch.float16, device=gpu) for _ in range(4)]

    def step(t, qo, out):
        q, k, v = x.split([Hq * D, Hk * D, Hk * D], 1)
        s = dict(starts=st, k_scales=t[2], v_scales=t[3])
        q = kernels.paged_append(k, v, t[0], t[1], c.table, c.lengths, cos=cos, sin=sin, q=q,
                                 q_out=qo, **s)
        kernels.paged_attention(qo.view(T, Hq, D), t[0], t[1], c.table, c.lengths, 0.1, out=out,
                                window=250, **s)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(mine, outs[0], outs[1])
    lens = [300, 0, 17, 64]
    for news in ([0, 0, 0, 0], [1, 1, 1, 1], [150, 1, 9, 0], [0, 0, 0, 200], [40, 70, 3, 50],
                 [1, 0, 1, 7]):
        lens = [a + n for a, n in zip(lens, news)]
        st.copy_(torch.tensor([0] + news).cumsum(0))
        c.lengths.copy_(torch.tensor(lens))
        x.copy_(torch.randn(x.shape, generator=gen))
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        step(c.t, outs[2], outs[3])
        torch.cuda.synchronize()
        n = sum(news)
        for o in outs:
            assert (o[n:] == 7.0).all() and not (n and (o[:n] == 7.0).all())
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
        assert outs[1].isfinite().all()
        for a, b in zip(mine, c.t):
            assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_q_in_place(gpu):
    """q_out may be q where its rows lie side by side."""
    c = Cache(gpu, 2, 2, 64, 16, FP16, 64, 35)
    c.lengths.fill_(20)
    k = torch.randn(40, 128, generator=c.g).half().to(gpu)
    q = torch.randn(40, 4, 64, generator=c.g).half().to(gpu)
    cos, sin = (x.to(gpu) for x in rope_rows(torch.arange(40), 64))
    s, kp, vp = c.pages()
    args = (k, k, kp, vp, c.table, c.lengths)
    want = kernels.paged_append(*args, cos=cos, sin=sin, q=q, **s)
    got = kernels.paged_append(*args, cos=cos, sin=sin, q=q, q_out=q, **s)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got.view(want.shape), want)
    with pytest.raises(RuntimeError, match="overlap"):
        kernels.paged_attention(q, kp, vp, c.table, c.lengths, 1.0, out=q.view(40, 256), **s)


def test_refusals(gpu):
    c = Cache(gpu, 2, 2, 64, 16, FP8, 64, 34)
    s, kp, vp = c.pages()
    k = torch.zeros(2, 128, dtype=torch.float16, device=gpu)
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=gpu)
    ok = dict(page_table=c.table, lengths=c.lengths, **s)

    def append(k=k, v=k, kp=kp, vp=vp, **kw):
        kernels.paged_append(k, v, kp, vp, **{**ok, **kw})

    def attend(q=q, kp=kp, vp=vp, **kw):
        kernels.paged_attention(q, kp, vp, **{**ok, "scale": 1.0, **kw})

    append()
    attend()
    for what, call in [
        ("k_scales", lambda: append(k_scales=None)),
        ("scales", lambda: append(kp=kp.to(FP16), vp=vp.to(FP16))),
        ("v_pages", lambda: append(vp=vp.transpose(3, 4).contiguous())),
        ("v_pages", lambda: append(vp=vp.view(torch.uint8))),
        ("k must be", lambda: append(k=k[:, :64])),
        ("rows", lambda: append(v=k[:1])),
        ("do not divide", lambda: append(k=torch.cat([k, k[:1]]), v=torch.cat([k, k[:1]]))),
        ("multiples of 8", lambda: append(k=torch.zeros(2, 132, dtype=FP16, device=gpu)[:, :128])),
        ("float16", lambda: append(k=k.float(), v=k)),
        ("cos and sin", lambda: append(cos=k[:1, :64].contiguous())),
        ("rows of 64", lambda: append(cos=k, sin=k)),
        ("k_norm_w", lambda: append(k_norm_w=k[0])),
        ("multiple of the KV", lambda: append(q=torch.zeros(2, 192, dtype=FP16, device=gpu))),
        ("need a q", lambda: append(q_norm_w=k[0, :64])),
        ("lengths", lambda: append(lengths=c.lengths.long())),
        ("starts", lambda: append(starts=c.lengths)),
        ("page_table", lambda: append(page_table=c.table.T)),
        ("page_table", lambda: attend(page_table=c.table.long())),
        ("window", lambda: attend(window=-1)),
        ("multiple of the KV", lambda: attend(q=q[:, :3].contiguous())),
        ("out must", lambda: attend(out=torch.zeros(2, 128, dtype=FP16, device=gpu))),
        ("workspace", lambda: attend(workspace=[torch.zeros(8, dtype=torch.uint8, device=gpu)] * 2)),
        ("q must be", lambda: attend(q=q[..., :32].contiguous())),
        ("GPU", lambda: attend(q=q.cpu())),
        ("pages' GPU", lambda: append(v=k.cpu())),
        ("GPU", lambda: append(kp=kp.cpu())),
    ]:
        with pytest.raises(RuntimeError, match=what):
            call()
    with pytest.raises(RuntimeError, match="power of two"):
        kernels.paged_cache_tensors(2, 1, 64, 48, FP8, gpu)
    torch.cuda.synchronize()
    # nothing to do
    assert kernels.paged_attention(q[:0], kp, vp, scale=1.0, **ok).shape == (0, 256)
    assert kernels.paged_append(k[:0], k[:0], kp, vp, q=q[:0], **ok).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-8, -1e-8, 1e-38, 1e-45])
@pytest.mark.parametrize("news,past", [([1, 1], [40, 69]), ([40, 33], [0, 70])])
def test_attention_any_scale(gpu, dtype, D, scale, news, past):
    """Scales below, at and next to zero, down to the smallest fp32 one, in both
    forms: blocks that no token has written have the scale 2^-127 in a cache of
    zeros, and what rows do not see has no weight all the same."""
    c = Cache(gpu, 2, 2, D, 16, dtype, 140, 38)
    for x in c.t:
        if x is not None:
            x.view(torch.uint8).zero_()
    c.fill([n + p for n, p in zip(news, past)])
    q = (torch.randn(sum(news), 4, D, generator=c.g) * 2).half().to(gpu)
    check_attend(c, q, news, scale)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rise", [16.0, 24.0, 26.0, 30.0])
def test_prompt_scores_that_rise(gpu, dtype, D, rise):
    """Scores that rise by 7.5 (in powers of two), which the running maximum
    leaves, and then further: the weights of 2^7.5 that wait for their product
    by then keep what the new maximum leaves of them."""
    c = Cache(gpu, 1, 1, D, 32, dtype, 160, 39)
    n, first = 40, 96
    k = torch.zeros(first + n, 1, D, dtype=torch.float64)
    v = torch.zeros_like(k)
    k[32:64, 0, 0] = 7.5
    k[70, 0, 0] = rise
    v[32:64, 0, :D - 1] = 1.0
    v[:, 0, D - 1] = 1.0  # (every block of one scale)
    c.model.put("k", 0, k)
    c.model.put("v", 0, v)
    c.upload()
    q = torch.zeros(n, 1, D, dtype=torch.float16, device=gpu)
    q[..., 0] = 1.0
    check_attend(c, q, [n], math.log(2.0))


def test_append_output_between_rows(gpu):
    """q_out may lie between the rows of a strided k and v, and a single token's
    fused row of q, k and v is rotated in place; over their rows it is refused."""
    c = Cache(gpu, 2, 2, 64, 16, FP16, 64, 41)
    c.lengths.fill_(20)
    T, S = 40, 40000
    buf = torch.randn(T, S, generator=c.g).half().to(gpu)
    k, v = buf[:, :128], buf[:, 20000:20128]
    q = torch.randn(T, 4, 64, generator=c.g).half().to(gpu)
    cos, sin = (x.to(gpu) for x in rope_rows(torch.arange(T), 64))
    s, kp, vp = c.pages()
    args = (kp, vp, c.table, c.lengths)

    def held():  # bits (there is garbage in the pool)
        return torch.cat([x.view(torch.int16).flatten() for x in (kp, vp)])

    want = kernels.paged_append(k, v, *args, cos=cos, sin=sin, q=q, **s)
    pages = held()
    between = buf[3, 128:128 + T * 256].view(T, 4, 64)
    got = kernels.paged_append(k, v, *args, cos=cos, sin=sin, q=q, q_out=between, **s)
    assert got.data_ptr() == between.data_ptr() and torch.equal(got, want)
    assert torch.equal(held(), pages)
    for bad in (buf[3, :T * 256], buf[3, 19968:19968 + T * 256]):
        with pytest.raises(RuntimeError, match="overlap"):
            kernels.paged_append(k, v, *args, q=q, q_out=bad, **s)
    one = torch.randn(1, 512, generator=c.g).half().to(gpu)
    q, k, v = one.split([256, 128, 128], 1)
    args = (kp, vp, c.table[:1], torch.ones(1, dtype=torch.int32, device=gpu))
    at = dict(cos=cos[5:6], sin=sin[5:6], **s)
    want = kernels.paged_append(k, v, *args, q=q, **at)
    pages = held()
    kernels.paged_append(k, v, *args, q=q, q_out=q, **at)
    assert torch.equal(q.view(1, 4, 64), want)
    assert torch.equal(held(), pages)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@pytest.mark.parametrize("D,new,past,window", [
    (64, 640, 3707, 0), (128, 640, 3707, 0),  # 137 steps in one run
    (64, 640, 7000, 4357), (128, 640, 7000, 4357),  # that begin past 0
    (64, 640, 8001, 0), (128, 640, 8001, 0),  # 270 steps in two parts
])
def test_prompt_long_runs(gpu, dtype, D, new, past, window):
    """Prompts of 320 units, two a CU: runs of far more steps than a workgroup
    looks up at once, and a long context's two parts of a unit.  Sampled rows and
    heads."""
    Hq, Hk, page = 64, 16, 32
    L = new + past
    P = -(-L // page)
    pool = P + 5
    g = torch.Generator().manual_seed(40)
    table = torch.randperm(pool, generator=g)[:P].to(torch.int32)
    kp, vp, ks, vs = kernels.paged_cache_tensors(pool, Hk, D, page, dtype, gpu)
    for x in (kp, vp):
        x.copy_(torch.randn(x.shape, generator=g).to(dtype))
    if dtype == FP8:  # scales from 2^-2 to 2
        for x in (ks, vs):
            x.view(torch.uint8).copy_(torch.randint(125, 129, x.shape, generator=g))
    q = torch.randn(new, Hq, D, generator=g).half()
    lengths = torch.tensor([L], dtype=torch.int32, device=gpu)
    y = kernels.paged_attention(q.to(gpu), kp, vp, table.view(1, P).to(gpu), lengths, 0.1,
                                k_scales=ks, v_scales=vs, window=window)
    torch.cuda.synchronize()
    y = y.cpu().double().view(new, Hq, D)
    pg = table.long()
    for h in (0, 7, 15):
        k = kp.cpu()[pg, h].double()               # (P, page, D)
        v = vp.cpu()[pg, h].double().mT            # (P, blocks, 16, D)
        ev = torch.zeros(1, P * page // 16, dtype=torch.int64)
        if dtype == FP8:
            ek, ev = (x.view(torch.uint8).cpu()[pg, h].long() - 127 for x in (ks, vs))
            k = k.view(P, -1, 16, D) * torch.exp2(ek.double())[..., None, None]
            v = v * torch.exp2(ev.double())[..., None, None]
            ev = ev.view(1, -1)
        k, v = (x.reshape(-1, 1, D)[:L] for x in (k, v))
        for i in (0, 290, new - 12):  # 48 rows of the KV head
            heads = slice(4 * h, 4 * h + 4)
            ref, tol = R.attend(q[i:i + 12, heads], k, v, ev, past + i, 0.1, window, dtype == FP8)
            d = (y[i:i + 12, heads] - ref).abs()
            assert (d <= tol).all(), (h, i, float((d / tol).max()))
