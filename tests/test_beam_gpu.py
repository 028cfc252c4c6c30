"""The selection of beam search (kernels.beam_select) against its formula in 64
bits: places exactly, scores to the rounding of an fp32 value.

The bound of a score: c = s + x - lse is fp32-rounded once, 2^-24 |c|; its fp64
sums are off by 4 * 6e-11 (the exponential's series: a term has up to four of them,
as it is added, in its lane, its part and its row) and 1e-13 (V terms), and by the
rounding of values up to |s| + |x| + |lse| < 2^17, 2^-36 = 1.5e-11: 3e-10."""

import math

import pytest
import torch

from glorcq_amd import kernels

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


def reference(logits, scores, num):
    """In fp64 on the CPU: (scores, parents, tokens)."""
    B, K = scores.shape
    x = logits.reshape(B, K, -1).double().cpu()
    V = x.shape[2]
    s = scores.double().cpu()
    m = x.amax(-1, keepdim=True)
    fine = torch.isfinite(m)
    lse = torch.where(fine, m + torch.log(torch.exp(x - torch.where(fine, m, 0.0))
                                          .sum(-1, keepdim=True)), m)
    c = s[..., None] + (x - lse)
    nan = (x.isnan() | (x == INF)).any(-1) | s.isnan() | (s == INF)
    none = (m[..., 0] == -INF) | (s == -INF)
    c = torch.where(none[..., None], -INF, torch.where(x == -INF, -INF, c))
    c = torch.where(nan[..., None], NAN, c)
    # (torch sorts NaN as the largest)
    v, i = c.view(B, K * V).sort(dim=1, descending=True, stable=True)
    return v[:, :num], i[:, :num] // V, i[:, :num] % V


def check(logits, scores, num):
    s, p, t = kernels.beam_select(logits, scores, num)
    torch.cuda.synchronize()
    assert s.dtype == torch.float32 and p.dtype == t.dtype == torch.int64
    rs, rp, rt = reference(logits, scores, num)
    assert torch.equal(p.cpu(), rp) and torch.equal(t.cpu(), rt)
    s = s.cpu().double()
    assert torch.equal(s.isnan(), rs.isnan())
    inf = rs.isinf()
    assert torch.equal(s[inf], rs[inf])
    ok = inf | rs.isnan()
    assert ((s - rs).abs() <= 2.0 ** -24 * rs.abs() + 3e-10)[~ok].all()
    return s, p, t


def make(gpu, B, K, V, dtype, seed, pad=0, amp=3.0):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(B * K, V + pad, generator=g) * amp
    rows[:, V:] = 1000.0
    scores = (-10 * torch.rand(B, K, generator=g)).to(gpu)
    return rows.to(dtype).to(gpu)[:, :V], scores


DTYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,K,V,num", [
    (1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 1, 3), (1, 2, 5, 10), (1, 4, 255, 8), (3, 5, 2047, 10),
    (2, 2, 2048, 4), (2, 2, 2049, 3), (1, 4, 8192, 8), (1, 64, 1000, 128), (1, 1, 50257, 128),
    (2, 16, 8193, 32), (1, 3, 151936, 6), (20, 8, 32001, 16), (300, 1, 900, 2), (5, 7, 100, 70),
])
def test_sizes(gpu, dtype, B, K, V, num):
    check(*make(gpu, B, K, V, dtype, 1), num)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [1, 3, 64])
def test_rows_of_a_wider_matrix(gpu, dtype, pad):
    """What lies behind a row's vocabulary is not looked at; rows begin anywhere."""
    x, s = make(gpu, 3, 4, 5003, dtype, 2, pad=pad)
    check(x, s, 8)
    check(x.unflatten(0, (3, 4)), s, 8)
    check(x.unflatten(0, (3, 4))[:, :1], s[:, :1].contiguous(), 8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("num", [1, 5, 16, 128])
def test_ties(gpu, dtype, num):
    """Equal logits, equal beams: the lowest places; 0 and -0 are equal."""
    x = torch.zeros(2 * 3, 9000, dtype=dtype, device=gpu)
    x[:, 1::3] = -0.0
    s = torch.tensor([[-1.0, -1.0, -0.5], [-2.0, -1.0, -1.0]], device=gpu)
    _, p, t = check(x, s, num)
    assert (p[0] == 2).all() and (p[1] == 1).all() and torch.equal(t[0].cpu(), torch.arange(num))
    x[:, 4000:8000:7] = 2.0
    check(x, s, num)
    y, _ = make(gpu, 1, 1, 20011, dtype, 3)
    check(y.expand(4, -1).contiguous(), torch.zeros(1, 4, device=gpu), num)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sorted_rows(gpu, dtype):
    """All of the best in one place: more than a group's share of a part."""
    x = torch.arange(16384, dtype=torch.float32).view(1, -1) / 64
    s = torch.zeros(1, 1, device=gpu)
    for row in (x, x.flip(1), x.view(1, 8, -1).mT.reshape(1, -1)):
        check(row.to(dtype).to(gpu), s, 64)
        check(row.to(dtype).to(gpu), s, 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("num", [1, 16, 128])
@pytest.mark.parametrize("how", ["random", "rising", "falling", "equal", "steps", "late", "masked",
                                 "jumps"])
def test_many_rows(gpu, dtype, num, how):
    """Rows in parts of several chunks of 2048: what stands in a later chunk, or
    only there; values that rise along the row, so that each chunk is better than
    those before; equal ones; sums whose largest term comes 1000 above the rest."""
    B, K, V = 12, 8, 49160
    x, s = make(gpu, B, K, V, dtype, 16)
    at = torch.arange(V, device=gpu, dtype=torch.float32)
    if how in ("rising", "falling"):
        x = ((at if how == "rising" else at.flip(0)) / 512 - 40).expand(B * K, -1)
    elif how == "equal":
        x = torch.full((B * K, V), 0.5, device=gpu)
    elif how == "steps":
        x = (at // 1000 % 7).expand(B * K, -1)
    elif how == "late":
        x = x.float() - 20 * (at < 47000)
    elif how == "masked":  # all of the first chunks of every part
        x = x.float().masked_fill((at % 6145) < 4500, -INF)
    elif how == "jumps":
        x = x.float() + 1000 * (at % 6145 > 6000) * (torch.arange(B * K, device=gpu) % 2)[:, None]
    x = x.to(dtype).contiguous()
    a, p, t = kernels.beam_select(x, s, num)
    # the formula in fp64, on the GPU
    y = x.double().view(B, K, V)
    c = (s.double()[..., None] + torch.log_softmax(y, -1)).view(B, K * V)
    v, i = c.sort(dim=1, descending=True, stable=True)
    v, i = v[:, :num], i[:, :num]
    assert torch.equal(p, i // V) and torch.equal(t, i % V)
    assert ((a.double() - v).abs() <= 2.0 ** -24 * v.abs() + 3e-10).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("num", [7, 64, 128])
@pytest.mark.parametrize("step", [0.0, 0.25, -0.25, 2.0])
@pytest.mark.parametrize("levels", [False, True])
def test_beams_far_apart(gpu, dtype, num, step, levels):
    """Most of a few beams' best are better than any of the others', more than a
    list holds; with levels (multiples of 1/2) many of them are the same."""
    x, _ = make(gpu, 2, 64, 9001, dtype, 41)
    if levels:
        x = (x.float() * 2).round().to(dtype) / 2
    scores = (torch.arange(64.0) * step).repeat(2, 1).to(gpu)
    check(x, scores, num)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("step", [0.0, 1.0])
def test_more_parts_than_threads(gpu, dtype, step):
    x, _ = make(gpu, 1, 16, 151936, dtype, 42)
    check(x, (torch.arange(16.0) * step).view(1, 16).to(gpu), 128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("num", [16, 100])
@pytest.mark.parametrize("at", [0, 9000, 29990])
def test_rows_mostly_of_the_lowest_value(gpu, dtype, num, at):
    x = torch.full((16, 30001), torch.finfo(dtype).min, dtype=dtype)
    x[:, at:at + 5] = torch.linspace(-2, 2, 80).reshape(16, 5).to(dtype)
    g = torch.Generator().manual_seed(43)
    check(x.to(gpu), -torch.rand(2, 8, generator=g).to(gpu), num)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_in_a_later_chunk(gpu, dtype):
    x, s = make(gpu, 12, 8, 49160, dtype, 17)
    x[3, 5000], x[11, 49159], x[20, 3000] = NAN, INF, -INF
    a, p, t = kernels.beam_select(x, s, 6)
    for b, k in ((0, 3), (1, 3)):
        assert a[b].isnan().all() and (p[b] == k).all() and t[b].tolist() == list(range(6))
    assert torch.isfinite(a[2:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("left", [0, 1, 5, 40, 3000])
def test_masked(gpu, dtype, left):
    """Few tokens allowed (none, in some beams): -inf comes last, by place."""
    x, s = make(gpu, 3, 4, 30011, dtype, 5)
    keep = torch.zeros(12, 30011, dtype=torch.bool, device=gpu)
    g = torch.Generator().manual_seed(6)
    for r in (0, 2, 5, 8, 9, 10, 11):
        keep[r, torch.randperm(30011, generator=g)[:left].to(gpu)] = True
    x = x.masked_fill(~keep, -INF)
    for num in (1, 8, 100):
        check(x, s, num)


@pytest.mark.parametrize("dtype", DTYPES)
def test_unused_beams(gpu, dtype):
    """A first step: beams with a score of -inf are chosen after everything else."""
    x, s = make(gpu, 2, 4, 1003, dtype, 7)
    s[:, 1:] = -INF
    _, p, _ = check(x, s, 8)
    assert (p == 0).all()
    x[:, 5:] = -INF  # 5 continuations, the rest by place
    check(x, s, 8)
    s[:] = -INF
    check(x, s, 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan(gpu, dtype):
    """NaN and +inf make all of a beam NaN, and that comes first."""
    for where in ("logit", "inf", "score", "inf score"):
        x, s = make(gpu, 2, 5, 2100, dtype, 8)
        if where == "logit":
            x[3, 2099] = NAN
        elif where == "inf":
            x[3, 17] = INF
        else:
            s[0, 3] = NAN if where == "score" else INF
        _, p, t = check(x, s, 9)
        assert (p[0] == 3).all() and t[0].tolist() == list(range(9)) and not (p[1] == 3).all()
    # beams of few tokens: the NaN ones, then the others
    x, s = make(gpu, 1, 5, 3, dtype, 9)
    x[1, 0], x[4, 2], x[2, 1] = NAN, INF, -INF
    for num in (2, 5, 6, 8, 15):
        check(x, s, num)
    x[:] = NAN
    check(x, s, 15)


def test_extreme_logits(gpu):
    """The largest and smallest values of the types, all in one row."""
    for dtype in DTYPES:
        f = torch.finfo(dtype)
        x = torch.zeros(2, 4000, dtype=dtype, device=gpu)
        x[0, 10], x[0, 3000], x[1, 7] = f.max, f.max, f.min
        x[1, 100:] = f.min
        s = torch.tensor([[-3.0, -1.0]], device=gpu)
        a, p, t = kernels.beam_select(x, s, 6)
        # (log 2 beside 65504 and more: the reference's fp64 is as good as any)
        rs, rp, rt = reference(x, s, 6)
        assert torch.equal(p.cpu(), rp) and torch.equal(t.cpu(), rt)
        assert torch.allclose(a.cpu().double(), rs, rtol=1e-6)


def test_large_logits(gpu):
    """Values beside which a shift by a few hundred rounds to nothing: of 3000
    logits two count, so that each has a half."""
    for size, tol in ((1e9, 1e-6), (1e12, 1e-3)):  # (fp64's steps there: 1e-7 and 1e-4)
        x = torch.zeros(1, 3000, device=gpu)
        x[0, 5], x[0, 2500] = size, size
        a, _, t = kernels.beam_select(x, torch.full((1, 1), -1.0, device=gpu), 2)
        assert t[0].tolist() == [5, 2500]
        assert ((a[0].double() + 1 + math.log(2)).abs() < tol + 2.0 ** -23).all()


@pytest.mark.parametrize("base", [2.0 ** 33, 1e10, 14e6 * 1024, -1e10, -(2.0 ** 34 - 2048), -2.0 ** 33])
@pytest.mark.parametrize("num", [4, 100])
def test_large_logits_in_later_chunks(gpu, base, num):
    """Logits that grow by 1024 along a part of several chunks, where 1024 is
    fp32's step: the largest are the whole sum.  They and their differences are
    exact in fp64, so a score is off by the fp64 rounding of lse, half a step of
    values up to 2^34 (2^-20), where log 2 comes in, once in each side, and the
    fp32 rounding of what is given."""
    B, K, V = 12, 8, 49160
    x = torch.full((B * K, V), base, device=gpu)
    at = torch.arange(V, device=gpu)
    x[:, at % 6145 > 5000] = base - 2048
    ones, twos = torch.arange(0, B * K, 2, device=gpu), torch.arange(1, B * K, 2, device=gpu)
    x[ones, 40001 + ones] = base + 1024   # one that counts
    x[twos, 9001 + twos] = base + 1024    # two, in different parts
    x[twos, 47003 + twos] = base + 1024
    s = -2 * torch.arange(K, device=gpu, dtype=torch.float32).expand(B, -1).contiguous()
    a, p, t = kernels.beam_select(x, s, num)
    rs, rp, rt = reference(x, s, num)
    assert torch.equal(p.cpu(), rp) and torch.equal(t.cpu(), rt)
    assert ((a.cpu().double() - rs).abs() <= 2.0 ** -24 * rs.abs() + 2 * 2.0 ** -20 + 3e-10).all()


def test_subnormal_logits_keep_their_order(gpu):
    x = torch.zeros(1, 3000, dtype=torch.float16, device=gpu)
    x[0, 2000], x[0, 1000], x[0, 500] = 3 * 2.0 ** -24, 2 * 2.0 ** -24, 2.0 ** -24
    _, _, t = check(x, torch.zeros(1, 1, device=gpu), 5)
    assert t[0].tolist() == [2000, 1000, 500, 0, 1]


def test_streams_and_graphs(gpu):
    """Calls on two streams at once, and graphs whose replays have other logits,
    with eager calls between."""
    x, s = make(gpu, 4, 4, 20011, torch.float16, 10)
    y, _ = make(gpu, 4, 4, 20011, torch.float16, 11)
    want = [kernels.beam_select(z, s, 8) for z in (x, y)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, z in zip(streams, (x, y)):
            with torch.cuda.stream(st):
                got.append(kernels.beam_select(z, s, 8))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for u, w in zip(got, want) for a, b in zip(u, w))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kernels.beam_select(x, s, 8))
        graphs.append(g)
    for seed in (12, 13, 14):
        x.copy_(make(gpu, 4, 4, 20011, torch.float16, seed)[0])
        want = kernels.beam_select(x, s, 8)
        for st, g in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(gpu):
    x, s = make(gpu, 2, 3, 100, torch.float16, 15)
    for args, what in (
            ((x, s, 0), "num"), ((x, s, -1), "num"), ((x, s, 129), "num"),
            ((x[:, :1].contiguous(), s, 4), "num"), ((x.double(), s, 2), "float32"),
            ((x.cpu(), s, 2), "GPU"), ((x, s.cpu(), 2), "scores"), ((x, s.half(), 2), "scores"),
            ((x, s[0], 2), "scores"), ((x[:5], s, 2), "rows"), ((x.T, s, 2), "rows"),
            ((x[:, ::2], s, 2), "contiguous"), ((x[:1].expand(6, -1), s, 2), "contiguous"),
            ((x.view(2, 3, 100).transpose(0, 1).contiguous().transpose(0, 1), s, 2), "contiguous"),
            ((x[:, :0], s, 1), "vocab"), ((x.new_zeros(65, 4), s.new_zeros(1, 65), 1), "beams")):
        with pytest.raises(RuntimeError, match=what):
            kernels.beam_select(*args)
    a, b, c = kernels.beam_select(x[:0], s[:0], 2)
    assert a.shape == b.shape == c.shape == (0, 2)
