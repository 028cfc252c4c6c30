"""The paged cache's operators restated in 64 bits on the CPU (formula by
formula, a sequence at a time), with the bounds that the kernels' 32-bit
arithmetic and their roundings stay within.

Roundings: fp32 2^-24, fp16 2^-11 of the value (half a step), e4m3 exact in
fp16.  Sums of n fp32 terms: n 2^-23 of the sum of magnitudes (the matrix
instructions may truncate where they align their terms).
"""

import math

import torch

BLOCK = 16
MIN_EXP = -32
NAN = float("nan")


def e4m3_of(x):
    """float64 -> the nearest e4m3 value (ties to even), |x| <= 448 (1 + tiny)."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def scale_exp(amax):
    """Smallest e >= MIN_EXP with amax <= 448 2^e."""
    e = MIN_EXP
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def head_norm_rope(x, w, cos, sin, eps):
    """x (T, H, D) fp16 -> (value, bound on the fp32 arithmetic's error)."""
    x = x.double()
    D = x.shape[-1]
    rel = 0.0
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
        # the sum of D squares (a tree of depth 10 at most, fma), /D, + eps,
        # rsqrt (1 ulp = 2 half steps), two products: half the sum's error counts
        rel = (12 / 2 + 2 + 3) * 2.0 ** -24
    if cos is None:
        return x, rel * x.abs()
    h = D // 2
    turned = torch.cat([-x[..., h:], x[..., :h]], -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    mag = (x * c).abs() + (turned * s).abs()
    return x * c + turned * s, (rel + 2 * 2.0 ** -24) * mag


class Model:
    """A cache of one layer as logical tokens: k, v[b] (L, Hk, D) float64 of
    the values held, ek, ev[b] (Hk, blocks) exponents (8 bits)."""

    def __init__(self, B, Hk, D, page, fp8, pool, gen, spare_nan=False):
        self.B, self.Hk, self.D, self.page, self.fp8, self.pool = B, Hk, D, page, fp8, pool
        self.k = [torch.zeros(0, Hk, D, dtype=torch.float64) for _ in range(B)]
        self.v = [torch.zeros(0, Hk, D, dtype=torch.float64) for _ in range(B)]
        self.ek = [torch.zeros(Hk, 0, dtype=torch.int64) for _ in range(B)]
        self.ev = [torch.zeros(Hk, 0, dtype=torch.int64) for _ in range(B)]

    def put(self, which, b, x):
        """Appends x (n, Hk, D) float64 to sequence b (block by block)."""
        old = getattr(self, which)[b]
        if not self.fp8:
            getattr(self, which)[b] = torch.cat([old, x.half().double()])
            return
        exps = getattr(self, "e" + which)[b]
        L, n = old.shape[0], x.shape[0]
        vals = torch.cat([old, x])
        nb = -(-(L + n) // BLOCK)
        exps = torch.cat([exps, torch.full((self.Hk, nb - exps.shape[1]), MIN_EXP)], 1)
        for i in range(L // BLOCK, nb):
            lo, hi = i * BLOCK, min((i + 1) * BLOCK, L + n)
            keep = max(0, min(L, hi) - lo)
            for h in range(self.Hk):
                new = vals[lo + keep:hi, h]
                fine = new[torch.isfinite(new)]
                e = scale_exp(float(fine.abs().max()) if fine.numel() else 0.0)
                if keep:
                    e = max(e, int(exps[h, i]))
                exps[h, i] = e
                c = vals[lo:hi, h] * 2.0 ** -e
                c = torch.where(torch.isfinite(c), c, torch.zeros((), dtype=c.dtype) + NAN)
                vals[lo:hi, h] = torch.where(torch.isnan(c), c, e4m3_of(c) * 2.0 ** e)
        getattr(self, which)[b] = vals
        getattr(self, "e" + which)[b] = exps


def attend(q, k, v, ev, first, scale, window, fp8):
    """q (n, Hq, D) fp16 at positions first .. ; k, v (L, Hk, D) float64 of one
    sequence; ev (Hk, blocks) exponents of the V blocks -> (out, bound)
    (n, Hq, D) float64.

    The bound, a row: 2^-11 of the output, and with p the softmax weights,
    u = 2^-24 (natural logs of a score t's error become p's relative error):
      score: D products summed, 2 D u sum |q k| scale; scale and exponent
             products, sums and exp2: 8 u (|t| + 32 + 1)
      p is rounded to fp16 (2^-11) against the largest weight 2^M of a block's
      share: 2^-25 absolute where it is subnormal.  With more than 32 rows a
      KV head the kernel's maximum m is a whole power of two that has followed
      the scores: m < M + 1 (ceil), so 2^-25 2^m <= 2 2^-25 2^M; and a weight
      still to be used when m follows is scaled by the power of two and rounded
      a second time, the first error then no larger than before in units of
      2^m: two of them, 4 2^-25 2^M at most
      sums over L positions: 2 L u
    """
    n, Hq, D = q.shape
    L, Hk = k.shape[:2]
    rep = Hq // Hk
    u = 2.0 ** -24
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(n):
        pos = first + i
        lo = max(0, pos - window + 1) if window else 0
        if pos < 0:
            continue
        for h in range(Hk):
            kk, vv = k[lo:pos + 1, h], v[lo:pos + 1, h]
            qq = q[i, h * rep:(h + 1) * rep].double()
            t = qq @ kk.T * scale
            p = torch.softmax(t, -1)
            r = p @ vv
            out[i, h * rep:(h + 1) * rep] = r
            mag = qq.abs() @ kk.abs().T * abs(scale)
            d = (2 * D * u * mag + 8 * u * (t.abs() + 33)).amax(-1, keepdim=True)
            pv = p @ vv.abs()
            e = ev[h][torch.arange(lo, pos + 1) // BLOCK].double() if fp8 else torch.zeros(len(kk))
            e = e.double()
            # the weights' subnormals: |code| 2^-25 2^M a position, over sum 2^t
            t2 = t * math.log2(math.e)
            M = (t2 + e).amax(-1, keepdim=True)
            total = torch.exp2(t2 - M).sum(-1, keepdim=True)
            codes = (vv * torch.exp2(-e)[:, None]).abs().sum(0)
            sub = (4 if n * rep > 32 else 1) * 2.0 ** -25 * codes / total
            tol[i, h * rep:(h + 1) * rep] = (
                2.0 ** -11 * r.abs() + 2.0 ** -25  # (fp16 subnormal outputs)
                + (2.0 ** -11 + 2 * d + 2 * L * u + 4 * u) * pv * 1.001 + sub)
    return out, tol
