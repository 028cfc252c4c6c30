"""The paged key/value cache's operators as cases that can be timed.

append   kernels.paged_append: the new tokens of a batch of sequences -- head
         RMSNorm of q and k, rotary embedding, k and v into the pages of a
         cache of fp16 values or of 8-bit ones (e4m3 codes, a power-of-two
         scale for each 16 tokens of a KV head) -- and the rotated q
attend   kernels.paged_attention: causal attention of those tokens over the
         pages, one token a sequence (decode steps) or many (prompts, chunks of
         prompts, both in one batch)

Sequences have lengths of their own; the pages of a sequence lie anywhere in
the pool.  32 query and 4 KV heads of 128 are the Qwen3-MoE-shaped model's
heads, 16 and 16 those of Qwen1.5-MoE-A2.7B; 64-wide heads and other ratios are
generic.

With `own` false `run` computes the operators with elementary torch
operations; `exact` restates them in 64 bits.

Layouts (BT = 16 tokens a block): k pages (pages, Hk, page, D), v pages (pages,
Hk, page / BT, D, BT), scales (pages, Hk, page / BT), page table (sequences,
pages a sequence), lengths (sequences) with the new tokens among them.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
BT = 16          # tokens of a scale block
EPS = 1e-6
FP8_MAX = 448.0  # largest e4m3 value
MIN_EXP = -32    # smallest scale: 2^MIN_EXP
THETA = 1e6


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _case(name, op, seqs, new, past, heads=(32, 4), dim=128, page=64, kv="fp8", norm=True,
          window=0, ones=0, lens=1):
    """new, past: (fewest, most) tokens a sequence brings and has behind it;
    equal ones make a batch of one shape.  ones: sequences, the first ones, that
    bring one token.  lens: the draw of the lengths."""
    return {"name": name, "op": op, "seqs": seqs, "ones": ones, "new_lo": new[0], "new_hi": new[1],
            "past_lo": past[0], "past_hi": past[1], "q_heads": heads[0], "kv_heads": heads[1],
            "dim": dim, "page": page, "kv": kv, "norm": norm, "window": window, "lens": lens}


def listed():
    return [
        # one decode token of one sequence: latency
        _case("append_one", "append", 1, (1, 1), (1000, 1000)),
        # a decode step of a serving batch, sequences of all lengths
        _case("append_batch", "append", 64, (1, 1), (3, 8000)),
        # prompts of a batch, each of its own length, or what is left of them
        _case("append_prompts", "append", 7, (37, 1900), (0, 700)),
        # the same without quantization or q/k norms, as many KV heads as query heads
        _case("append_prompts_fp16", "append", 3, (500, 1100), (0, 50), heads=(16, 16), page=16,
              kv="fp16", norm=False),
        # one decode token of one sequence over a short context: latency
        _case("decode_one", "attend", 1, (1, 1), (516, 516)),
        # one sequence with a long context
        _case("decode_long", "attend", 1, (1, 1), (130001, 130001)),
        # a decode step of a serving batch, sequences of all lengths
        _case("decode_batch", "attend", 64, (1, 1), (3, 8000)),
        # a batch of one length over a cache of fp16 values
        _case("decode_fp16", "attend", 16, (1, 1), (3999, 3999), kv="fp16"),
        # as many KV heads as query heads, 64 wide, small pages
        _case("decode_mha", "attend", 33, (1, 1), (10, 2100), heads=(16, 16), dim=64, page=16),
        # a prompt
        _case("prompt", "attend", 1, (4096, 4096), (0, 0)),
        # a chunk of a prompt with a long context behind it
        _case("chunk_long", "attend", 1, (512, 512), (30000, 30000)),
        # decode tokens and chunks of prompts in one batch, a sliding window
        _case("mixed_window", "attend", 22, (90, 700), (0, 6000), page=32, window=4096, ones=14),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_BYTES, MOST_FLOPS = 2.6e8, 2.5e11
HEADS = ((32, 4), (16, 16), (32, 8), (16, 2), (12, 4), (28, 4), (8, 1), (64, 4))


def draw(rng):
    op = rng.choice(("append", "attend", "attend"))
    many = rng.random() < 0.5  # prompts or decode steps
    heads = rng.choice(HEADS)
    kv = rng.choice(("fp8", "fp8", "fp16"))
    dim = rng.choice((128, 128, 64))
    page = rng.choice((16, 32, 64, 128))
    window = rng.choice((0, 0, 0, _log_int(rng, 16, 5000))) if op == "attend" else 0
    if many:
        seqs = _log_int(rng, 1, 12)
        hi = _log_int(rng, 2, 4000 // seqs)
        lo = rng.choice((1, hi, max(1, hi // 3)))
        past_hi = rng.choice((0, _log_int(rng, 1, 12000 // seqs)))
    else:
        seqs = _log_int(rng, 1, 96)
        lo, hi = 1, rng.choice((1, 1, 1, 2, 5))
        past_hi = _log_int(rng, 1, min(60000, 250000 // seqs))
    past_lo = rng.choice((0, past_hi, past_hi // 4))
    c = _case("", op, seqs, (lo, hi), (past_lo, past_hi), heads, dim, page, kv,
              rng.random() < 0.7, window, rng.choice((0, seqs // 2)) if many else 0,
              rng.randrange(1 << 20))
    del c["name"]
    while (w := work(c))["bytes"] > MOST_BYTES or w["flops"] > MOST_FLOPS:
        # to the work of the largest listed ones
        at = "past_hi" if c["past_hi"] > c["new_hi"] else "new_hi"
        c[at] = c[at] * 2 // 3
        for k in ("new", "past"):
            c[k + "_lo"] = min(c[k + "_lo"], c[k + "_hi"])
    return c


def _lengths(c):
    """(new, past): tokens each sequence brings and has behind it."""
    r = random.Random(c["lens"])
    new = [r.randint(c["new_lo"], c["new_hi"]) if b >= c["ones"] else 1 for b in range(c["seqs"])]
    past = [r.randint(c["past_lo"], c["past_hi"]) for _ in range(c["seqs"])]
    return new, past


def work(c):
    new, past = _lengths(c)
    T, Hq, Hk, D = sum(new), c["q_heads"], c["kv_heads"], c["dim"]
    size = 1 if c["kv"] == "fp8" else 2
    block = 2 * D * size + (2 / BT if c["kv"] == "fp8" else 0)  # k and v of a token and KV head
    if c["op"] == "append":
        # q, k, v, cos and sin read; q and the pages written
        return {"bytes": T * (2 * D * (2 * Hq + 2 * Hk + 2) + Hk * block),
                "flops": T * D * (Hq + Hk) * 8}
    w = c["window"] or 1 << 30
    pairs = read = 0
    for n, p in zip(new, past):
        # the query at position q sees min(q + 1, window) positions
        a, b = p + 1, p + n
        full = max(0, min(b, w) - a + 1)
        pairs += full * (a + min(b, w)) // 2 + (n - full) * w
        read += b - max(0, a - w)
    return {"bytes": read * Hk * block + 2 * T * Hq * D * 2, "flops": 4 * D * Hq * pairs}


# ---------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------
def _quantized(x):
    """Blocks (..., BT tokens' values) -> (e4m3 codes, scales as e8m0)."""
    amax = x.abs().amax(-1).amax(-1)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-30) / FP8_MAX)).clamp(min=MIN_EXP)
    q = (x / torch.exp2(e)[..., None, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    new, past = _lengths(c)
    B, Hq, Hk, D, page = c["seqs"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    T, P = sum(new), -(-max(n + p for n, p in zip(new, past)) // page)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = {"op": c["op"], "page": page, "window": c["window"], "scale": D ** -0.5, "T": T,
         "heads": (Hq, Hk, D), "max_new": max(new)}
    # pages of the sequences, anywhere in a pool with some pages to spare
    used = [-(-(n + p) // page) for n, p in zip(new, past)]
    pool = sum(used) + 3
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32).cpu()
    table = torch.zeros(B, P, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    s["table"] = table.to(DEV)
    s["lengths"] = torch.tensor([n + p for n, p in zip(new, past)], dtype=torch.int32).to(DEV)
    ends = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    s["starts"] = ends.to(DEV)
    s["uniform"] = min(new) == max(new)  # the same number of new tokens a sequence
    # what the cache holds: keys with a few wide channels, values around 1
    width = 1.0 + 7.0 * (torch.rand(Hk, 1, D, generator=g, device=DEV) > 0.97)
    k = normal(pool, Hk, page, D) * width
    v = normal(pool, Hk, page // BT, D, BT)
    s["k_scales"] = s["v_scales"] = None
    if c["kv"] == "fp8":
        k, ks = _quantized(k.view(pool, Hk, page // BT, BT, D))
        v, vs = _quantized(v)
        s["k_pages"], s["v_pages"] = k.reshape(pool, Hk, page, D), v
        s["k_scales"], s["v_scales"] = ks, vs
    else:
        s["k_pages"], s["v_pages"] = k.half(), v.half()
    if c["op"] == "attend":
        # queries after norm and rotation
        s["q"] = (normal(T, Hq, D) * 1.5).half()
        return s
    # the projections' outputs, side by side as one launch makes them
    qkv = normal(T, (Hq + 2 * Hk) * D).half()
    s["q"], s["k"], s["v"] = qkv.split([Hq * D, Hk * D, Hk * D], dim=1)
    s["qw"] = s["kw"] = None
    if c["norm"]:
        s["qw"] = (0.5 + torch.rand(D, generator=g, device=DEV)).half()
        s["kw"] = (0.5 + torch.rand(D, generator=g, device=DEV)).half()
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)]).double().to(DEV)
    ang = pos[:, None] * THETA ** (-torch.arange(0, D, 2, device=DEV).double() / D)
    s["cos"], s["sin"] = (f(torch.cat([ang, ang], 1)).half() for f in (torch.cos, torch.sin))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return _plain_append(s) if s["op"] == "append" else _plain_attend(s)


def _run_own(s):
    from glorcq_amd import kernels

    starts = None if s["uniform"] else s["starts"]
    if s["op"] == "append":
        Hq, Hk, D = s["heads"]
        q = kernels.paged_append(
            s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], starts=starts,
            k_scales=s["k_scales"], v_scales=s["v_scales"], cos=s["cos"], sin=s["sin"], q=s["q"],
            q_norm_w=s["qw"], k_norm_w=s["kw"], eps=EPS)
        return {"q": q, **_cache(s)}
    return kernels.paged_attention(
        s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["scale"], starts=starts,
        k_scales=s["k_scales"], v_scales=s["v_scales"], window=s["window"])


def _cache(s):
    return {k: s[k] for k in ("k_pages", "v_pages", "k_scales", "v_scales") if s[k] is not None}


def _tokens(s):
    """Of each new token: its sequence, its place among the sequence's new
    ones, its position."""
    t = torch.arange(s["T"], device=DEV)
    starts = s["starts"].long()
    b = torch.searchsorted(starts, t, right=True) - 1
    i = t - starts[b]
    new = starts[1:] - starts[:-1]
    return b, i, s["lengths"].long()[b] - new[b] + i


def _head_norm_rope(x, w, cos, sin):
    """x (T, H, D) in 64 bits: a value next to a border of the 8-bit codes
    should fall on its side."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return x * cos.double()[:, None] + turned * sin.double()[:, None]


def _plain_append(s):
    Hq, Hk, D = s["heads"]
    T, page = s["T"], s["page"]
    q = _head_norm_rope(s["q"].view(T, Hq, D).double(), s["qw"], s["cos"], s["sin"]).half()
    k = _head_norm_rope(s["k"].view(T, Hk, D).double(), s["kw"], s["cos"], s["sin"])
    v = s["v"].view(T, Hk, D).double()
    b, i, pos = _tokens(s)
    at = s["table"].long()[b, pos // page]
    blk, j = pos % page // BT, pos % BT
    if s["k_scales"] is None:
        s["k_pages"][at, :, pos % page] = k.half()
        s["v_pages"][at, :, blk, :, j] = v.half()
        return {"q": q, **_cache(s)}
    # the blocks that get new tokens: up to `n` of each sequence
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    first = s["lengths"].long() - new                       # position of the first new token
    n = (s["max_new"] + BT - 2) // BT + 1
    nb = first[:, None] // BT + torch.arange(n, device=DEV)  # (B, n): blocks of the sequence
    touched = (nb * BT < s["lengths"][:, None]) & (new[:, None] > 0)
    row = torch.where(touched, nb, 0)
    pg = s["table"].long().gather(1, row * BT // page)[touched]
    bi = (row * BT % page // BT)[touched]                    # (blocks,)
    pos_in = nb[touched][:, None] * BT + torch.arange(BT, device=DEV)
    seq = torch.arange(len(new), device=DEV)[:, None].expand_as(nb)[touched]
    lo, hi = first[seq][:, None], s["lengths"].long()[seq][:, None]
    fresh = (pos_in >= lo) & (pos_in < hi)                   # (blocks, BT)
    kept = (pos_in < lo).view(-1, 1, BT, 1)
    src = torch.where(fresh, s["starts"].long()[seq][:, None] + pos_in - lo, 0)

    def put(x, old, old_exp):
        """x (blocks, Hk, BT, D) new values, old codes of the same shape ->
        codes and exponents of the blocks."""
        x = torch.where(fresh[:, None, :, None], x, 0.0)
        fine = torch.isfinite(x)
        m, e = torch.frexp(torch.where(fine, x, 0.0).abs().amax((-1, -2)))
        # the smallest e with amax <= 448 2^e; 448 = 0.875 2^9
        e = torch.where(m == 0, MIN_EXP, e - 9 + (m > 0.875).int()).clamp(min=MIN_EXP)
        any_kept = kept.any(2).view(-1, 1)
        old_e = torch.where(any_kept, old_exp, MIN_EXP)
        e = torch.maximum(e, old_e)
        codes = torch.where(fine, x * torch.exp2(-e.double())[..., None, None], float("nan"))
        back = old.double() * torch.exp2((old_e - e).double())[..., None, None]
        # what lies behind the last token is zero
        codes = torch.where(kept, back, codes).float().to(torch.float8_e4m3fn)
        return codes, (e + 127).to(torch.uint8)

    def exps(x):
        return x.view(torch.uint8)[pg, :, bi].int() - 127

    kp = s["k_pages"].view(-1, Hk, page // BT, BT, D).view(torch.uint8)
    vp = s["v_pages"].view(torch.uint8)
    ck, ek = put(k[src].transpose(1, 2), kp[pg, :, bi].view(torch.float8_e4m3fn),
                 exps(s["k_scales"]))
    cv, ev = put(v[src].transpose(1, 2), vp[pg, :, bi].view(torch.float8_e4m3fn).mT,
                 exps(s["v_scales"]))
    kp[pg, :, bi] = ck.view(torch.uint8)
    vp[pg, :, bi] = cv.view(torch.uint8).mT
    s["k_scales"].view(torch.uint8)[pg, :, bi] = ek
    s["v_scales"].view(torch.uint8)[pg, :, bi] = ev
    return {"q": q, **_cache(s)}


def _plain_attend(s):
    Hq, Hk, D = s["heads"]
    B, N, page = len(s["lengths"]), s["max_new"], s["page"]
    pages = s["table"].long()
    k, v = s["k_pages"][pages].float(), s["v_pages"][pages].float()
    if s["k_scales"] is not None:
        k = k.view(B, -1, Hk, page // BT, BT, D) * s["k_scales"][pages].float()[..., None, None]
        v = v * s["v_scales"][pages].float()[..., None, None]
    k = k.reshape(B, -1, Hk, page, D).transpose(1, 2).reshape(B, Hk, -1, D)
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(B, Hk, -1, D)
    L = k.shape[2]
    # queries as (sequence, new token), the missing ones of token 0
    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(N, device=DEV)
    there = i < new[:, None]
    q = s["q"][torch.where(there, starts[:-1, None] + i, 0)].float()  # (B, N, Hq, D)
    q = q.view(B, N, Hk, Hq // Hk, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D)
    at = (lengths - new)[:, None] + i                                # (B, N)
    p = torch.arange(L, device=DEV)
    sees = p <= at[..., None]
    if s["window"]:
        sees &= p > at[..., None] - s["window"]
    t = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    t = t.view(B, Hk, N, Hq // Hk, L).masked_fill_(~sees[:, None, :, None], -math.inf)
    t = torch.exp(t - t.amax(-1, keepdim=True))
    total = t.sum(-1, keepdim=True)
    # a position that nothing of the sequence sees counts for nothing, whatever is in it
    v = torch.where((p < lengths[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(t.view(B, Hk, -1, L), v).view(B, Hk, N, Hq // Hk, D) / total
    b, i, _ = _tokens(s)
    return o.permute(0, 2, 1, 3, 4).reshape(B, N, Hq * D)[b, i].half()


# ---------------------------------------------------------------------------
# the operators' definition in 64 bits, a sequence at a time
# ---------------------------------------------------------------------------
def _e4m3(x):
    """The e4m3 value nearest to x (ties to even), |x| <= 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(c, seed):
    s = prepare(c, seed)
    new, past = _lengths(c)
    Hq, Hk, D = s["heads"]
    page, rep = c["page"], Hq // Hk
    fp8 = c["kv"] == "fp8"
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    ks = s["k_scales"].double() if fp8 else None
    vs = s["v_scales"].double() if fp8 else None
    lo, out = 0, []
    if c["op"] == "attend":
        for b, (n, m) in enumerate(zip(new, past)):
            pg = s["table"][b, :-(-(n + m) // page)].long()
            k, v = kp[pg].unflatten(2, (page // BT, BT)), vp[pg].mT  # (pages, Hk, blocks, BT, D)
            if fp8:
                k, v = k * ks[pg][..., None, None], v * vs[pg][..., None, None]
            k, v = (x.transpose(0, 1).reshape(Hk, -1, D)[:, :n + m] for x in (k, v))
            q = s["q"][lo:lo + n].double().view(n, Hk, rep, D)
            at = torch.arange(m, m + n, device=DEV)
            p = torch.arange(n + m, device=DEV)
            hidden = p > at[:, None]
            if c["window"]:
                hidden |= p <= at[:, None] - c["window"]
            rows = torch.empty(n, Hk, rep, D, dtype=torch.float64, device=DEV)
            for h in range(Hk):
                t = torch.einsum("nrd,pd->nrp", q[:, h], k[h]) * D ** -0.5
                t = torch.softmax(t.masked_fill(hidden[:, None], -math.inf), -1)
                rows[:, h] = torch.einsum("nrp,pd->nrd", t, v[h])
            out.append(rows.view(n, Hq * D))
            lo += n
        return torch.cat(out)
    T = sum(new)
    half = D // 2

    def turned(x, w):
        x = x.double().reshape(T, -1, D)
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
        a, b = x[..., :half], x[..., half:]
        cos, sin = s["cos"].double()[:, None], s["sin"].double()[:, None]
        return torch.cat([a * cos[..., :half] - b * sin[..., :half],
                          b * cos[..., half:] + a * sin[..., half:]], -1)

    q, k = turned(s["q"], s["qw"]), turned(s["k"], s["kw"])
    v = s["v"].double().reshape(T, Hk, D)
    kp = kp.unflatten(2, (page // BT, BT))  # (pages, Hk, blocks, BT, D)
    for b, (n, m) in enumerate(zip(new, past)):
        first, last = m // BT, (m + n - 1) // BT
        blocks = torch.arange(first, last + 1, device=DEV)
        pg, bi = s["table"][b].long()[blocks * BT // page], blocks % (page // BT)
        keep = m - first * BT  # tokens of the first block that were there
        for x, pages, scales, mt in ((k, kp, ks, False), (v, vp, vs, True)):
            old = pages[pg, :, bi]
            old = old.mT if mt else old.clone()  # (blocks, Hk, BT, D)
            if not fp8:
                flat = old.transpose(1, 2).reshape(-1, Hk, D)
                flat = torch.cat([flat[:keep], x[lo:lo + n].half().double(), flat[keep + n:]])
                res = flat.view(-1, BT, Hk, D).transpose(1, 2)
            else:
                pad = torch.zeros((last + 1) * BT - m - n, Hk, D, dtype=torch.float64, device=DEV)
                front = torch.zeros(keep, Hk, D, dtype=torch.float64, device=DEV)
                vals = torch.cat([front, x[lo:lo + n], pad]).view(-1, BT, Hk, D).transpose(1, 2)
                need = vals.abs().amax((-1, -2)) / FP8_MAX
                e = torch.ceil(torch.log2(need)).clamp(min=MIN_EXP)
                e = torch.where(torch.exp2(e) < need, e + 1, e)
                e = torch.where((torch.exp2(e - 1) >= need) & (e > MIN_EXP), e - 1, e)
                if keep:
                    e[0] = torch.maximum(e[0], torch.log2(scales[pg[0], :, bi[0]]))
                res = _e4m3(vals / torch.exp2(e)[..., None, None])
                if keep:
                    f = torch.exp2(torch.log2(scales[pg[0], :, bi[0]]) - e[0])[:, None, None]
                    res[0, :, :keep] = _e4m3(old[0, :, :keep] * f)
                scales[pg, :, bi] = torch.exp2(e)
            pages[pg, :, bi] = res.mT if mt else res
        lo += n
    res = {"q": q.reshape(T, Hq, D), "k_pages": kp.flatten(2, 3), "v_pages": vp}
    if fp8:
        res |= {"k_scales": ks, "v_scales": vs}
    return res
