"""Operators of generation over the paged key/value cache as cases that can be
timed (the cache itself: perf/operators.py).

sinks    kernels.paged_attention with a window and sinks: the token at position
         p attends to the first S positions and to (p - W, p]; pages that lie
         between the two are not in the cache any more
copy     kernels.paged_copy: pages of all layers of a cache to other pages of
         it (a fork that is about to write the page it shares, up to its last
         token) or to another cache's (a pool moved to one of another size)
beam     kernels.beam_select: the best continuations of each prompt over its
         beams and the vocabulary, by their log-probabilities

32 query and 4 KV heads of 128, 48 layers and a vocabulary of 151936 are the
Qwen3-MoE-shaped model's, 24 layers and 16 and 16 heads those of
Qwen1.5-MoE-A2.7B; other sizes are generic.

With `own` false `run` computes the operators with elementary torch
operations; `exact` restates them in 64 bits.

Layouts (BT = 16 tokens a block): k pages ([layers,] pages, Hk, page, D), v
pages ([layers,] pages, Hk, page / BT, D, BT), scales ([layers,] pages, Hk,
page / BT), page table (sequences, pages a sequence; -1: no page), lengths
(sequences) with the new tokens among them.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
BT = 16          # tokens of a scale block
FP8_MAX = 448.0  # largest e4m3 value


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _sinks(name, seqs, new, past, window, sinks, heads=(32, 4), dim=128, page=64, kv="fp8",
           ones=0, lens=1):
    """new, past: (fewest, most) tokens a sequence brings and has behind it.
    ones: sequences, the first ones, that bring one token."""
    return {"name": name, "op": "sinks", "seqs": seqs, "ones": ones, "new_lo": new[0],
            "new_hi": new[1], "past_lo": past[0], "past_hi": past[1], "window": window,
            "sinks": sinks, "q_heads": heads[0], "kv_heads": heads[1], "dim": dim, "page": page,
            "kv": kv, "lens": lens}


def _copy(name, layers, pairs, parents, tokens=None, moved=False, heads=4, dim=128, page=64,
          kv="fp8", lens=1):
    """pairs: pages copied, from `parents` pages.  tokens: (fewest, most) of a
    page, None for whole ones.  moved: to another pool."""
    return {"name": name, "op": "copy", "layers": layers, "pairs": pairs, "parents": parents,
            "whole": tokens is None, "tokens_lo": tokens[0] if tokens else page,
            "tokens_hi": tokens[1] if tokens else page, "moved": moved, "kv_heads": heads,
            "dim": dim, "page": page, "kv": kv, "lens": lens}


def _beam(name, prompts, beams, vocab, num, dtype="fp16", pad=0, masked=False):
    """num: continuations kept of each prompt.  pad: columns behind the
    vocabulary's.  masked: most of the vocabulary is not allowed."""
    return {"name": name, "op": "beam", "prompts": prompts, "beams": beams, "vocab": vocab,
            "num": num, "dtype": dtype, "pad": pad, "masked": masked}


def listed():
    return [
        # one token of a long conversation that keeps a short window: latency
        _sinks("sink_one", 1, (1, 1), (5000, 5000), 1020, 4),
        # a decode step of a serving batch, some sequences not past their window
        _sinks("sink_batch", 64, (1, 1), (3, 20000), 4096, 4),
        # far positions behind a wide window, many sinks, fp16 values
        _sinks("sink_far", 5, (1, 1), (150000, 300000), 16000, 100, heads=(16, 2), page=128,
               kv="fp16"),
        # a prompt longer than its window
        _sinks("sink_prompt", 1, (5000, 5000), (0, 0), 1024, 4),
        # decode tokens and chunks of prompts in one batch, 64-wide heads, as
        # many KV heads as query heads, odd window and sinks
        _sinks("sink_mixed", 22, (90, 700), (0, 6000), 1001, 37, heads=(16, 16), dim=64, page=32,
               ones=14),
        # one prompt's beams part: three forks copy the page that they share
        _copy("copy_fork", 48, 3, 1, (21, 21)),
        # a beam step of a batch of prompts, 7 of 8 beams of each from another one
        _copy("copy_beams", 48, 56, 17, (1, 63)),
        # a cache moved to a smaller pool
        _copy("copy_pool", 24, 97, 97, moved=True, heads=16, page=32, kv="fp16"),
        # a beam step of one prompt: latency
        _beam("beam_one", 1, 4, 151936, 8),
        # a beam step of a batch of prompts
        _beam("beam_batch", 16, 8, 151936, 16),
        # first step: one beam a prompt, fp32 logits, rows of an odd width
        _beam("beam_first", 32, 1, 50001, 10, "fp32"),
        # most tokens masked out by a grammar, rows of a padded matrix
        _beam("beam_masked", 3, 5, 32000, 10, "bf16", pad=77, masked=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = ((32, 4), (16, 16), (32, 8), (16, 2), (12, 4), (28, 4), (8, 1), (64, 4))
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def draw(rng):
    op = rng.choice(("sinks", "sinks", "copy", "beam"))
    kv = rng.choice(("fp8", "fp8", "fp16"))
    dim = rng.choice((128, 128, 64))
    page = rng.choice((16, 32, 64, 128))
    if op == "sinks":
        heads = rng.choice(HEADS)
        sinks, lens = _log_int(rng, 1, 200), rng.randrange(1 << 20)
        if rng.random() < 0.5:  # prompts, or decode steps
            seqs = _log_int(rng, 1, 12)
            hi = _log_int(rng, 2, 5000 // seqs)
            lo = rng.choice((1, hi, max(1, hi // 3)))
            past_hi = rng.choice((0, _log_int(rng, 1, 12000 // seqs)))
            ones = rng.choice((0, seqs // 2))
        else:
            seqs, ones = _log_int(rng, 1, 96), 0
            lo, hi = 1, rng.choice((1, 1, 1, 2, 5))
            past_hi = _log_int(rng, 1, min(100000, 400000 // seqs))
        past_lo = rng.choice((0, past_hi, past_hi // 4))
        window = _log_int(rng, 16, min(16000, max(50, past_hi + hi)))
        c = _sinks("", seqs, (lo, hi), (past_lo, past_hi), window, sinks, heads, dim, page, kv,
                   ones, lens)
    elif op == "copy":
        pairs = _log_int(rng, 1, 200)
        tokens = rng.choice((None, (1, page), (1, page)))
        c = _copy("", _log_int(rng, 1, 64), pairs, rng.choice((pairs, max(1, pairs // 5))), tokens,
                  rng.random() < 0.4, rng.choice(HEADS)[1], dim, page, kv, rng.randrange(1 << 20))
    else:
        prompts, beams = _log_int(rng, 1, 32), _log_int(rng, 1, 16)
        c = _beam("", prompts, beams, _log_int(rng, 500, 160000),
                  rng.choice((beams, 2 * beams, 2 * beams)), rng.choice(sorted(DTYPES)),
                  rng.choice((0, 0, _log_int(rng, 1, 100))), rng.random() < 0.25)
    del c["name"]
    # to the work of the largest listed ones
    most = [work(x) for x in listed() if x["op"] == op]
    while any(work(c)[k] > max(m[k] for m in most) for k in ("bytes", "flops")):
        at = {"sinks": "past_hi", "copy": "pairs", "beam": "prompts"}[op]
        if op == "sinks" and (c["new_hi"] > c["past_hi"] or c["past_hi"] > 2 * c["window"]):
            at = "new_hi" if c["new_hi"] > c["past_hi"] else "window"
        elif op == "beam" and c["prompts"] == 1:
            at = "vocab"
        c[at] = max(1, c[at] * 2 // 3)
        for k in ("new", "past") if op == "sinks" else ():
            c[k + "_lo"] = min(c[k + "_lo"], c[k + "_hi"])
        if op == "copy":
            c["parents"] = min(c["parents"], c["pairs"])
    return c


def _lengths(c):
    """(new, past): tokens each sequence brings and has behind it."""
    r = random.Random(c["lens"])
    new = [r.randint(c["new_lo"], c["new_hi"]) if b >= c["ones"] else 1 for b in range(c["seqs"])]
    past = [r.randint(c["past_lo"], c["past_hi"]) for _ in range(c["seqs"])]
    return new, past


def _copied(c):
    """Tokens of each copied page."""
    r = random.Random(c["lens"])
    return [r.randint(c["tokens_lo"], c["tokens_hi"]) for _ in range(c["pairs"])]


def _block_bytes(c):
    """k and v of a token and KV head, with its share of their scales."""
    return 2 * c["dim"] * (1 if c["kv"] == "fp8" else 2) + (2 / BT if c["kv"] == "fp8" else 0)


def work(c):
    if c["op"] == "beam":
        n = c["prompts"] * c["beams"] * c["vocab"]
        # logits and scores read, scores, parents and tokens written; of each
        # logit a comparison, an exponential and a sum
        return {"bytes": n * DTYPES[c["dtype"]].itemsize
                + c["prompts"] * (4 * c["beams"] + 20 * c["num"]), "flops": 4 * n}
    if c["op"] == "copy":
        blocks = sum(-(-n // BT) for n in _copied(c))
        return {"bytes": 2 * blocks * BT * c["layers"] * c["kv_heads"] * _block_bytes(c), "flops": 0}
    new, past = _lengths(c)
    w, s = c["window"], c["sinks"]
    pairs = read = 0
    for n, p in zip(new, past):
        # the token at position i sees min(i + 1, w) positions of its window and
        # what of the sinks lies before it
        pairs += sum(min(i + 1, w) + min(s, max(0, i + 1 - w)) for i in range(p, p + n))
        lo = max(0, p + 1 - w)
        read += p + n - lo + min(s, lo)
    T, Hq, Hk, D = sum(new), c["q_heads"], c["kv_heads"], c["dim"]
    return {"bytes": read * Hk * _block_bytes(c) + 2 * T * Hq * D * 2, "flops": 4 * D * Hq * pairs}


# ---------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------
def _quantized(x):
    """Blocks (..., BT tokens' values) -> (e4m3 codes, scales as e8m0)."""
    amax = x.abs().amax(-1).amax(-1)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-30) / FP8_MAX)).clamp(min=-32)
    q = (x / torch.exp2(e)[..., None, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"sinks": _prepare_sinks, "copy": _prepare_copy, "beam": _prepare_beam}[c["op"]](c, g)


def _prepare_sinks(c, g):
    new, past = _lengths(c)
    B, Hq, Hk, D, page = c["seqs"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    T, P = sum(new), -(-max(n + p for n, p in zip(new, past)) // page)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    # the pages that a sequence still has, anywhere in a pool with some to spare
    have = []
    for n, p in zip(new, past):
        lo = max(0, p + 1 - c["window"]) // page
        first = min(-(-c["sinks"] // page), lo)
        have.append(list(range(first)) + list(range(lo, -(-(n + p) // page))))
    pool = sum(len(h) for h in have) + 3
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32).cpu()
    table = torch.full((B, P), -1, dtype=torch.int32)
    at = 0
    for b, h in enumerate(have):
        table[b, h] = order[at:at + len(h)]
        at += len(h)
    s = {"op": "sinks", "page": page, "window": c["window"], "sinks": c["sinks"],
         "scale": D ** -0.5, "T": T, "heads": (Hq, Hk, D), "max_new": max(new),
         "most": max(n + p - max(0, p + 1 - c["window"]) for n, p in zip(new, past)),
         "uniform": min(new) == max(new), "table": table.to(DEV),
         "lengths": torch.tensor([n + p for n, p in zip(new, past)], dtype=torch.int32).to(DEV),
         "starts": torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEV)}
    # keys with a few wide channels, values around 1, queries after norm and rotation
    width = 1.0 + 7.0 * (torch.rand(Hk, 1, D, generator=g, device=DEV) > 0.97)
    k = normal(pool, Hk, page, D) * width
    v = normal(pool, Hk, page // BT, D, BT)
    s["k_scales"] = s["v_scales"] = None
    if c["kv"] == "fp8":
        k, s["k_scales"] = _quantized(k.view(pool, Hk, page // BT, BT, D))
        s["v_pages"], s["v_scales"] = _quantized(v)
        s["k_pages"] = k.reshape(pool, Hk, page, D)
    else:
        s["k_pages"], s["v_pages"] = k.half(), v.half()
    s["q"] = (normal(T, Hq, D) * 1.5).half()
    return s


def _prepare_copy(c, g):
    L, Hk, D, page, n = c["layers"], c["kv_heads"], c["dim"], c["page"], c["pairs"]

    def pools(pages):
        def values(*shape):
            if c["kv"] == "fp16":
                return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float16)
            code = torch.randint(0, 254, shape, generator=g, device=DEV, dtype=torch.uint8)
            return (code + (code >= 127)).view(torch.float8_e4m3fn)  # (no NaN: 127 and 255)

        k = values(L, pages, Hk, page, D)
        v = values(L, pages, Hk, page // BT, D, BT)
        if c["kv"] == "fp16":
            return k, v, None, None
        ks, vs = (torch.randint(112, 128, (L, pages, Hk, page // BT), generator=g, device=DEV,
                                dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2))
        return k, v, ks, vs

    m = c["parents"]
    pages = m + 3 if c["moved"] else m + n + 3
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    s = {"op": "copy", "pools": pools(pages), "to": None, "page": page,
         "src": [order[i % m] for i in range(n)], "tokens": None if c["whole"] else _copied(c)}
    if c["moved"]:
        s["to"] = pools(n + 2)
        s["dst"] = list(range(n))
    else:
        s["dst"] = order[m:m + n]
    return s


def _prepare_beam(c, g):
    B, K, V = c["prompts"], c["beams"], c["vocab"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    # a prompt's beams say much the same; a few tokens stand out
    x = normal(B, 1, V) * 2 + normal(B, K, V) * 0.7
    x += 9 * (torch.rand(B, 1, V, generator=g, device=DEV) < 30 / V) * normal(B, K, V).abs()
    if c["masked"]:
        x.masked_fill_(torch.rand(B, K, V, generator=g, device=DEV) < 0.97, -math.inf)
    rows = torch.zeros(B * K, V + c["pad"], dtype=DTYPES[c["dtype"]], device=DEV)
    rows[:, :V] = x.view(B * K, V)
    scores = -20 * torch.rand(B, 1, generator=g, device=DEV) - normal(B, K).abs()
    return {"op": "beam", "logits": rows[:, :V], "num": min(c["num"], K * V),
            "scores": scores.sort(1, descending=True).values.contiguous()}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"sinks": _plain_sinks, "copy": _plain_copy, "beam": _plain_beam}[s["op"]](s)


def _run_own(s):
    from glorcq_amd import kernels

    if s["op"] == "sinks":
        return kernels.paged_attention(
            s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["scale"],
            starts=None if s["uniform"] else s["starts"], k_scales=s["k_scales"],
            v_scales=s["v_scales"], window=s["window"], sinks=s["sinks"])
    if s["op"] == "copy":
        k, v, ks, vs = s["pools"]
        kernels.paged_copy(k, v, s["src"], s["dst"], k_scales=ks, v_scales=vs, tokens=s["tokens"],
                           to=s["to"])
        return _pools(s)
    scores, parents, tokens = kernels.beam_select(s["logits"], s["scores"], s["num"])
    return {"scores": scores, "parents": parents, "tokens": tokens}


def _pools(s):
    """The pools that were written, whole."""
    to = s["to"] or s["pools"]
    return {n: t for n, t in zip(("k_pages", "v_pages", "k_scales", "v_scales"), to)
            if t is not None}


def _plain_sinks(s):
    Hq, Hk, D = s["heads"]
    B, N, page, W, S = len(s["lengths"]), s["max_new"], s["page"], s["window"], s["sinks"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    first = lengths - new                                            # of the new tokens
    # the positions that a sequence's tokens see: sinks, then the windows'
    lo = (first + 1 - W).clamp(min=0)[:, None]                       # (B, 1)
    j = torch.arange(S + s["most"], device=DEV)
    p = torch.where(j < S, j, lo + j - S)                            # (B, M)
    there = torch.where(j < S, p < lo, p < lengths[:, None])
    at = torch.where(there, p, lengths[:, None] - 1)
    pg, blk = s["table"].long().gather(1, at // page), at % page // BT
    k = _values(s["k_pages"].view(-1, Hk, page, D), (pg, slice(None), at % page))
    v = _values(s["v_pages"], (pg, slice(None), blk, slice(None), at % BT))
    if s["k_scales"] is not None:
        k *= s["k_scales"].float()[pg, :, blk][..., None]
        v *= s["v_scales"].float()[pg, :, blk][..., None]
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()  # (B, Hk, M, D)
    # queries as (sequence, new token), the missing ones of token 0
    i = torch.arange(N, device=DEV)
    q = s["q"][torch.where(i < new[:, None], starts[:-1, None] + i, 0)].float()
    q = q.view(B, N, Hk, Hq // Hk, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D)
    pos = (first[:, None] + i)[..., None]                            # (B, N, 1)
    p, there = p[:, None], there[:, None]                            # (B, 1, M)
    sees = there & (p <= pos) & ((p < S) | (p > pos - W))
    t = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    t = t.view(B, Hk, N, Hq // Hk, -1).masked_fill_(~sees[:, None, :, None], -math.inf)
    t = torch.exp(t - t.amax(-1, keepdim=True))
    total = t.sum(-1, keepdim=True)
    o = torch.matmul(t.view(B, Hk, N * (Hq // Hk), -1), v).view(B, Hk, N, Hq // Hk, D) / total
    row = torch.arange(s["T"], device=DEV)
    b = torch.searchsorted(starts, row, right=True) - 1
    return o.permute(0, 2, 1, 3, 4).reshape(B, N, Hq * D)[b, row - starts[b]].half()


def _values(pages, at):
    """pages[at] in 32 bits (8-bit types are indexed as bytes)."""
    if pages.dtype == torch.float8_e4m3fn:
        return pages.view(torch.uint8)[at].view(pages.dtype).float()
    return pages[at].float()


def _plain_copy(s):
    src, dst = (torch.tensor(x).to(DEV) for x in (s["src"], s["dst"]))
    to = s["to"] or s["pools"]
    page = s["page"]
    if s["tokens"] is not None:
        blocks = (torch.tensor(s["tokens"]).to(DEV) + BT - 1) // BT
        kept = torch.arange(page // BT, device=DEV) < blocks[:, None]  # (pairs, blocks)
        kept = kept[None, :, None, :, None]
    for x, y in zip(s["pools"], to):
        if x is None:
            continue
        # (layers, pages, heads, blocks, words of a block): values as words of 64
        # bits, scales as bytes
        word = torch.uint8 if x.dim() == 4 else torch.int64
        x, y = (t.view(word).view(*t.shape[:3], page // BT, -1) for t in (x, y))
        y[:, dst] = x[:, src] if s["tokens"] is None else torch.where(kept, x[:, src], y[:, dst])
    return _pools(s)


def _plain_beam(s):
    B, K = s["scores"].shape
    N = s["num"]
    x = s["logits"].double().view(B, K, -1)
    V = x.shape[2]
    m = x.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    c = (s["scores"].double()[..., None] + (x - lse)).view(B, K * V)
    # the N largest; of those equal to the last of them, the lowest places
    last = c.topk(N).values[:, -1:]
    above, equal = c > last, c == last
    take = above | (equal & (equal.cumsum(1) <= N - above.sum(1, keepdim=True)))
    place = torch.arange(K * V, device=DEV)
    place = K * V - torch.where(take, K * V - place, 0).topk(N).values  # ascending
    val, order = c.gather(1, place).sort(dim=1, descending=True, stable=True)
    place = place.gather(1, order)
    return {"scores": val.float(), "parents": place // V, "tokens": place % V}


# ---------------------------------------------------------------------------
# the operators' definition in 64 bits, a sequence or prompt at a time
# ---------------------------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "copy":
        to, res = s["to"] or s["pools"], []
        for x, y in zip(s["pools"], to):
            if x is None:
                continue
            x, y = (t.double().view(*t.shape[:3], c["page"] // BT, -1) for t in (x, y))
            for i, j, n in zip(s["src"], s["dst"], _copied(c)):
                y[:, j, :, :-(-n // BT)] = x[:, i, :, :-(-n // BT)]
            res.append(y)
        return {n: y.view(t.shape) for (n, t), y in zip(_pools(s).items(), res)}
    if c["op"] == "beam":
        B, K, V = c["prompts"], c["beams"], c["vocab"]
        score, parent, token = [], [], []
        for b in range(B):
            logp = torch.log_softmax(s["logits"][b * K:(b + 1) * K].double(), -1)
            v = (logp + s["scores"][b].double()[:, None]).flatten()
            v, i = v.sort(dim=0, descending=True, stable=True)
            score.append(v[:s["num"]])
            parent.append(i[:s["num"]] // V)
            token.append(i[:s["num"]] % V)
        return {"scores": torch.stack(score), "parents": torch.stack(parent),
                "tokens": torch.stack(token)}
    new, past = _lengths(c)
    Hq, Hk, D = s["heads"]
    page, rep = c["page"], Hq // Hk
    out, lo = [], 0
    for b, (n, m) in enumerate(zip(new, past)):
        # the sequence's pages end to end, those that it has not as page 0
        pg = s["table"][b, :-(-(n + m) // page)].long()
        keep = pg.ge(0).nonzero()[:, 0]
        p = (keep[:, None] * page + torch.arange(page, device=DEV)).flatten()
        pg = pg[keep]
        k = s["k_pages"].view(torch.uint8)[pg].view(s["k_pages"].dtype).double()
        v = s["v_pages"].view(torch.uint8)[pg].view(s["v_pages"].dtype).double()
        k, v = k.unflatten(2, (page // BT, BT)), v.mT  # (pages, Hk, blocks, BT, D)
        if c["kv"] == "fp8":
            k = k * s["k_scales"].double()[pg][..., None, None]
            v = v * s["v_scales"].double()[pg][..., None, None]
        k, v = (x.transpose(0, 1).reshape(Hk, -1, D) for x in (k, v))
        q = s["q"][lo:lo + n].double().view(n, Hk, rep, D)
        lo += n
        i = torch.arange(m, m + n, device=DEV)[:, None]
        hidden = (p > i) | ((p <= i - c["window"]) & (p >= c["sinks"]))
        rows = torch.empty(n, Hk, rep, D, dtype=torch.float64, device=DEV)
        for h in range(Hk):
            t = torch.einsum("nrd,pd->nrp", q[:, h], k[h]) * D ** -0.5
            t = torch.softmax(t.masked_fill(hidden[:, None], -math.inf), -1)
            rows[:, h] = torch.einsum("nrp,pd->nrd", t, v[h])
        out.append(rows.view(n, Hq * D))
    return torch.cat(out)
