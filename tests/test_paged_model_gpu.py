"""The Qwen3-MoE-shaped model (2 layers at full width, glorcq_amd.synthetic_model)
over a paged cache: prompts of different lengths in one forward, decode steps
under a captured graph.

Checks: an fp16 paged cache gives the logits of the same model over the static
cache, each prompt alone, within 2 % of their range (the bar of the model tests:
the attention's sums and roundings differ), prompt and teacher-forced decode
steps both; graph replays give the bits of eager steps, fp16 and 8 bits; pages
are given back and used again."""

import pytest
import torch

import paged_ref as R
from glorcq_amd import kernels
from glorcq_amd.graph_wrapper import _static_cache
from glorcq_amd.paged_cache import GLoRCQPagedWrapper, PagedKVCache, PagedStep, paged_forward
from glorcq_amd.synthetic_model import build_qwen3_moe, qwen3_moe_config

pytestmark = pytest.mark.gpu

VOCAB = 1024
_CACHE = {}


def _model(dev):
    if "m" not in _CACHE:
        cfg = qwen3_moe_config(num_hidden_layers=2, vocab_size=VOCAB, max_position_embeddings=512)
        _CACHE["m"] = build_qwen3_moe(cfg, dev, seed=0)[0]
    return _CACHE["m"]


def _prompts(lens, dev, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, VOCAB, (n,), generator=g).to(dev) for n in lens]


@torch.no_grad()
def _static_logits(model, prompt, cont, dev):
    """Logits after the prompt and after each forced token, static cache."""
    cache = _static_cache(model, 1, 256, dev, torch.float16)
    out = [model(input_ids=prompt[None], cache_position=torch.arange(len(prompt), device=dev),
                 past_key_values=cache, use_cache=True, return_dict=False)[0][0, -1]]
    for i, t in enumerate(cont):
        pos = torch.tensor([len(prompt) + i], device=dev)
        out.append(model(input_ids=t.view(1, 1), cache_position=pos, past_key_values=cache,
                         use_cache=True, return_dict=False)[0][0, -1])
    return torch.stack(out).float()


@pytest.mark.parametrize("lens", [(5, 33, 70), (1,), (130, 2)])
@torch.no_grad()
def test_fp16_pages_match_static_cache(gpu, lens):
    model = _model(gpu)
    prompts = _prompts(lens, gpu)
    g = torch.Generator().manual_seed(8)
    cont = torch.randint(0, VOCAB, (4, len(lens)), generator=g).to(gpu)
    w = GLoRCQPagedWrapper(model, max_batch_size=len(lens), max_seq_len=160, page_size=32,
                           cache_dtype=torch.float16)
    w.capture_graph()
    got = [w.prefill(prompts).clone()]
    for t in cont:
        got.append(w.replay(t).clone())
    torch.cuda.synchronize()
    got = torch.stack(got).float()  # (steps, batch, vocab)
    for b, p in enumerate(prompts):
        ref = _static_logits(model, p, cont[:, b], gpu)
        err = float((got[:, b] - ref).abs().max())
        assert err <= 0.02 * float(ref.abs().max()), (b, err)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float16])
@torch.no_grad()
def test_replays_match_eager_steps(gpu, dtype):
    model = _model(gpu)
    prompts = _prompts((40, 7, 64), gpu)
    w = GLoRCQPagedWrapper(model, max_batch_size=3, max_seq_len=80, page_size=16,
                           cache_dtype=dtype)
    out, secs = w.generate(prompts, max_new_tokens=12)
    assert secs > 0 and [len(o) for o in out] == [52, 19, 76]
    token = torch.argmax(w.prefill(prompts), -1)
    toks = [token]
    for _ in range(11):
        pos = torch.tensor([w.cache.length(b) for b in range(3)], device=gpu)
        w.cache.extend(1)
        logits = paged_forward(model, token, pos, PagedStep(w.cache))
        assert bool(torch.isfinite(logits).all())
        token = torch.argmax(logits, -1)
        toks.append(token)
    torch.cuda.synchronize()
    for b, p in enumerate(prompts):
        assert torch.equal(out[b][:len(p)], p)
        assert torch.equal(out[b][len(p):], torch.stack(toks, 1)[b])


@torch.no_grad()
def test_continued_prompts_and_room(gpu):
    """A prompt in two parts beside a decode token in one step; a wrapper stops
    where its longest sequence is full; a released sequence's pages serve
    another."""
    model = _model(gpu)
    a, b = _prompts((90, 20), gpu)
    w = GLoRCQPagedWrapper(model, max_batch_size=2, max_seq_len=96, page_size=32,
                           cache_dtype=torch.float16)
    cache = w.cache

    def step(parts):
        lens = [len(p) for p in parts]
        past = [cache.length(i) for i in range(2)]
        cache.extend(lens)
        st = torch.tensor([0] + lens).cumsum(0)
        pos = torch.cat([torch.arange(p, p + n) for p, n in zip(past, lens)])
        return paged_forward(model, torch.cat(parts), pos.to(gpu),
                             PagedStep(cache, st.to(torch.int32).to(gpu)),
                             last=(st[1:] - 1).to(gpu))

    step([a[:50], b[:19]])
    got = step([a[50:], b[19:]]).float()  # 40 tokens and 1
    for i, p in enumerate((a, b)):
        ref = _static_logits(model, p, [], gpu)[0]
        assert float((got[i] - ref).abs().max()) <= 0.02 * float(ref.abs().max())
    cache.release(0)
    again = step([b, b[:0]]).float()
    assert float((again[0] - got[1]).abs().max()) <= 0.02 * float(got[1].abs().max())
    out, _ = w.generate([a, b], max_new_tokens=100)
    assert [len(o) for o in out] == [97, 27]
    with pytest.raises(RuntimeError, match="max_seq_len"):
        w.replay(torch.zeros(2, dtype=torch.long, device=gpu))


@pytest.mark.parametrize("batch", [3, 4])
@torch.no_grad()
def test_one_kv_head(gpu, batch):
    """A model of 4 query heads and one KV head: the batched projections' items
    are heads, as many of them as sequences for a batch of 4."""
    cfg = qwen3_moe_config(num_hidden_layers=1, vocab_size=VOCAB, max_position_embeddings=512)
    cfg.num_attention_heads, cfg.num_key_value_heads = 4, 1
    model = build_qwen3_moe(cfg, gpu, seed=1)[0]
    prompts = _prompts([9, 40, 3, 17][:batch], gpu)
    g = torch.Generator().manual_seed(8)
    cont = torch.randint(0, VOCAB, (3, batch), generator=g).to(gpu)
    w = GLoRCQPagedWrapper(model, max_batch_size=batch, max_seq_len=64, page_size=16,
                           cache_dtype=torch.float16)
    w.capture_graph()
    got = [w.prefill(prompts).clone()] + [w.replay(t).clone() for t in cont]
    torch.cuda.synchronize()
    got = torch.stack(got).float()
    for b, p in enumerate(prompts):
        ref = _static_logits(model, p, cont[:, b], gpu)
        err = float((got[:, b] - ref).abs().max())
        assert err <= 0.02 * float(ref.abs().max()), (b, err)


@torch.no_grad()
def test_capture_before_any_step(gpu):
    """A step captured before an eager one of its shape: the eager one's
    workspace is zeroed all the same."""
    cache = PagedKVCache(1, 1, 64, 2, 5000, page_size=16, dtype=torch.float16, device=gpu)
    cache.extend(4800)
    kp, vp, _, _ = cache.layers[0]
    g = torch.Generator().manual_seed(4)
    for x in (kp, vp):
        x.copy_(torch.randn(x.shape, generator=g))
    q = torch.randn(2, 4, 64, generator=g).half().to(gpu)
    step = PagedStep(cache)

    def run():
        return kernels.paged_attention(q, kp, vp, step.page_table, step.lengths, 0.1,
                                       workspace=step.workspace(q))

    want = kernels.paged_attention(q, kp, vp, step.page_table, step.lengths, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    for _ in range(2):
        assert torch.equal(run(), want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_wrapper_refusals(gpu):
    w = GLoRCQPagedWrapper(_model(gpu), max_batch_size=2, max_seq_len=32, page_size=16)
    a, b = _prompts((4, 5), gpu)
    for what, call in (
            ("no captured step", lambda: w.replay(a[:2])),
            ("2 1-D prompts", lambda: w.prefill([a])),
            ("2 1-D prompts", lambda: w.prefill([a, b[:0]])),
            ("2 1-D prompts", lambda: w.prefill([a[None], b])),
            ("max_seq_len", lambda: w.prefill([a, b.repeat(10)]))):
        with pytest.raises(RuntimeError, match=what):
            call()
    w.capture_graph()
    with pytest.raises(RuntimeError, match="input_ids must be"):
        w.replay(a[:1])


class _Rounded:
    """paged_append for fp16 pages that then hold what 8-bit ones would: each
    block's values as e4m3 codes of its scale, worked out on the CPU in 64 bits
    (paged_ref.Model)."""

    def __init__(self, append):
        self.append, self.layers = append, {}

    def __call__(self, k, v, k_pages, v_pages, page_table, lengths, starts=None, **kw):
        out = self.append(k, v, k_pages, v_pages, page_table, lengths, starts=starts, **kw)
        _, Hk, page, D = k_pages.shape
        B, table = len(lengths), page_table.cpu().long()
        m = self.layers.setdefault(k_pages.data_ptr(), R.Model(B, Hk, D, page, True, 0, None))
        st = [i * len(k) // B for i in range(B + 1)] if starts is None else starts.tolist()
        kp, vp = k_pages.cpu(), v_pages.cpu()
        for b, L in enumerate(lengths.tolist()):
            pos = torch.arange(L)
            pg, at = table[b, pos // page], pos % page
            fresh = pos >= L - (st[b + 1] - st[b])
            m.put("k", b, kp[pg, :, at][fresh].double())
            m.put("v", b, vp[pg, :, at // 16, :, at % 16][fresh].double())
            kp[pg, :, at] = m.k[b].half()
            vp[pg, :, at // 16, :, at % 16] = m.v[b].half()
        k_pages.copy_(kp)
        v_pages.copy_(vp)
        return out


@torch.no_grad()
def test_e4m3_pages_cost_their_rounding_alone(gpu, monkeypatch):
    """The default cache, prompts and captured decode steps: the logits of a run
    over fp16 pages whose values are rounded as 8-bit ones are, within the other
    tests' 2 % of their range; and in the first layer, whose inputs are the same
    bits, codes that are the same or neighbours (a value of the fp16 pages has
    been rounded before)."""
    model = _model(gpu)
    lens = (40, 7, 64)
    prompts = _prompts(lens, gpu)
    g = torch.Generator().manual_seed(11)
    cont = torch.randint(0, VOCAB, (12, 3), generator=g).to(gpu)
    a = GLoRCQPagedWrapper(model, max_batch_size=3, max_seq_len=80, page_size=32)
    assert a.cache.layers[0][0].dtype == torch.float8_e4m3fn
    a.capture_graph()
    got = [a.prefill(prompts).clone()] + [a.replay(t).clone() for t in cont]
    b = GLoRCQPagedWrapper(model, max_batch_size=3, max_seq_len=80, page_size=32,
                           cache_dtype=torch.float16)
    monkeypatch.setattr(kernels, "paged_append", _Rounded(kernels.paged_append))
    want = [b.prefill(prompts)]
    for t in cont:
        pos = torch.tensor([b.cache.length(i) for i in range(3)], device=gpu)
        b.cache.extend(1)
        want.append(paged_forward(model, t, pos, PagedStep(b.cache)))
    torch.cuda.synchronize()
    got, want = torch.stack(got).float(), torch.stack(want).float()
    err = (got - want).abs().amax((0, 2))
    assert (err <= 0.02 * want.abs().amax((0, 2))).all(), err
    # 16-token blocks of the sequences' tokens (both caches gave out the same pages)
    assert torch.equal(a.cache.page_table, b.cache.page_table)
    (kq, vq, ks, vs), (kf, vf) = a.cache.layers[0], b.cache.layers[0][:2]
    table = a.cache.page_table.cpu().long()
    for q, s, f, rows in ((kq, ks, kf, True), (vq, vs, vf, False)):
        q, s, f = q.cpu().double(), s.cpu().view(torch.uint8).double() - 127, f.cpu().double()
        q, f = (x.unflatten(2, (2, 16)) if rows else x.mT for x in (q, f))  # (.., blocks, 16, D)
        step = torch.exp2(s)[..., None, None]
        q = q * step
        # one step: 2^-3 of the larger value, 2^-9 of the scale where codes are subnormal
        # (a scale may differ too, where the largest value was rounded over its border)
        near = (q - f).abs() <= 2.0 ** -3 * torch.maximum(q.abs(), f.abs()) + 2.0 ** -8 * step
        same = q == f
        n = differ = 0
        for i, L in enumerate(lens):
            for p in range(L + len(cont)):
                at = (table[i, p // 32], slice(None), p % 32 // 16, p % 16)
                assert near[at].all()
                n, differ = n + same[at].numel(), differ + int((~same[at]).sum())
        # a value is next to a border of two codes (4 bits) by an fp16 rounding (11
        # bits) once in 2^7
        assert differ <= n * 2.0 ** -6, (differ, n)
