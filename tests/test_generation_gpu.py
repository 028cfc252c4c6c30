"""Generation over shared pages on the Qwen3-MoE-shaped model (2 layers at full
width): forks, beams, a window with sinks, a pool moved to another size."""

import math

import pytest
import torch

import glorcq_amd.paged_cache as PC
from glorcq_amd.paged_cache import GLoRCQPagedWrapper, PagedStep, paged_forward
from test_paged_forks import _search
from test_paged_model_gpu import VOCAB, _model, _prompts

pytestmark = pytest.mark.gpu

FP8, FP16 = torch.float8_e4m3fn, torch.float16


def _wrapper(model, batch, **kw):
    a = dict(max_seq_len=160, page_size=16, cache_dtype=FP8)
    return GLoRCQPagedWrapper(model, max_batch_size=batch, **{**a, **kw})


def _one(w, seq, prompt):
    """A prompt into sequence `seq` alone; its last logits."""
    lens = [len(prompt) if b == seq else 0 for b in range(w.max_batch_size)]
    w.cache.extend(lens)
    starts = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(w.device)
    return paged_forward(w.model, prompt, torch.arange(len(prompt), device=w.device),
                         PagedStep(w.cache, starts), last=torch.tensor([len(prompt) - 1]).to(w.device))


@pytest.mark.parametrize("dtype", [FP8, FP16])
@torch.no_grad()
def test_forks_are_sequences_of_their_own(gpu, dtype):
    """A prompt forked twice, and the three continued by other tokens (replays
    of one graph): bit for bit what three caches of the prompt give."""
    model = _model(gpu)
    prompt = _prompts((37,), gpu)[0]
    a, b = (_wrapper(model, 3, cache_dtype=dtype) for _ in range(2))
    for w in (a, b):
        w.capture_graph()
    la = _one(a, 0, prompt)
    a.cache.fork(0, 1)
    a.cache.fork(0, 2)
    assert a.cache.pages - a.cache.free_pages == 3
    lb = [_one(b, i, prompt) for i in range(3)]
    assert all(torch.equal(la, x) for x in lb)
    g = torch.Generator().manual_seed(4)
    for i in range(30):
        t = torch.randint(0, VOCAB, (3,), generator=g).to(gpu)
        assert torch.equal(a.replay(t).clone(), b.replay(t)), i
        if i == 12:  # sequences 0 and 1 from 2, the third goes on by itself
            for w in (a, b):
                w.cache.reorder([2, 2, 1])


@torch.no_grad()
def test_one_beam_is_greedy(gpu):
    model = _model(gpu)
    prompts = _prompts((40, 7), gpu)
    w = _wrapper(model, 2)
    greedy, _ = w.generate(prompts, max_new_tokens=20)
    out, scores, secs = w.generate_beams(prompts, 1, max_new_tokens=20)
    assert secs > 0 and len(scores) == 2
    assert all(torch.equal(a, b) for a, b in zip(out, greedy))


@pytest.mark.parametrize("dtype", [FP8, FP16])
@torch.no_grad()
def test_beam_scores_are_their_texts(gpu, dtype):
    """The score of a prompt's best text is the sum of its tokens'
    log-probabilities when the text is forced on the same model, to the
    difference that a prompt's and a step's roundings make (2 % of the logits'
    range a token, the bar of the model tests; and 10 % on top of 8-bit codes)."""
    model = _model(gpu)
    prompts = _prompts((21, 50), gpu)
    K, n = 4, 15
    w = _wrapper(model, 2 * K, cache_dtype=dtype)
    out, scores, _ = w.generate_beams(prompts, K, max_new_tokens=n)
    one = _wrapper(model, 1, cache_dtype=FP16)
    for p, text, score in zip(prompts, out, scores):
        assert torch.equal(text[:len(p)], p) and len(text) == len(p) + n
        one.cache.reset()
        one.cache.extend(len(text))
        st = torch.tensor([0, len(text)], dtype=torch.int32, device=gpu)
        logits = paged_forward(model, text, torch.arange(len(text), device=gpu),
                               PagedStep(one.cache, st))[len(p) - 1:-1].float()
        logp = torch.log_softmax(logits, -1).gather(1, text[len(p):, None]).mean()
        tol = 2 * (0.02 if dtype == FP16 else 0.12) * float(logits.abs().max())
        assert abs(float(logp) - score) <= tol
    # the same beams again, and with another batch in between
    again, s2, _ = w.generate_beams(prompts, K, max_new_tokens=n)
    assert s2 == scores and all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.parametrize("K,eos,penalty,steps", [(1, None, 1.0, 6), (4, 2, 1.0, 20), (3, 7, 0.5, 20),
                                                 (8, None, 1.0, 30)])
@torch.no_grad()
def test_beam_search(gpu, monkeypatch, K, eos, penalty, steps):
    """The whole search over a chain of tokens in the model's place: texts
    exactly, scores to the fp32 rounding of each step's sums."""
    V = 50
    g = torch.Generator().manual_seed(K)
    table = (2 * torch.randn(V, V, generator=g)).half().to(gpu)

    def chain(model, ids, positions, step, last=None):
        x = table[ids]
        return x if last is None else x[last]

    w = _wrapper(_model(gpu), 2 * K)
    monkeypatch.setattr(PC, "paged_forward", chain)
    prompts = [torch.tensor([3, 9], device=gpu), torch.tensor([8], device=gpu)]
    out, scores, _ = w.generate_beams(prompts, K, max_new_tokens=steps, eos_token_id=eos,
                                      length_penalty=penalty)
    logp = torch.log_softmax(table.double().cpu(), -1)
    for p, text, score in zip(prompts, out, scores):
        want, value = _search(logp, logp[int(p[-1])], K, steps, eos, penalty)
        assert tuple(text[len(p):].tolist()) == want
        assert math.isclose(score, value, rel_tol=steps * 2.0 ** -23)


@pytest.mark.parametrize("dtype", [FP8, FP16])
@torch.no_grad()
def test_window_with_freed_pages(gpu, dtype):
    """A sequence that outgrows its pool: the same tokens as with a pool that
    keeps everything, and the logits of a window short of its end are those
    without one."""
    model = _model(gpu)
    prompts = _prompts((40, 13), gpu)
    kw = dict(max_seq_len=400, page_size=16, cache_dtype=dtype, window=48, sinks=5)
    small, big = _wrapper(model, 2, pages=12, **kw), _wrapper(model, 2, **kw)
    a, _ = small.generate(prompts, max_new_tokens=200)
    held = small.cache.pages - small.cache.free_pages
    assert held <= 2 * 6 and small.cache.length(0) > 200
    b, _ = big.generate(prompts, max_new_tokens=200)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    none = _wrapper(model, 2, max_seq_len=400, cache_dtype=dtype)
    for w in (big, none):
        w.capture_graph()
    x, y = (w.prefill([p[:20] for p in prompts[:1]] + [prompts[1]]) for w in (big, none))
    assert torch.equal(x, y)
    for i in range(60):
        t = torch.full((2,), 17 + i, device=gpu)
        x, y = big.replay(t).float(), none.replay(t).float()
        if i < 20:  # nothing is behind the window yet
            assert torch.allclose(x, y, atol=1e-3 * float(y.abs().max()))
    assert not torch.allclose(x, y, atol=1e-3 * float(y.abs().max()))


@torch.no_grad()
def test_resize(gpu):
    """A pool that grows, and shrinks to what is used: the same logits, bit for
    bit, once the step is captured again."""
    model = _model(gpu)
    prompts = _prompts((40, 7, 64), gpu)
    w = _wrapper(model, 3, pages=14)
    first = w.generate(prompts, max_new_tokens=8)[0]
    w.prefill(prompts)
    pos = lambda: torch.tensor([w.cache.length(b) for b in range(3)], device=gpu)  # noqa: E731
    t = torch.tensor([1, 2, 3], device=gpu)
    logits = []
    for pages in (None, 40, 12):
        if pages is not None:
            w.cache.resize(pages)
            with pytest.raises(RuntimeError, match="captured over"):
                w.replay(t)
        at = pos()
        w.cache.extend(1)
        logits.append(paged_forward(model, t, at, PagedStep(w.cache)).clone())
    v = _wrapper(model, 3, pages=30)
    v.capture_graph()
    v.prefill(prompts)
    for x in logits:
        assert torch.equal(x, v.replay(t))
    assert all(torch.equal(a, b) for a, b in zip(first, w.generate(prompts, max_new_tokens=8)[0]))


def test_refusals(gpu):
    w = _wrapper(_model(gpu), 4)
    prompts = _prompts((5, 6), gpu)
    for args, kw in (((prompts, 3), {}), ((prompts, 0), {}), ((prompts, 4), {}), ((prompts, 1), {}),
                     ((prompts, 2), dict(max_new_tokens=0)), ((prompts[:1], 65), {})):
        with pytest.raises(RuntimeError):
            w.generate_beams(*args, **kw)
    out, _, _ = w.generate_beams(prompts, 2, max_new_tokens=1)
    assert [len(x) for x in out] == [6, 7]


@pytest.mark.parametrize("dtype", [FP8, FP16])
@torch.no_grad()
def test_a_done_prompt_leaves_the_others_as_they_are(gpu, monkeypatch, dtype):
    """One of two prompts ends in its first steps, and the graph is replayed with
    its sequences empty: the other's text and score are those beside a prompt
    that goes on, and its beams have the pages."""
    K, n, eos = 3, 40, 5
    forward = PC.paged_forward
    likes = torch.zeros(2, 1, VOCAB, device=gpu)
    likes[0, :, eos], likes[1, :, eos] = 30, -math.inf

    def biased(model, ids, positions, step, last=None):
        x = forward(model, ids, positions, step, last)
        return (x.view(2, -1, VOCAB) + likes.to(x.dtype)).view(x.shape)

    monkeypatch.setattr(PC, "paged_forward", biased)
    model = _model(gpu)
    prompts = _prompts((60, 21), gpu)
    w = _wrapper(model, 2 * K, cache_dtype=dtype)
    texts, scores, _ = w.generate_beams(prompts, K, max_new_tokens=n)
    # the prompts' 4 and 2 pages, of which each beam copies the last one; of the
    # long search 4 pages each in the end, the first one shared
    small = _wrapper(model, 2 * K, cache_dtype=dtype, pages=6 + 2 * (K - 1) + 1)
    out, got, _ = small.generate_beams(prompts, K, max_new_tokens=n, eos_token_id=eos)
    assert len(out[0]) < 60 + 5 and int(out[0][-1]) == eos
    assert torch.equal(out[1], texts[1]) and got[1] == scores[1]
    assert [small.cache.length(b) for b in range(2 * K)] == [0] * K + [21 + n - 1] * K


@pytest.mark.parametrize("dtype", [FP8, FP16])
@torch.no_grad()
def test_beam_scores_are_their_steps(gpu, dtype):
    """The score of a text is the sum of its tokens' log-probabilities in a cache
    that is replayed with that text alone, in 64 bits: the same kernels on the
    same rows, so what differs is the rounding of each step's sum to fp32, 2^-24
    of it (it grows, so of the last one), and the selection's 3e-10."""
    model = _model(gpu)
    prompts = _prompts((21, 50), gpu)
    K, n = 4, 15
    w = _wrapper(model, 2 * K, cache_dtype=dtype)
    out, scores, _ = w.generate_beams(prompts, K, max_new_tokens=n)
    assert len({tuple(t[-n:].tolist()) for t in out}) == 2
    w = _wrapper(model, 2 * K, cache_dtype=dtype)
    w.capture_graph()
    # each prompt's K sequences all have the text (the prompts' forward with the
    # search's rows: other numbers of rows take other kernels)
    x = w._prefill(prompts, K).repeat_interleave(K, 0)
    for b in range(2 * K):
        if b % K:
            w.cache.fork(b - b % K, b)
    total = [0.0, 0.0]
    for i in range(n):
        logp = torch.log_softmax(x.double(), -1)
        token = torch.stack([t[len(p) + i] for p, t in zip(prompts, out)]).repeat_interleave(K)
        for p in range(2):
            total[p] += float(logp[p * K, token[p * K]])
        if i < n - 1:
            x = w.replay(token)
    for score, t in zip(scores, total):
        assert abs(score - t / n) <= (n * 2.0 ** -24 * abs(t) + n * 3e-10) / n


@pytest.mark.parametrize("dtype", [FP8, FP16])
@torch.no_grad()
def test_sequences_go_on_after_a_resize(gpu, dtype):
    """Steps, a pool of another size, a step captured over it with the sequences
    kept, and so on: bit for bit the steps of a cache that stays as it is."""
    model = _model(gpu)
    prompts = _prompts((40, 7, 64), gpu)
    a, b = (_wrapper(model, 3, cache_dtype=dtype, pages=30) for _ in range(2))
    for w in (a, b):
        w.capture_graph()
    assert torch.equal(a.prefill(prompts), b.prefill(prompts))
    g = torch.Generator().manual_seed(9)
    for pages in (None, 16, 50):
        if pages:
            a.cache.resize(pages)
            with pytest.raises(RuntimeError, match="captured over"):
                a.replay(torch.zeros(3, dtype=torch.long, device=gpu))
            a.capture_graph(keep=True)
        assert a.cache.lengths.tolist() == b.cache.lengths.tolist()
        for i in range(12):
            t = torch.randint(0, VOCAB, (3,), generator=g).to(gpu)
            assert torch.equal(a.replay(t).clone(), b.replay(t)), (pages, i)
    a.capture_graph()  # (as before: an empty cache)
    assert a.cache.free_pages == 50 and a.cache.lengths.tolist() == [0] * 3


@torch.no_grad()
def test_a_resize_gives_memory_back(gpu):
    """A wrapper with a captured step does not keep the pools that it was
    captured over, nor the step."""
    model = _model(gpu)
    w = _wrapper(model, 2, pages=4000)
    w.generate(_prompts((5, 9), gpu), max_new_tokens=3)
    w.cache.reset()
    size = lambda: sum(t.numel() * t.element_size() for t in w.cache.pools)  # noqa: E731
    torch.cuda.synchronize()
    was, held = size(), torch.cuda.memory_allocated(gpu)
    w.cache.resize(40)
    torch.cuda.synchronize()
    assert w.graph is None and torch.cuda.memory_allocated(gpu) <= held - (was - size())
    out, _ = w.generate(_prompts((5, 9), gpu), max_new_tokens=3)  # captured again
    assert [len(t) for t in out] == [8, 12]


@torch.no_grad()
def test_a_resize_takes_its_own_steps_alone(gpu):
    """A wrapper that went over to another cache keeps its step when the first
    one is resized, and is asked for a new one when its own is."""
    model = _model(gpu)
    w, other = _wrapper(model, 2, pages=20), _wrapper(model, 2, pages=20)
    w.capture_graph()
    first, w.cache = w.cache, other.cache
    t = torch.tensor([1, 2], device=gpu)
    with pytest.raises(RuntimeError, match="captured over"):
        w.replay(t)
    w.capture_graph()
    first.resize(10)
    w.prefill(_prompts((5, 9), gpu))
    a = w.replay(t).clone()
    w.cache.resize(10)
    assert w.graph is None
    other.capture_graph()
    other.prefill(_prompts((5, 9), gpu))
    assert torch.equal(a, other.replay(t))
