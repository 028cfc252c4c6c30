"""Shared pages, windows and moves of a paged cache (host side, on the CPU): the
tokens that each sequence reads through its page table, as operations follow each
other; and the host's side of a beam search."""

import math
import random

import pytest
import torch

from glorcq_amd import kernels
from glorcq_amd.paged_cache import GLoRCQPagedWrapper, PagedKVCache, PagedStep, _Beams


class Tokens(PagedKVCache):
    """A cache whose pages hold the names of tokens, and what each sequence
    should read."""

    def __init__(self, **kw):
        a = dict(layers=2, kv_heads=1, head_dim=64, max_seqs=5, max_seq_len=150, page_size=16,
                 device="cpu")
        super().__init__(**{**a, **kw})
        self.held = {}
        self.texts = [[] for _ in range(self.max_seqs)]
        self.names = 0
        self.copies = []

    def _copy_pages(self, src, dst, tokens):
        self.copies.append((src, dst, tokens))
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for s, d, n in zip(src, dst, tokens):
            for i in range(self.page_size):
                self.held[d, i] = self.held.get((s, i)) if i < n else None

    def _move_pages(self, src, pools):
        was = self.held
        self.held = {(d, i): was.get((s, i)) for d, s in enumerate(src)
                     for i in range(self.page_size)}

    def step(self, new):
        """extend, and the new tokens written as the append does."""
        self.extend(new)
        new = [new] * self.max_seqs if isinstance(new, int) else new
        written = []
        for b, n in enumerate(new):
            for i in range(self.length(b) - n, self.length(b)):
                at = (int(self.page_table[b, i // self.page_size]), i % self.page_size)
                assert at[0] >= 0
                written.append(at)
                self.names += 1
                self.held[at] = self.names
                self.texts[b].append(self.names)
        assert len(set(written)) == len(written)  # nobody writes another's page
        self.check(new)

    def check(self, new=None):
        size = self.page_size
        have = []
        for b in range(self.max_seqs):
            L = self.length(b)
            assert L == len(self.texts[b])
            row = self.page_table[b].tolist()
            assert all(p == -1 for p in row[-(-L // size):])
            first = L - (new[b] if new else 0)
            lo = max(0, first + 1 - self.window) if self.window else 0
            for i in range(L):
                if i < self.sinks or i >= lo or not self.window:
                    assert self.held[row[i // size], i % size] == self.texts[b][i], (b, i)
            own = [p for p in row if p >= 0]
            assert len(set(own)) == len(own)
            have += own
        assert self.free_pages + len(set(have)) == self.pages
        assert [self._refs[p] for p in range(self.pages)] == [have.count(p)
                                                            for p in range(self.pages)]
        assert self.lengths.tolist() == [self.length(b) for b in range(self.max_seqs)]


def test_forks_share_until_they_write():
    c = Tokens(pages=40)
    c.step([37, 0, 0, 0, 0])
    for b in (1, 2):
        c.fork(0, b)
        c.texts[b] = list(c.texts[0])
        c.check()
    assert c.free_pages == 37 and not c.copies
    c.step([0, 1, 0, 0, 0])  # sequence 1 writes: it copies, and shares two pages
    assert c.copies == [([c._own[0][2]], [c._own[1][2]], [5])] and c.free_pages == 36
    c.step([1, 0, 1, 0, 0])  # one of two copies, the other keeps the page
    assert len(c.copies) == 2 and len(c.copies[1][0]) == 1
    c.step(1)
    assert len(c.copies) == 2
    c.release(1)
    c.texts[1] = []
    c.check()
    c.step([20, 3, 20, 0, 0])
    c.reset()
    c.texts = [[] for _ in range(5)]
    c.check()
    assert c.free_pages == 40


def test_a_full_page_is_never_copied():
    c = Tokens(pages=20)
    c.step([32, 0, 0, 0, 0])
    for b in (1, 2, 3, 4):
        c.fork(0, b)
        c.texts[b] = list(c.texts[0])
    c.step(1)
    assert not c.copies and c.free_pages == 20 - 2 - 5


def test_reorder():
    c = Tokens(pages=60)
    c.step([20, 33, 5, 0, 40])
    c.reorder([1, 1, 4, 1, 0])
    t = c.texts
    c.texts = [list(t[i]) for i in (1, 1, 4, 1, 0)]
    c.check()
    c.step(1)
    assert len(c.copies) == 1 and len(c.copies[0][0]) == 2  # two of three that share
    before = c.page_table.clone()
    c.reorder(range(5))
    assert torch.equal(before, c.page_table)
    c.reorder([4, 3, 2, 1, 0])  # a permutation copies nothing
    c.texts.reverse()
    c.step([0, 1, 0, 1, 0])
    assert len(c.copies) == 1


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (20, 5), (33, 16), (47, 33), (200, 4)])
def test_window_frees_pages(window, sinks):
    c = Tokens(max_seq_len=400, window=window, sinks=sinks, max_seqs=2)
    c.step([70, 3])
    most = 0
    for n in [1] * 40 + [17, 0, 33] + [1] * 50:
        c.step([n, 1])
        most = max(most, sum(p >= 0 for p in c.page_table[0].tolist()))
    # (the 33 tokens of one step see no less than window + 32 positions)
    assert most <= -(-sinks // 16) + (window + 33) // 16 + 3
    assert PagedStep(c).visible(0) == (window, sinks)
    assert PagedStep(c).visible(window) == (window, sinks)
    assert PagedStep(c).visible(window + 1) == (window, sinks)
    if window > 1:
        assert PagedStep(c).visible(window - 1) == (window - 1, 0)


def test_resize_compacts():
    c = Tokens(pages=50, window=40, sinks=3)
    c.step([70, 20, 33, 0, 100])
    c.fork(4, 3)
    c.texts[3] = list(c.texts[4])
    c.step([1, 1, 0, 0, 3])
    c.release(1)
    c.texts[1] = []
    used = c.pages - c.free_pages
    with pytest.raises(RuntimeError, match="in use"):
        c.resize(used - 1)
    c.check()
    for pages in (used, used + 30):
        c.resize(pages)
        c.check()
        assert c.pages == pages and c.layers[1][0].shape[0] == pages
        assert sorted({p for own in c._own for p in own if p >= 0}) == list(range(used))
    c.step([1, 17, 1, 1, 1])
    empty = Tokens(pages=5)
    empty.resize(2)
    assert empty.free_pages == 2


def test_any_order():
    """Random operations; a step that the pool has no room for changes nothing."""
    for seed in range(30):
        r = random.Random(seed)
        w = r.choice((0, 0, 1, 18, 40))
        c = Tokens(pages=r.choice((14, 25, 60)), window=w, sinks=r.randrange(20) if w else 0)
        for _ in range(60):
            op = r.random()
            if op < 0.6:
                new = 1 if r.random() < 0.4 else [r.choice((0, 0, 1, 5, 40)) for _ in range(5)]
                was = (c.page_table.clone(), c.lengths.clone(), c.free_pages)
                try:
                    c.step(new)
                except RuntimeError as e:
                    assert "pages needed" in str(e) or "max_seq_len" in str(e)
                    assert torch.equal(was[0], c.page_table) and torch.equal(was[1], c.lengths)
                    assert was[2] == c.free_pages
            elif op < 0.75:
                b, d = r.randrange(5), r.randrange(5)
                c.release(d)
                c.texts[d] = []
                c.fork(b, d)
                c.texts[d] = list(c.texts[b])
            elif op < 0.9:
                parents = [r.randrange(5) for _ in range(5)]
                c.reorder(parents)
                c.texts = [list(c.texts[p]) for p in parents]
            elif op < 0.95:
                c.resize(max(c.pages - c.free_pages, 10))
            else:
                c.release(r.randrange(5))
                c.texts = [t if c.length(b) else [] for b, t in enumerate(c.texts)]
            if op >= 0.6:
                assert c.free_pages + len({p for o in c._own for p in o if p >= 0}) == c.pages


def test_refusals():
    c = Tokens()
    c.step([3, 4, 0, 0, 0])
    for f in (lambda: c.fork(0, 1), lambda: c.fork(0, 5), lambda: c.fork(-1, 2),
              lambda: c.reorder([0, 1]), lambda: c.reorder([0, 1, 2, 3, 5]),
              lambda: c.reorder([0, 1, 2, 3, -1]), lambda: c.resize(1), lambda: Tokens(sinks=3),
              lambda: Tokens(window=-1), lambda: Tokens(window=4, sinks=-1)):
        with pytest.raises(RuntimeError):
            f()
    c.check()


def _search(table, first, K, steps, eos, penalty):
    """A beam search over a chain of tokens (log-probabilities by the token
    before), written out: (text, score)."""
    beams, done = [((), 0.0)], []
    for step in range(1, steps + 1):
        options = []
        for k, (text, s) in enumerate(beams):
            row = table[text[-1]] if text else first
            options += [(-(s + float(x)), k, v, text) for v, x in enumerate(row)]
        options.sort()
        best, beams = options[:2 * K], []
        for i, (s, _, v, text) in enumerate(best):
            if v == eos:
                if i < K:
                    done.append((-s / step ** penalty, text + (v,)))
            elif len(beams) < K:
                beams.append((text + (v,), -s))
        done = sorted(done, key=lambda x: -x[0])[:K]
        if len(done) == K and done[-1][0] >= beams[0][1] / step ** penalty:
            return done[0][1], done[0][0]
    done += [(s / steps ** penalty, t) for t, s in beams]
    s, t = max(done, key=lambda x: x[0])
    return t, s


@pytest.mark.parametrize("K,eos,penalty,steps", [(1, None, 1.0, 6), (3, None, 1.0, 9), (4, 2, 1.0, 12),
                                                 (2, 0, 0.0, 12), (5, 3, 2.0, 10), (4, 2, 1.0, 1)])
def test_beam_bookkeeping(K, eos, penalty, steps):
    """The same search with the host's class, its selection done in fp64."""
    for seed in range(5):
        g = torch.Generator().manual_seed(seed)
        V, P = 12, 2
        table = torch.log_softmax(2 * torch.randn(V, V, generator=g, dtype=torch.float64), -1)
        first = torch.log_softmax(torch.randn(P, V, generator=g, dtype=torch.float64), -1)
        search = _Beams(P, K, eos, penalty)
        logp = first[:, None]
        scores = torch.zeros(P, 1, dtype=torch.float64)
        for step in range(1, steps + 1):
            c = (scores[..., None] + logp).flatten(1)
            v, i = c.sort(dim=1, descending=True, stable=True)
            v, i = v[:, :2 * K], i[:, :2 * K]
            parents = search.advance(torch.cat([v, (i // V).double(), (i % V).double()], 1).tolist(),
                                     step)
            assert len(parents) == P * K and all(r // K == p // K for r, p in enumerate(parents))
            if step == steps or search.done():
                break
            scores = torch.tensor(search.scores, dtype=torch.float64)
            logp = table[torch.tensor(search.tokens)].view(P, K, V)
        texts, values = search.best(step)
        for p in range(P):
            text, score = _search(table, first[p], K, steps, eos, penalty)
            assert math.isclose(values[p], score, rel_tol=1e-12)
            assert tuple(texts[p]) == text


class _Visits(list):
    """A list that counts the entries that are looked at."""
    seen = 0

    def __getitem__(self, i):
        _Visits.seen += len(range(len(self))[i]) if isinstance(i, slice) else 1
        return super().__getitem__(i)

    def __iter__(self):
        for i in range(len(self)):
            yield self[i]


def test_a_window_walks_each_page_once():
    """A step looks at the pages that leave the window with it, however many left
    before: of long sequences, their forks, and those that others became."""
    c = Tokens(max_seqs=4, max_seq_len=100000, pages=60, window=100, sinks=20)

    def visited(new):
        for b in range(4):
            c._own[b] = _Visits(c._own[b])
        _Visits.seen = 0
        c.extend(new)
        return _Visits.seen

    for _ in range(500):
        c.extend([100, 0, 0, 0])
    assert c.length(0) == 50000 and c.pages - c.free_pages <= 2 + 9 + 7
    # (a step of 100 tokens is followed by one that leaves (100 + 15) // 16 pages)
    assert visited([1, 0, 0, 0]) <= 7 + 1
    assert max(visited([1, 0, 0, 0]) for _ in range(39)) <= 2
    c.fork(0, 1)
    assert max(visited([1, 1, 0, 0]) for _ in range(40)) <= 4
    c.reorder([3, 1, 0, 1])
    assert [c.length(b) for b in range(4)] == [0, 50080, 50080, 50080]
    assert max(visited([0, 1, 1, 1]) for _ in range(40)) <= 6
    # a sequence that begins again frees what it has then
    c.release(1)
    for _ in range(30):
        c.extend([0, 20, 0, 0])
        kept = [i for i, p in enumerate(c.page_table[1].tolist()) if p >= 0]
        L = c.length(1)
        assert kept == [i for i in range(-(-L // 16))
                        if i < 2 or i >= max(0, L - 20 + 1 - 100) // 16]
    c.resize(50)
    assert visited(1) <= 16
    c.reset()
    assert c.free_pages == 50


@pytest.mark.parametrize("window", [0, 70])
def test_reordering_touches_what_differs(window):
    """Beams that share a long prompt change places: references are counted for
    the pages in which they differ, not for the prompt's."""
    c = Tokens(max_seqs=6, max_seq_len=10000, pages=660, window=window, sinks=20 if window else 0)
    c.extend([9990, 0, 0, 0, 0, 0])
    c.texts[0] = list(range(9990))
    c.held = {(p, i): 16 * j + i for j, p in enumerate(c._own[0]) for i in range(16)}
    c.names = 10000
    for b in range(1, 6):
        c.fork(0, b)
        c.texts[b] = list(c.texts[0])
    c.step(1)
    r = random.Random(window)
    for parents in ([1, 0, 3, 2, 5, 4], [5, 0, 1, 2, 3, 4], [0, 0, 1, 1, 4, 4], [3] * 6,
                    [0, 1, 2, 3, 4, 5], [2, 2, 2, 0, 4, 1], [5, 4, 5, 4, 5, 4]):
        c._refs = _Visits(c._refs)
        _Visits.seen = 0
        c.reorder(parents)
        # (a sequence's own pages are its last two; their references, before and after)
        assert _Visits.seen <= 6 * 8
        c._refs = list.copy(c._refs)
        c.texts = [list(c.texts[p]) for p in parents]
        c.check()
        c.step([r.choice((0, 1)) for _ in range(6)])
        c.reorder(range(6))
    for b in (3, 0, 5, 1, 2):
        c.release(b)
        c.texts[b] = []
        c.check()
    # sequences of other lengths, and empty ones
    c.step([3, 0, 40, 0, 0, 17])
    for parents in ([4, 0, 0, 1, 2, 5], [0, 3, 3, 0, 4, 4], [4] * 6, [3, 0, 1, 1, 1, 1]):
        c.reorder(parents)
        c.texts = [list(c.texts[p]) for p in parents]
        c.check()
        try:
            c.step(1)
        except RuntimeError as e:
            assert "max_seq_len" in str(e)


class _Device(torch.Tensor):
    """A tensor that counts what is uploaded to it."""
    uploads = 0

    def copy_(self, *args, **kw):
        _Device.uploads += 1
        return super().copy_(*args, **kw)


class _Wrapper(GLoRCQPagedWrapper):
    """Beam search's host side alone: a cache on the CPU, and a chain of tokens
    (logits by the token before) in the model's place."""

    def __init__(self, table, batch, **kw):
        self.max_batch_size, self.max_seq_len = batch, kw.get("max_seq_len", 150)
        self.cache = Tokens(max_seqs=batch, **kw)
        for name in ("page_table", "lengths"):  # (on the CPU it would be the host's own)
            setattr(self.cache, name, getattr(self.cache, name).clone().as_subclass(_Device))
        self.device = torch.device("cpu")
        self.static_input_ids = torch.zeros(batch, dtype=torch.long)
        self.table = table
        self.steps = []  # (sequences' lengths, uploads since the last step)

    def _ready(self):
        pass

    def _prefill(self, prompts, each):
        self.cache.reset()
        new = [n for p in prompts for n in [len(p)] + [0] * (each - 1)]
        self.cache.extend(new)
        _Device.uploads = 0
        return self.table[torch.stack([p[-1] for p in prompts])]

    def _replayed(self):
        """What the graph reads is what the host has."""
        c = self.cache
        assert c.page_table.tolist() == c._table.tolist()
        assert c.lengths.tolist() == [c.length(b) for b in range(c.max_seqs)]
        self.steps.append((c.lengths.tolist(), _Device.uploads))
        _Device.uploads = 0

    def _replay(self, input_ids, new):
        self.cache.extend(new)
        self._replayed()
        return self.table[input_ids]


def _select(logits, scores, num):
    """kernels.beam_select in fp64 on the CPU."""
    B, K = scores.shape
    c = scores.double()[..., None] + torch.log_softmax(logits.double(), -1).view(B, K, -1)
    v, i = c.flatten(1).sort(dim=1, descending=True, stable=True)
    v, i, V = v[:, :num], i[:, :num], c.shape[2]
    return v.float(), i // V, i % V


def test_beams_upload_a_table_a_step(monkeypatch):
    """A step of a beam search brings the device the page table and the lengths
    once, however many sequences fork or change places."""
    monkeypatch.setattr(kernels, "beam_select", _select)
    g = torch.Generator().manual_seed(1)
    w = _Wrapper(2 * torch.randn(40, 40, generator=g), 12)
    prompts = [torch.tensor([3] * 20), torch.tensor([5] * 37), torch.tensor([9])]
    w.generate_beams(prompts, 4, max_new_tokens=30)
    assert len(w.steps) == 29
    assert w.steps[0][0] == [21] * 4 + [38] * 4 + [2] * 4
    assert all(n <= 2 for _, n in w.steps)
    # forks, moves and ends by themselves bring theirs at once
    w.cache.reset()
    w.cache.extend([20] + [0] * 11)
    for f in (lambda c: c.fork(0, 3), lambda c: c.reorder([3, 0] + [0] * 10),
              lambda c: c.release(2), lambda c: c.resize(30)):
        f(w.cache)
        w._replayed()
    # a search that the pool has no room for leaves the device what the host has
    w = _Wrapper(w.table, 8, pages=6)
    with pytest.raises(RuntimeError, match="pages needed"):
        w.generate_beams([torch.tensor([3] * 40)] * 1 + [torch.tensor([7])], 4, max_new_tokens=30)
    w._replayed()


def test_prompts_that_are_done_give_their_pages_back(monkeypatch):
    """Two prompts end early; the third's long search has their pages, and finds
    what it finds alone.  Nobody's results change when another one ends."""
    monkeypatch.setattr(kernels, "beam_select", _select)
    g = torch.Generator().manual_seed(2)
    V, eos = 40, 0
    table = torch.randn(V, V, generator=g)
    table[:20, 20:] = table[20:, :20] = -50  # two groups of tokens:
    table[:20, eos] += 9                     # one ends soon, one never
    prompts = [torch.tensor([3] * 50), torch.tensor([25] * 20), torch.tensor([7] * 33)]
    K, n = 3, 80
    # 7 pages of prompts, each of whose beams copies one; the long search's beams
    # at 100 tokens have 7 pages each, but the prompt's first, which they share
    w = _Wrapper(table, 3 * K, pages=1 + K * 6 + 1)
    out, scores, _ = w.generate_beams(prompts, K, max_new_tokens=n, eos_token_id=eos)
    assert len(w.steps) == n - 1 and [len(t) for t in out][1] == 20 + n
    ends = [next(i for i, (lens, _) in enumerate(w.steps) if lens[b * K:b * K + K] == [0] * K)
            for b in (0, 2)]
    assert max(ends) < 20
    for lens, _ in w.steps[max(ends):]:
        assert lens[:K] == lens[2 * K:] == [0] * K and min(lens[K:2 * K]) > 0
    for b, p in enumerate(prompts):
        one = _Wrapper(table, K)
        text, score, _ = one.generate_beams([p], K, max_new_tokens=n, eos_token_id=eos)
        assert torch.equal(text[0], out[b]) and score[0] == scores[b]
    logp = torch.log_softmax(table.double(), -1)
    for p, t, s in zip(prompts, out, scores):
        want, value = _search(logp, logp[int(p[-1])], K, n, eos, 1.0)
        assert tuple(t[len(p):].tolist()) == want
        assert math.isclose(s, value, rel_tol=n * 2.0 ** -23)
    # all of the cache can be used again
    w.cache.reset()
    assert w.cache.free_pages == w.cache.pages


def test_an_end_is_one_token(monkeypatch):
    """A list of them would never be found among the tokens: it is refused."""
    monkeypatch.setattr(kernels, "beam_select", _select)
    g = torch.Generator().manual_seed(3)
    w = _Wrapper(torch.randn(20, 20, generator=g), 2)
    prompt = [torch.tensor([4, 5])]
    for bad in ([2], [2, 3], (1,), 2.0, "2", torch.tensor([1, 2])):
        with pytest.raises(RuntimeError, match="eos_token_id"):
            w.generate_beams(prompt, 2, max_new_tokens=4, eos_token_id=bad)
    a = w.generate_beams(prompt, 2, max_new_tokens=9, eos_token_id=7)
    b = w.generate_beams(prompt, 2, max_new_tokens=9, eos_token_id=torch.tensor(7))
    assert torch.equal(a[0][0], b[0][0]) and a[1] == b[1]
