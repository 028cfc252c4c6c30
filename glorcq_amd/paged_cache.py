"""A paged key/value cache for a model, and greedy generation over it.

The static cache of the graph wrapper holds one position for the whole batch
and max_seq_len positions a sequence in fp16.  Here every sequence has a length
of its own, memory is taken a page at a time from one pool a layer, and values
are e4m3 codes with a power-of-two scale for each 16 tokens of a head (half the
bytes), or fp16.  Logits differ from the static cache's by these roundings, and
with fp16 pages by k's and q's, which are rounded once, after norm and rotation,
where the static path rounds between them too.  No reference counterpart (its model path has the static cache
alone, inference/graph_wrapper.py:69-149).

* `PagedKVCache` -- the pools of all layers, the page table and the lengths:
  which pages belong to which sequence is decided on the host, between steps.
  Sequences may share pages (forks, beams); a page is copied when one of them is
  about to write it.  With a window, pages that no later token sees are freed;
* `PagedStep` -- one step's view of it, what a fused decoder layer takes as
  `past_key_values`;
* `paged_forward` -- a model's forward over the new tokens of a batch;
* `GLoRCQPagedWrapper` -- prompts of different lengths, then decode steps as
  replays of one captured graph: greedy, or beams.
"""

from __future__ import annotations

import operator
import time
import weakref
from collections import Counter

import torch

from . import kernels


class PagedKVCache:
    """Pages of `page_size` tokens for `layers` layers and up to `max_seqs`
    sequences of up to `max_seq_len` tokens; `pages` of them in each layer's
    pool (default: enough for all sequences at full length).  With a `window`,
    tokens attend to their last `window` positions and to the first `sinks` of
    their sequence (in layers whose own window is not smaller), and `extend`
    frees the pages that lie between: a sequence then needs about sinks + window
    tokens' pages, however long it gets up to max_seq_len (prompts, all of
    theirs).  Positions stay the sequence's own, in the model's rotation too."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, max_seqs: int, max_seq_len: int,
                 page_size: int = 64, pages: int | None = None,
                 dtype: torch.dtype = torch.float8_e4m3fn, device="cuda",
                 window: int = 0, sinks: int = 0):
        if max_seqs < 1 or max_seq_len < 1:
            raise RuntimeError("max_seqs and max_seq_len must be positive")
        if window < 0 or sinks < 0 or (sinks and not window):
            raise RuntimeError("window and sinks must be >= 0, and sinks need a window")
        each = -(-max_seq_len // page_size)
        self.page_size, self.max_seqs, self.max_seq_len = page_size, max_seqs, max_seq_len
        self.window, self.sinks = window, sinks
        self.pages = max_seqs * each if pages is None else pages
        if self.pages < 1:
            raise RuntimeError("a cache needs a page")
        self._wrappers = weakref.WeakSet()  # whose captured steps run over the pools
        self._shape = (kv_heads, head_dim, page_size, dtype, device, layers)
        self._take_pools(kernels.paged_cache_tensors(self.pages, *self._shape))
        self.device = self.pools[0].device
        # (a page that no sequence has: out of range, so that nothing reads or writes it)
        self._table = torch.full((max_seqs, each), -1, dtype=torch.int32)
        self.page_table = self._table.to(self.device)
        self.lengths = torch.zeros(max_seqs, dtype=torch.int32, device=self.device)
        self._changed = [False, False]  # page table and lengths, since they were uploaded
        self._workspaces: dict = {}
        self._len = [0] * max_seqs
        # pages of each sequence's positions (-1: freed behind the window), and
        # how many sequences have each
        self._own: list[list[int]] = [[] for _ in range(max_seqs)]
        self._refs = [0] * self.pages
        self._free = list(range(self.pages - 1, -1, -1))
        # the first page behind the sinks that a window has not left yet
        self._behind = [-(-sinks // page_size)] * max_seqs

    @classmethod
    def for_model(cls, model, max_seqs: int, max_seq_len: int, **kwargs):
        """A cache of the model's layers, heads and device."""
        c = model.config
        head_dim = getattr(c, "head_dim", None) or c.hidden_size // c.num_attention_heads
        return cls(c.num_hidden_layers, c.num_key_value_heads, head_dim, max_seqs, max_seq_len,
                   device=next(model.parameters()).device, **kwargs)

    def _take_pools(self, pools) -> None:
        """All layers' pools, one behind the other, and each layer's; `pools_key`
        is theirs alone."""
        self.pools, self.pools_key = pools, object()
        self.layers = [tuple(None if x is None else x[i] for x in pools)
                       for i in range(pools[0].shape[0])]

    def length(self, seq: int) -> int:
        return self._len[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, new) -> None:
        """Makes room for `new` tokens a sequence (one number for all, or one a
        sequence) and counts them: the next step's tokens.  Raises, with nothing
        changed, where a sequence would pass max_seq_len or the pool runs out.
        A shared page that would get tokens is copied first, and pages that lie
        behind the new tokens' window are freed."""
        uniform = isinstance(new, int)
        new = [new] * self.max_seqs if uniform else [int(n) for n in new]
        if len(new) != self.max_seqs or min(new) < 0:
            raise RuntimeError(f"new must hold {self.max_seqs} token counts >= 0")
        # (on the path of every decode step: without windows and forks, sums and
        # compares of a few numbers a sequence)
        size, window, refs = self.page_size, self.window, self._refs
        lens = [L + n for L, n in zip(self._len, new)]
        if max(lens) > self.max_seq_len:
            b = next(b for b, L in enumerate(lens) if L > self.max_seq_len)
            raise RuntimeError(f"sequence {b} would have {lens[b]} tokens "
                               f"(max_seq_len {self.max_seq_len})")
        need = [-(-L // size) - len(own) for L, own in zip(lens, self._own)]
        behind, copied = [], []  # behind: (sequence, first page, the one after the last)
        left = {}                # references given up
        for b, L in enumerate(self._len):
            if window and new[b]:
                first, end = self._behind[b], (L + 1 - window) // size
                if first < end:
                    behind.append((b, first, end))
                    for page in self._own[b][first:end]:
                        left[page] = left.get(page, 0) + 1
            if L % size and refs[page := self._own[b][-1]] > 1 and new[b] \
                    and refs[page] - left.get(page, 0) > 1:  # (the last one that has it keeps it)
                copied.append(b)
                left[page] = left.get(page, 0) + 1
        given = [p for p, n in left.items() if refs[p] == n]
        wanted, there = sum(need) + len(copied), len(self._free) + len(given)
        if wanted > there:
            raise RuntimeError(f"{wanted} pages needed, {there} free")
        self._free.extend(given)
        for p, n in left.items():
            refs[p] -= n
        for b, first, end in behind:
            self._own[b][first:end] = [-1] * (end - first)
            self._table[b, first:end] = -1
            self._behind[b] = end
        if copied:
            pairs = [(self._own[b][-1], self._take_page(b, len(self._own[b]) - 1),
                      self._len[b] % size) for b in copied]
            self._copy_pages(*map(list, zip(*pairs)))
        if wanted:
            for b, n in enumerate(need):
                for _ in range(n):
                    self._take_page(b, len(self._own[b]))
        self._len = lens
        if wanted or behind:
            self._changed[0] = True
        if uniform and not self._changed[1]:
            self.lengths.add_(new[0])
        else:
            self._changed[1] = True
        self._upload()

    def _take_page(self, seq: int, i: int) -> int:
        """A free page as the sequence's i-th."""
        page = self._free.pop()
        self._refs[page] = 1
        self._own[seq][i:i + 1] = [page]
        self._table[seq, i] = page
        return page

    def _copy_pages(self, src, dst, tokens) -> None:
        k, v, ks, vs = self.pools
        kernels.paged_copy(k, v, src, dst, k_scales=ks, v_scales=vs, tokens=tokens)

    def _give_back(self, pages) -> None:
        for p in pages:
            if p >= 0:
                self._refs[p] -= 1
                if self._refs[p] == 0:
                    self._free.append(p)

    def _set_row(self, seq: int, own) -> None:
        self._own[seq] = list(own)
        self._table[seq].fill_(-1)
        if own:
            self._table[seq, :len(own)] = torch.tensor(own, dtype=torch.int32)

    def _upload(self) -> None:
        """Brings the device the page table and the lengths, where they changed."""
        table, lens = self._changed
        if table:
            self.page_table.copy_(self._table)
        if lens:
            self.lengths.copy_(torch.tensor(self._len, dtype=torch.int32))
        self._changed = [False, False]

    def release(self, seq: int) -> None:
        """Gives a sequence's pages back (those that it shares stay the others');
        its length is 0 again."""
        self._release(seq)
        self._upload()

    def _release(self, seq):
        self._give_back(reversed(self._own[seq]))
        self._own[seq] = []
        self._len[seq] = 0
        self._behind[seq] = -(-self.sinks // self.page_size)
        self._table[seq].fill_(-1)
        self._changed = [True, True]

    def fork(self, src: int, dst: int) -> None:
        """Makes the empty sequence dst one with src's tokens.  They share its
        pages; the last one is copied when either gets a token."""
        self._fork(src, dst)
        self._upload()

    def _fork(self, src, dst):  # (without the upload: the next extend's will do)
        for b in (src, dst):
            if not 0 <= b < self.max_seqs:
                raise RuntimeError(f"no sequence {b}")
        if self._len[dst]:
            raise RuntimeError(f"sequence {dst} is not empty (release it first)")
        if src == dst:
            return
        for p in self._own[src]:
            if p >= 0:
                self._refs[p] += 1
        self._len[dst], self._behind[dst] = self._len[src], self._behind[src]
        self._set_row(dst, self._own[src])
        self._changed = [True, True]

    def reorder(self, parents) -> None:
        """Sequence b becomes what sequence parents[b] was (parents: one a
        sequence); pages that nobody has any more are freed."""
        self._reorder(parents)
        self._upload()

    def _reorder(self, parents):
        parents = [int(p) for p in parents]
        if len(parents) != self.max_seqs or not all(0 <= p < self.max_seqs for p in parents):
            raise RuntimeError(f"parents must hold {self.max_seqs} sequences")
        moved = [b for b, p in enumerate(parents) if p != b]
        if not moved:
            return
        lens = [self._len[p] for p in parents]
        # a sequence that several become, once for each beyond the first, beside
        # one that nobody does: the pages that both begin with (beams, their
        # prompt's) are had as often as before
        children = Counter(parents)
        more = [p for p in sorted(children) for _ in range(children[p] - 1)]
        gone = [b for b in range(self.max_seqs) if b not in children]
        tails = []
        for p, b in zip(more, gone):
            n = _same(self._own[p], self._own[b])
            for page in self._own[p][n:]:
                if page >= 0:
                    self._refs[page] += 1
            tails.append(self._own[b][n:])
        for pages in tails:
            self._give_back(pages)
        own = [list(self._own[parents[b]]) for b in moved]
        for b, pages in zip(moved, own):
            self._own[b] = pages
        self._table[moved] = self._table[[parents[b] for b in moved]]
        self._behind = [self._behind[p] for p in parents]
        self._changed[0] = True
        if lens != self._len:
            self._len = lens
            self._changed[1] = True

    def resize(self, pages: int) -> None:
        """Moves the pages that sequences have to the front of new pools of
        `pages` pages each, and lets the old ones go, with wrappers' steps that
        were captured over them (GLoRCQPagedWrapper.capture_graph(keep=True)
        captures them again)."""
        live = sorted({p for own in self._own for p in own if p >= 0})
        if pages < max(len(live), 1):
            raise RuntimeError(f"{len(live)} pages are in use")
        pools = kernels.paged_cache_tensors(pages, *self._shape)
        self._move_pages(live, pools)
        place = {p: i for i, p in enumerate(live)}
        over = [w for w in self._wrappers if w._graph_pools is self.pools_key]
        self._take_pools(pools)
        if over:
            torch.cuda.synchronize(self.device)  # (no replay is under way)
        for w in over:
            w.graph = w.static_logits = None
        self.pages = pages
        self._refs = [self._refs[p] for p in live] + [0] * (pages - len(live))
        self._free = list(range(pages - 1, len(live) - 1, -1))
        for b, own in enumerate(self._own):
            self._set_row(b, [place.get(p, -1) for p in own])
        self._changed[0] = True
        self._upload()

    def _move_pages(self, src, pools) -> None:
        k, v, ks, vs = self.pools
        kernels.paged_copy(k, v, src, list(range(len(src))), k_scales=ks, v_scales=vs, to=pools)

    def reset(self) -> None:
        for b in range(self.max_seqs):
            self._give_back(reversed(self._own[b]))
            self._own[b] = []
        self._len = [0] * self.max_seqs
        self._behind = [-(-self.sinks // self.page_size)] * self.max_seqs
        self._table.fill_(-1)
        self._changed = [True, True]
        self._upload()

    def workspace(self, q: torch.Tensor):
        """The attention workspace of steps of q's shape, one for all layers:
        steps of one cache run in order.  None for the first one under graph
        capture (its zeros would be written by replays alone)."""
        ws = self._workspaces.get(q.shape)
        if ws is None and torch.cuda.is_current_stream_capturing():
            return None
        if ws is None:
            ws = self._workspaces[q.shape] = kernels.paged_attention_workspace(
                q, self.layers[0][0], self.page_table)
        return ws


def _same(a: list, b: list) -> int:
    """How many entries two lists have in common at their front."""
    lo, hi = 0, min(len(a), len(b))
    while lo < hi:
        mid = (lo + hi + 1) // 2
        if a[lo:mid] == b[lo:mid]:
            lo = mid
        else:
            hi = mid - 1
    return lo


class PagedStep:
    """The new tokens of a step, after cache.extend: rows [starts[b],
    starts[b + 1]) of the step are sequence b's (starts int32 on the device), or
    without starts the same number each."""

    def __init__(self, cache: PagedKVCache, starts: torch.Tensor | None = None):
        self.cache, self.starts = cache, starts
        self.page_table, self.lengths = cache.page_table, cache.lengths

    def visible(self, window: int) -> tuple[int, int]:
        """Window and sinks of a layer whose own window is this (0: none)."""
        c = self.cache
        return (c.window, c.sinks) if c.window and not 0 < window < c.window else (window, 0)

    def workspace(self, q):
        # (a step whose sequences bring one token each, as decode steps do, is
        # run again and again; others take the stream's)
        if self.starts is None and q.shape[0] == self.cache.max_seqs:
            return self.cache.workspace(q)
        return None


def paged_forward(model, input_ids: torch.Tensor, positions: torch.Tensor, step: PagedStep,
                  last: torch.Tensor | None = None) -> torch.Tensor:
    """Logits of a causal LM whose decoder layers are fused
    (decoder.fuse_decoder_layers) over a step's tokens: input_ids and positions
    (T,) -> (T, vocab), or of the rows `last` alone.  Without starts the rows
    run as T sequences of one token, otherwise as one row of tokens."""
    from .decoder import GLoRCQQwen3DecoderLayer

    inner = model.model
    if not all(isinstance(layer, GLoRCQQwen3DecoderLayer) for layer in inner.layers):
        raise RuntimeError("paged_forward needs fused decoder layers (decoder.fuse_decoder_layers)")
    T = input_ids.shape[0]
    shape = (T, 1) if step.starts is None else (1, T)
    h = inner.embed_tokens(input_ids.view(shape))
    pe = inner.rotary_emb(h, positions.view(shape))
    for layer in inner.layers:
        h = layer(h, position_embeddings=pe, past_key_values=step)
    h = h.reshape(T, -1)
    if last is not None:
        h = h[last]
    return model.lm_head(inner.norm(h))


class GLoRCQPagedWrapper:
    """Generation over a paged cache, greedy or by beams: prompts of different
    lengths in one forward, then one captured graph's replay a token.

    Usage:
        wrapper = GLoRCQPagedWrapper(model, max_batch_size=4, max_seq_len=4096)
        outputs, seconds = wrapper.generate(prompts, max_new_tokens=128)
        outputs, scores, seconds = wrapper.generate_beams(prompt, num_beams=4)
    """

    def __init__(self, model, max_batch_size=1, max_seq_len=4096, page_size=64, pages=None,
                 cache_dtype=torch.float8_e4m3fn, window=0, sinks=0):
        self.model = model
        self.max_batch_size, self.max_seq_len = max_batch_size, max_seq_len
        self.cache = PagedKVCache.for_model(model, max_batch_size, max_seq_len,
                                            page_size=page_size, pages=pages, dtype=cache_dtype,
                                            window=window, sinks=sinks)
        self.device = self.cache.device
        self.static_input_ids = torch.zeros(max_batch_size, dtype=torch.long, device=self.device)
        self.static_logits = None
        self.graph = self._graph_pools = None
        self.graph_stream = torch.cuda.Stream(device=self.device)
        self.last_timing = {}

    def _step(self):
        return paged_forward(self.model, self.static_input_ids, self.cache.lengths.long() - 1,
                             PagedStep(self.cache))

    @torch.no_grad()
    def capture_graph(self, keep=False):
        """Warm-up steps on a side stream, then one decode step captured.  The
        cache is emptied, or with `keep` its sequences stay; meanwhile they have
        no tokens (one before position 0 is written nowhere)."""
        self.model.eval()
        cache = self.cache
        if keep:
            cache.lengths.zero_()
        else:
            cache.reset()
        try:
            s = torch.cuda.Stream(device=self.device)
            s.wait_stream(torch.cuda.current_stream(self.device))
            with torch.cuda.stream(s):
                for _ in range(3):
                    self._step()
            torch.cuda.current_stream(self.device).wait_stream(s)
            torch.cuda.synchronize(self.device)
            self.graph, graph = None, torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=self.graph_stream):
                self.static_logits = self._step()
            self.graph, self._graph_pools = graph, cache.pools_key
            cache._wrappers.add(self)
        finally:
            if keep:
                cache._changed[1] = True
                cache._upload()

    @torch.no_grad()
    def prefill(self, prompts):
        """The prompts' forward into an empty cache -> the logits after each
        one's last token (batch, vocab)."""
        return self._prefill(prompts, 1)

    def _prefill(self, prompts, each):
        """prefill of prompts of `each` sequences, into the first one of each."""
        lens = [int(p.shape[0]) if p.dim() == 1 else 0 for p in prompts]
        if len(prompts) * each != self.max_batch_size or min(lens) < 1:
            raise RuntimeError(
                f"{self.max_batch_size // each} 1-D prompts of at least one token needed")
        self.cache.reset()
        new = [n for m in lens for n in [m] + [0] * (each - 1)]
        self.cache.extend(new)
        starts = torch.tensor([0] + new).cumsum(0)
        pos = torch.cat([torch.arange(n) for n in lens])
        step = PagedStep(self.cache, starts.to(torch.int32).to(self.device))
        return paged_forward(self.model, torch.cat([p.to(self.device) for p in prompts]),
                             pos.to(self.device), step,
                             last=(starts[each::each] - 1).to(self.device))

    @torch.no_grad()
    def replay(self, input_ids):
        """One decode step: (batch,) ids, the sequences' next tokens -> the
        captured logits buffer (batch, vocab)."""
        return self._replay(input_ids, 1)

    def _replay(self, input_ids, new):
        """replay, with what cache.extend takes."""
        if self._graph_pools not in (None, self.cache.pools_key):
            raise RuntimeError("the step was captured over pools that the cache no longer has "
                               "(capture_graph; with keep=True the sequences stay)")
        if self.graph is None:
            raise RuntimeError("no captured step (capture_graph, which empties the cache)")
        if input_ids.shape != self.static_input_ids.shape:
            raise RuntimeError(f"input_ids must be ({self.max_batch_size},)")
        self.static_input_ids.copy_(input_ids)
        self.cache.extend(new)
        self.graph.replay()
        return self.static_logits

    def _ready(self):
        if self.graph is None or self._graph_pools is not self.cache.pools_key:
            self.capture_graph()

    @torch.no_grad()
    def generate(self, prompts, max_new_tokens=100):
        """Greedy generation from a list of 1-D prompts; returns (list of prompt
        + generated ids, seconds).  Sequences stop together, at max_new_tokens
        or where the longest reaches max_seq_len."""
        self._ready()
        t0 = time.time()
        token = torch.argmax(self.prefill(prompts), dim=-1)
        tokens = [token]
        torch.cuda.synchronize(self.device)
        t1 = time.time()
        room = self.max_seq_len - max(int(p.shape[0]) for p in prompts)
        for _ in range(min(max_new_tokens - 1, room)):
            token = torch.argmax(self.replay(token), dim=-1)
            tokens.append(token)
        torch.cuda.synchronize(self.device)
        t2 = time.time()
        self.last_timing = {"prefill_s": t1 - t0, "decode_s": t2 - t1,
                            "decode_tokens": len(tokens) - 1}
        new = torch.stack(tokens, 1)
        return [torch.cat([p.to(self.device), new[b]]) for b, p in enumerate(prompts)], t2 - t0

    @torch.no_grad()
    def generate_beams(self, prompts, num_beams, max_new_tokens=100, eos_token_id=None,
                       length_penalty=1.0):
        """Beam search from a list of 1-D prompts, max_batch_size / num_beams of
        them: returns (list of prompt + generated ids, list of their scores,
        seconds), each prompt's best.  A score is the sum of the generated
        tokens' log-probabilities over their number ** length_penalty.

        A step takes each prompt's 2 num_beams best continuations
        (kernels.beam_select).  Those that end in eos_token_id are finished, if
        they are among the first num_beams; the others go on, num_beams of them,
        sharing their pages with their parents.  A prompt is done when it has
        num_beams finished ones and its best beam, as it is, scores below all of
        them; its pages are the other prompts' from then on.  All stop at max_new_tokens, or where the longest reaches
        max_seq_len."""
        K = num_beams
        if K < 1 or 2 * K > 128 or self.max_batch_size % K:
            raise RuntimeError("num_beams must be in [1, 64] and divide max_batch_size "
                               f"({self.max_batch_size})")
        if max_new_tokens < 1:
            raise RuntimeError("max_new_tokens must be positive")
        if eos_token_id is not None:
            try:
                eos_token_id = operator.index(eos_token_id)
            except TypeError:
                raise RuntimeError(f"eos_token_id must be one token (got {eos_token_id!r})") from None
        self._ready()
        t0 = time.time()
        logits = self._prefill(prompts, K)
        P, vocab = logits.shape
        if vocab < 2 * K:
            raise RuntimeError(f"a vocabulary of {vocab} has no {2 * K} continuations")
        search = _Beams(P, K, eos_token_id, length_penalty)
        room = self.max_seq_len - max(int(p.shape[0]) for p in prompts)
        try:
            step = self._search(search, logits, min(max_new_tokens, room + 1))
        finally:
            self.cache._upload()
        texts, values = search.best(step)
        t1 = time.time()
        self.last_timing = {"beams_s": t1 - t0, "steps": step}
        out = [torch.cat([p.to(self.device), torch.tensor(t, dtype=torch.long).to(self.device)])
               for p, t in zip(prompts, texts)]
        return out, values, t1 - t0

    def _search(self, search, logits, steps):
        """A beam search from the prompts' logits on; the steps it took.  (Forks
        and moves reach the device with the tokens of the step after them.)"""
        P, K = search.P, search.K
        for p in range(P):
            for j in range(1, K):
                self.cache._fork(p * K, p * K + j)
        scores = logits.new_zeros((P, 1), dtype=torch.float32)
        for step in range(1, steps + 1):
            best = kernels.beam_select(logits, scores, 2 * K)
            # (one copy to the host; int64 and fp32 are exact in fp64 up to 2^53)
            found = torch.cat([x.double() for x in best], 1).tolist()
            parents = search.advance(found, step)
            if step == steps or search.done():
                break
            if step > 1:  # (a first step's beams are all their prompt's)
                self.cache._reorder(parents)
            new = [0 if d else 1 for d in search.ended for _ in range(K)]
            for b in range(P * K):
                if new[b] == 0 and self.cache.length(b):
                    self.cache._release(b)
            scores = torch.tensor(search.scores, dtype=torch.float32).to(self.device)
            logits = self._replay(torch.tensor(search.tokens).to(self.device),
                                  new if any(search.ended) else 1)
        return step


class _Beams:
    """The host's side of a beam search: beams and finished texts of each prompt."""

    def __init__(self, prompts, beams, eos, penalty):
        self.P, self.K, self.eos, self.penalty = prompts, beams, eos, penalty
        self.scores = [[0.0] * beams for _ in range(prompts)]
        self.tokens = [0] * (prompts * beams)
        self._texts = [None] * (prompts * beams)  # (text before, token)
        self._finished = [[] for _ in range(prompts)]  # (score, text), the best first
        self.ended = [False] * prompts

    def advance(self, found, step):
        """found: of each prompt, its 2 K best continuations' scores, parents and
        tokens, one behind the other.  Returns each sequence's parent.  (A prompt
        that is done stays as it is, whatever is found of it.)"""
        K, parents, texts = self.K, [], []
        for p, row in enumerate(found):
            if self.ended[p]:
                parents += range(p * K, p * K + K)
                texts += self._texts[p * K:p * K + K]
                continue
            n = len(row) // 3
            live = []
            for i in range(n):
                score, parent, token = row[i], p * K + int(row[n + i]), int(row[2 * n + i])
                if token == self.eos:
                    if i < K:
                        self._finish(p, score, (self._texts[parent], token), step)
                elif len(live) < K:
                    live.append((score, parent, token))
            self.scores[p] = [s for s, _, _ in live]
            for j, (_, parent, token) in enumerate(live):
                self.tokens[p * K + j] = token
                parents.append(parent)
                texts.append((self._texts[parent], token))
            done = self._finished[p]
            if len(done) == K and done[-1][0] >= self._value(live[0][0], step):
                self.ended[p] = True
        self._texts = texts
        return parents

    def _value(self, score, tokens):
        return score / tokens ** self.penalty

    def _finish(self, p, score, text, tokens):
        done = self._finished[p]
        done.append((self._value(score, tokens), text))
        done.sort(key=lambda x: -x[0])
        del done[self.K:]

    def done(self):
        return all(self.ended)

    def best(self, step):
        """Texts and scores; beams that are still going count as they are."""
        texts, values = [], []
        for p in range(self.P):
            all_of = list(self._finished[p])
            if not self.ended[p]:
                all_of += [(self._value(s, step), self._texts[p * self.K + j])
                           for j, s in enumerate(self.scores[p])]
            value, text = max(all_of, key=lambda x: x[0])
            tokens = []
            while text is not None:
                text, token = text
                tokens.append(token)
            texts.append(tokens[::-1])
            values.append(value)
        return texts, values
