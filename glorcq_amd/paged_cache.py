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
  which pages belong to which sequence is decided on the host, between steps;
* `PagedStep` -- one step's view of it, what a fused decoder layer takes as
  `past_key_values`;
* `paged_forward` -- a model's forward over the new tokens of a batch;
* `GLoRCQPagedWrapper` -- prompts of different lengths, then decode steps as
  replays of one captured graph.
"""

from __future__ import annotations

import time

import torch

from . import kernels


class PagedKVCache:
    """Pages of `page_size` tokens for `layers` layers and up to `max_seqs`
    sequences of up to `max_seq_len` tokens; `pages` of them in each layer's
    pool (default: enough for all sequences at full length)."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, max_seqs: int, max_seq_len: int,
                 page_size: int = 64, pages: int | None = None,
                 dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
        if max_seqs < 1 or max_seq_len < 1:
            raise RuntimeError("max_seqs and max_seq_len must be positive")
        each = -(-max_seq_len // page_size)
        self.page_size, self.max_seqs, self.max_seq_len = page_size, max_seqs, max_seq_len
        self.pages = max_seqs * each if pages is None else pages
        if self.pages < 1:
            raise RuntimeError("a cache needs a page")
        self.layers = [kernels.paged_cache_tensors(self.pages, kv_heads, head_dim, page_size,
                                                   dtype, device) for _ in range(layers)]
        self.device = self.layers[0][0].device if layers else torch.device(device)
        # (a page that no sequence has: out of range, so that nothing reads or writes it)
        self._table = torch.full((max_seqs, each), -1, dtype=torch.int32)
        self.page_table = self._table.to(self.device)
        self.lengths = torch.zeros(max_seqs, dtype=torch.int32, device=self.device)
        self._workspaces: dict = {}
        self._len = [0] * max_seqs
        self._own: list[list[int]] = [[] for _ in range(max_seqs)]
        self._free = list(range(self.pages - 1, -1, -1))

    @classmethod
    def for_model(cls, model, max_seqs: int, max_seq_len: int, **kwargs):
        """A cache of the model's layers, heads and device."""
        c = model.config
        head_dim = getattr(c, "head_dim", None) or c.hidden_size // c.num_attention_heads
        return cls(c.num_hidden_layers, c.num_key_value_heads, head_dim, max_seqs, max_seq_len,
                   device=next(model.parameters()).device, **kwargs)

    def length(self, seq: int) -> int:
        return self._len[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, new) -> None:
        """Makes room for `new` tokens a sequence (one number for all, or one a
        sequence) and counts them: the next step's tokens.  Raises, with nothing
        changed, where a sequence would pass max_seq_len or the pool runs out."""
        uniform = isinstance(new, int)
        new = [new] * self.max_seqs if uniform else [int(n) for n in new]
        if len(new) != self.max_seqs or min(new) < 0:
            raise RuntimeError(f"new must hold {self.max_seqs} token counts >= 0")
        need = []
        for b, n in enumerate(new):
            if self._len[b] + n > self.max_seq_len:
                raise RuntimeError(f"sequence {b} would have {self._len[b] + n} tokens "
                                   f"(max_seq_len {self.max_seq_len})")
            need.append(max(0, -(-(self._len[b] + n) // self.page_size) - len(self._own[b])))
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages needed, {len(self._free)} free")
        for b, n in enumerate(new):
            for _ in range(need[b]):
                page = self._free.pop()
                self._table[b, len(self._own[b])] = page
                self._own[b].append(page)
            self._len[b] += n
        if any(need):
            self.page_table.copy_(self._table)
        if uniform:
            self.lengths.add_(new[0])
        else:
            self._upload_lengths()

    def _upload_lengths(self):
        self.lengths.copy_(torch.tensor(self._len, dtype=torch.int32))

    def release(self, seq: int) -> None:
        """Gives a sequence's pages back; its length is 0 again."""
        self._free.extend(reversed(self._own[seq]))
        self._own[seq] = []
        self._len[seq] = 0
        self._table[seq].fill_(-1)
        self.page_table.copy_(self._table)
        self._upload_lengths()

    def reset(self) -> None:
        for b in range(self.max_seqs):
            self._free.extend(reversed(self._own[b]))
            self._own[b] = []
        self._len = [0] * self.max_seqs
        self._table.fill_(-1)
        self.page_table.copy_(self._table)
        self.lengths.zero_()

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


class PagedStep:
    """The new tokens of a step, after cache.extend: rows [starts[b],
    starts[b + 1]) of the step are sequence b's (starts int32 on the device), or
    without starts the same number each."""

    def __init__(self, cache: PagedKVCache, starts: torch.Tensor | None = None):
        self.cache, self.starts = cache, starts
        self.page_table, self.lengths = cache.page_table, cache.lengths

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
    """Greedy generation over a paged cache: prompts of different lengths in one
    forward, then one captured graph's replay a token.

    Usage:
        wrapper = GLoRCQPagedWrapper(model, max_batch_size=4, max_seq_len=4096)
        outputs, seconds = wrapper.generate(prompts, max_new_tokens=128)
    """

    def __init__(self, model, max_batch_size=1, max_seq_len=4096, page_size=64, pages=None,
                 cache_dtype=torch.float8_e4m3fn):
        self.model = model
        self.max_batch_size, self.max_seq_len = max_batch_size, max_seq_len
        self.cache = PagedKVCache.for_model(model, max_batch_size, max_seq_len,
                                            page_size=page_size, pages=pages, dtype=cache_dtype)
        self.device = self.cache.device
        self.static_input_ids = torch.zeros(max_batch_size, dtype=torch.long, device=self.device)
        self.static_logits = None
        self.graph = None
        self.graph_stream = torch.cuda.Stream(device=self.device)
        self.last_timing = {}

    def _step(self):
        return paged_forward(self.model, self.static_input_ids, self.cache.lengths.long() - 1,
                             PagedStep(self.cache))

    @torch.no_grad()
    def capture_graph(self):
        """Warm-up steps on a side stream, then one decode step captured.  The
        cache is empty meanwhile (a token before position 0 is written nowhere)."""
        self.model.eval()
        self.cache.reset()
        s = torch.cuda.Stream(device=self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(s):
            for _ in range(3):
                self._step()
        torch.cuda.current_stream(self.device).wait_stream(s)
        torch.cuda.synchronize(self.device)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self.graph_stream):
            self.static_logits = self._step()

    @torch.no_grad()
    def prefill(self, prompts):
        """The prompts' forward into an empty cache -> the logits after each
        one's last token (batch, vocab)."""
        lens = [int(p.shape[0]) if p.dim() == 1 else 0 for p in prompts]
        if len(prompts) != self.max_batch_size or min(lens) < 1:
            raise RuntimeError(f"{self.max_batch_size} 1-D prompts of at least one token needed")
        self.cache.reset()
        self.cache.extend(lens)
        starts = torch.tensor([0] + lens).cumsum(0)
        pos = torch.cat([torch.arange(n) for n in lens])
        step = PagedStep(self.cache, starts.to(torch.int32).to(self.device))
        return paged_forward(self.model, torch.cat([p.to(self.device) for p in prompts]),
                             pos.to(self.device), step, last=(starts[1:] - 1).to(self.device))

    @torch.no_grad()
    def replay(self, input_ids):
        """One decode step: (batch,) ids, the sequences' next tokens -> the
        captured logits buffer (batch, vocab)."""
        if self.graph is None:
            raise RuntimeError("no captured step (capture_graph, which empties the cache)")
        if input_ids.shape != self.static_input_ids.shape:
            raise RuntimeError(f"input_ids must be ({self.max_batch_size},)")
        self.static_input_ids.copy_(input_ids)
        self.cache.extend(1)
        self.graph.replay()
        return self.static_logits

    @torch.no_grad()
    def generate(self, prompts, max_new_tokens=100):
        """Greedy generation from a list of 1-D prompts; returns (list of prompt
        + generated ids, seconds).  Sequences stop together, at max_new_tokens
        or where the longest reaches max_seq_len."""
        if self.graph is None:
            self.capture_graph()
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
