"""Operators of the paged key/value cache: appending a batch's new tokens
(head RMSNorm and rotary embedding on the way) and their causal attention over
the pages, for sequences of lengths of their own.  No reference counterpart:
its model path keeps one static cache a batch (inference/graph_wrapper.py:69-149).

A layer's cache is a pool of pages, in blocks of 16 tokens:

  k_pages  (pages, Hk, page, D)            fp16, or float8_e4m3fn codes
  v_pages  (pages, Hk, page // 16, D, 16)  of the same type (a block's 16
                                           values of a column side by side)
  k_scales, v_scales  (pages, Hk, page // 16) float8_e8m0fnu, with codes only:
                      a block's values are code * scale

page a power of two in [16, 1024], D 64 or 128.  page_table (B, n) int32 names
the pages of each sequence's positions, lengths (B,) int32 its tokens with the
new ones among them, and the new tokens are rows of q, k and v: rows
[starts[b], starts[b + 1]) are sequence b's (starts (B + 1,) int32), or without
starts T / B rows each.  All three are on the device and may change between
replays of a captured graph.  Rows behind starts[B] are left as they were.
"""

from __future__ import annotations

import ctypes
import struct
from array import array

import torch

from .. import _lib
from . import _require, _zeroed_buffer, workspace as _stream_scratch

BLOCK = 16  # tokens of a scale block

_FP8, _FP16, _E8M0 = torch.float8_e4m3fn, torch.float16, torch.float8_e8m0fnu

# The C ABI's parameter structures, packed in one go (a ctypes.Structure costs
# about 4 us of host time a call, this 1): glq_paged_cache, then the call's own.
_CACHE = "6P7q"
_append_params = struct.Struct(_CACHE + "Pq3P5q4PqPfi").pack
_attention_params = struct.Struct(_CACHE + "Pq2P2q2P2qfi").pack
_copy_params = struct.Struct("4Pq4Pq4q3Pq").pack
assert struct.calcsize(_CACHE + "Pq3P5q4PqPfi") == ctypes.sizeof(_lib.PagedAppendParams)
assert struct.calcsize(_CACHE + "Pq2P2q2P2qfi") == ctypes.sizeof(_lib.PagedAttentionParams)
assert struct.calcsize("4Pq4Pq4q3Pq") == ctypes.sizeof(_lib.PagedCopyParams)

# attention counters: (device index, stream handle) -> zero-filled uint8 tensor
_counters: dict = {}
_ws_bytes: dict = {}


def paged_cache_tensors(pages: int, kv_heads: int, head_dim: int = 128, page_size: int = 64,
                        dtype: torch.dtype = torch.float8_e4m3fn, device="cuda",
                        layers: int | None = None):
    """Zero-filled (k_pages, v_pages, k_scales, v_scales) of one layer's cache
    (the scales None for fp16 pages), or of `layers` layers, one behind the other
    (layers, pages, ...)."""
    if page_size < BLOCK or page_size > 1024 or page_size & (page_size - 1):
        raise RuntimeError(f"page_size must be a power of two in [16, 1024] (got {page_size})")
    if dtype not in (torch.float16, torch.float8_e4m3fn):
        raise RuntimeError(f"pages are float16 or float8_e4m3fn (got {dtype})")
    blocks = page_size // BLOCK
    size = 1 if dtype == torch.float8_e4m3fn else 2

    def zeros(*shape):  # (fp8 types have no fill of their own everywhere)
        return torch.zeros(*stack, *shape[:-1], shape[-1] * size, dtype=torch.uint8,
                           device=device).view(dtype)

    stack = () if layers is None else (layers,)
    k = zeros(pages, kv_heads, page_size, head_dim)
    v = zeros(pages, kv_heads, blocks, head_dim, BLOCK)
    if size == 2:
        return k, v, None, None
    ks, vs = (torch.zeros(*stack, pages, kv_heads, blocks, dtype=torch.uint8, device=device)
              .view(torch.float8_e8m0fnu) for _ in range(2))
    return k, v, ks, vs


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _check(t, name, dev, dtype) -> None:
    """A contiguous tensor of the pages' device and this type (the common case
    first: the checks are on the path of every decode step)."""
    if type(t) is torch.Tensor and t.get_device() == dev and t.dtype is dtype \
            and t.is_contiguous():
        return
    _require(t, name, dtype)
    if t.get_device() != dev:
        raise RuntimeError(f"{name} is on {t.device}, the pages on cuda:{dev}")


def _cache_view(k_pages, v_pages, k_scales, v_scales, page_table, lengths, starts, T):
    """The cache's checks: the C ABI's descriptor (its 13 values), the pages'
    device index, KV heads and head width."""
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() != 4:
        raise RuntimeError("k_pages must be (pages, Hk, page, D)")
    dtype, dev = k_pages.dtype, k_pages.get_device()
    if dtype is not _FP8 and dtype is not _FP16:
        raise RuntimeError(f"k_pages must be float16 or float8_e4m3fn (got {dtype})")
    if dev < 0:
        raise RuntimeError("k_pages must be a GPU tensor (glorcq_amd runs on the GPU only)")
    _check(k_pages, "k_pages", dev, dtype)
    _check(v_pages, "v_pages", dev, dtype)
    pages, Hk, page, D = k_pages.shape
    blocks = page // BLOCK
    if page < BLOCK or page > 1024 or page & (page - 1):
        raise RuntimeError(f"a page holds a power of two of tokens in [16, 1024] (got {page})")
    if v_pages.shape != (pages, Hk, blocks, D, BLOCK):
        raise RuntimeError(f"v_pages must be ({pages}, {Hk}, {blocks}, {D}, {BLOCK})")
    if dtype is _FP16:
        if k_scales is not None or v_scales is not None:
            raise RuntimeError("fp16 pages have no scales")
    else:
        for s, n in ((k_scales, "k_scales"), (v_scales, "v_scales")):
            if s is None:
                raise RuntimeError(f"8-bit pages need {n}")
            _check(s, n, dev, _E8M0)
            if s.shape != (pages, Hk, blocks):
                raise RuntimeError(f"{n} must be ({pages}, {Hk}, {blocks})")
    if not isinstance(page_table, torch.Tensor) or page_table.get_device() != dev \
            or page_table.dtype is not torch.int32 or page_table.dim() != 2:
        raise RuntimeError(f"page_table must be an int32 tensor (B, n) on cuda:{dev}")
    B, n = page_table.shape
    stride, one = page_table.stride()
    if B <= 1:
        stride = n
    if (one != 1 and n > 1) or stride < n:
        raise RuntimeError("page_table must have contiguous rows that do not overlap")
    _check(lengths, "lengths", dev, torch.int32)
    if lengths.shape != (B,):
        raise RuntimeError(f"lengths must be ({B},)")
    if starts is not None:
        _check(starts, "starts", dev, torch.int32)
        if starts.shape != (B + 1,):
            raise RuntimeError(f"starts must be ({B + 1},)")
    elif T % B if B else T:
        raise RuntimeError(f"{T} rows do not divide over {B} sequences (give starts)")
    return (k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scales), _ptr(v_scales),
            page_table.data_ptr(), lengths.data_ptr(), B, n, stride, pages, Hk, D, page), dev, Hk, D


def _rows(t, name, width, dev):
    """(T, width) rows, or (T, heads, D) ones, each contiguous: T, row stride."""
    if not isinstance(t, torch.Tensor) or t.get_device() != dev or t.dtype is not _FP16:
        raise RuntimeError(f"{name} must be a float16 tensor on the pages' GPU, cuda:{dev}")
    nd = t.dim()
    if nd == 3 and t.shape[1] * t.shape[2] == width:
        T, heads, D = t.shape
        stride, head, one = t.stride()
        if T and heads > 1 and head != D:
            raise RuntimeError(f"{name}'s heads must be contiguous within a row")
    elif nd == 2 and t.shape[1] == width:
        T = t.shape[0]
        stride, one = t.stride()
    else:
        raise RuntimeError(f"{name} must be (T, {width}) (got {tuple(t.shape)})")
    if one != 1 and T:
        raise RuntimeError(f"{name} must have contiguous rows")
    return T, stride if T > 1 else width


def _launch(fn, name, params, dev) -> None:
    if torch.cuda.current_device() == dev:
        rc = fn(params, _lib.stream_handle(torch.device("cuda", dev)))
    else:
        with torch.cuda.device(dev):
            rc = fn(params, _lib.stream_handle(torch.device("cuda", dev)))
    if rc:
        _lib.check(rc, name)


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor,
                 starts: torch.Tensor | None = None, k_scales: torch.Tensor | None = None,
                 v_scales: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, q: torch.Tensor | None = None,
                 q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
                 eps: float = 1e-6, q_out: torch.Tensor | None = None):
    """Writes the new tokens' k (T, Hk*D) and v into their positions' pages,
    one launch (glq_paged_append): each k head normalized (k_norm_w (D,), None:
    not) and rotated (cos/sin (T or 1, D), None: not) and rounded once to the
    pages' type; with q (T, Hq*D) -- or item-major (n, T, R), a batched GEMV's
    output over R-row slices -- its heads likewise, returned as q_out (T, Hq, D)
    fp16 (else None; q itself where its rows lie side by side, apart from all
    other inputs).  Rows of k, v and q may be slices of a wider matrix; a 3-D q whose last dimension is D is
    (T, Hq, D), never item-major.
    8-bit pages: a block's scale is the smallest power of two that takes its
    values to e4m3's 448; tokens that a block already had are scaled along when
    it grows.  Infinities and NaN are stored as NaN.  Pages that get tokens must
    belong to one sequence."""
    lib = _lib.load()
    if not isinstance(k, torch.Tensor):
        raise RuntimeError("k must be a tensor")
    T = k.shape[0] if k.dim() else 0
    cache, dev, Hk, D = _cache_view(k_pages, v_pages, k_scales, v_scales, page_table, lengths,
                                    starts, T)
    T, k_stride = _rows(k, "k", Hk * D, dev)
    Tv, v_stride = _rows(v, "v", Hk * D, dev)
    if Tv != T:
        raise RuntimeError(f"k has {T} rows, v {Tv}")
    if k_norm_w is not None:
        _check(k_norm_w, "k_norm_w", dev, _FP16)
        if k_norm_w.shape != (D,):
            raise RuntimeError(f"k_norm_w must be ({D},)")
    if (cos is None) != (sin is None):
        raise RuntimeError("cos and sin come together")
    cs_stride = 0
    if cos is not None:
        _check(cos, "cos", dev, _FP16)
        _check(sin, "sin", dev, _FP16)
        n = cos.numel()
        if cos.shape[-1:] != (D,) or sin.shape != cos.shape or (n != D and n != T * D):
            raise RuntimeError(f"cos and sin must hold 1 or {T} rows of {D}")
        cs_stride = D if n > D else 0
    Hq = item_rows = q_stride = 0
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() not in (2, 3):
            raise RuntimeError("q must be (T, Hq*D), (T, Hq, D) or item-major (n, T, R)")
        if q.dim() == 3 and q.shape[2] != D and q.shape[1] == T:  # item-major
            _check(q, "q", dev, _FP16)
            item_rows = q.shape[2]
            if item_rows % D:
                raise RuntimeError(f"q's items must be of whole heads ({D})")
            Hq = q.shape[0] * item_rows // D
        else:
            Hq = (q.shape[1] if q.dim() == 2 else q.shape[1] * q.shape[2]) // D
            Tq, q_stride = _rows(q, "q", Hq * D, dev)
            if Tq != T:
                raise RuntimeError(f"k has {T} rows, q {Tq}")
        if Hq == 0 or Hq % Hk:
            raise RuntimeError(f"q's heads ({Hq}) must be a multiple of the KV heads ({Hk})")
        if q_norm_w is not None:
            _check(q_norm_w, "q_norm_w", dev, _FP16)
            if q_norm_w.shape != (D,):
                raise RuntimeError(f"q_norm_w must be ({D},)")
        if q_out is None:
            q_out = q.new_empty((T, Hq, D))
        else:
            _check(q_out, "q_out", dev, _FP16)
            if q_out.numel() != T * Hq * D:
                raise RuntimeError(f"q_out must be ({T}, {Hq}, {D})")
    elif q_out is not None or q_norm_w is not None:
        raise RuntimeError("q_out and q_norm_w need a q")
    _launch(lib.glq_paged_append, "glq_paged_append", _append_params(
        *cache, _ptr(starts), T, k.data_ptr(), v.data_ptr(), _ptr(q), k_stride, v_stride, q_stride,
        Hq, item_rows, _ptr(q_norm_w), _ptr(k_norm_w), _ptr(cos), _ptr(sin), cs_stride,
        _ptr(q_out), eps, 0), dev)
    return q_out


def _workspace_bytes(B, T, Hq, Hk) -> tuple[int, int]:
    """Bytes of the counters and of the scratch, memoized (functions of the sizes)."""
    n = _ws_bytes.get((B, T, Hq, Hk))
    if n is None:
        lib = _lib.load()
        n = (lib.glq_paged_attention_counter_bytes(B, T, Hq, Hk),
             lib.glq_paged_attention_scratch_bytes(B, T, Hq, Hk))
        if min(n) < 0:
            raise RuntimeError("invalid paged attention shapes")
        _ws_bytes[(B, T, Hq, Hk)] = n
    return n


def _new_workspace(n, device) -> tuple[torch.Tensor, torch.Tensor]:
    return (torch.zeros(max(n[0], 256), dtype=torch.uint8, device=device),
            torch.empty(n[1], dtype=torch.uint8, device=device))


def paged_attention_workspace(q: torch.Tensor, k_pages: torch.Tensor, page_table: torch.Tensor):
    """A workspace (counters, zero between calls; scratch) for paged_attention
    at these sizes and smaller ones (keep it for the calls that follow; calls
    that share it must not overlap)."""
    return _new_workspace(_workspace_bytes(page_table.shape[0], q.shape[0],
                                           q.shape[1:].numel() // k_pages.shape[3],
                                           k_pages.shape[1]), k_pages.device)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, scale: float,
                    starts: torch.Tensor | None = None, k_scales: torch.Tensor | None = None,
                    v_scales: torch.Tensor | None = None, window: int = 0,
                    out: torch.Tensor | None = None,
                    workspace: tuple[torch.Tensor, torch.Tensor] | None = None,
                    sinks: int = 0) -> torch.Tensor:
    """Causal attention of the new tokens' q (T, Hq, D) fp16 (paged_append's
    result) over their sequences' pages -> (T, Hq*D) fp16 (glq_paged_attention).
    The token at position p attends to (p - window, p], or [0, p] with window
    0, and to the sequence's first `sinks` positions up to its own; pages that
    lie between need not be there (id -1).  scale may be 0 or negative.  Scores, softmax and sums are fp32, the
    weights in the product with V fp16.  `out` (apart from q): rows behind
    starts[B] keep what they held.  `workspace`: from paged_attention_workspace;
    None takes one of the stream's, or under graph capture one of the call's own,
    so that graphs may be replayed on several streams."""
    lib = _lib.load()
    if not isinstance(q, torch.Tensor) or q.dim() not in (2, 3):
        raise RuntimeError("q must be (T, Hq, D) or (T, Hq*D)")
    T = q.shape[0]
    cache, dev, Hk, D = _cache_view(k_pages, v_pages, k_scales, v_scales, page_table, lengths,
                                    starts, T)
    _check(q, "q", dev, _FP16)
    width = q.shape[1] if q.dim() == 2 else q.shape[1] * q.shape[2]
    if width % D or (q.dim() == 3 and q.shape[2] != D):
        raise RuntimeError(f"q must be (T, Hq, {D}) or (T, Hq*{D})")
    Hq = width // D
    if Hq == 0 or Hq % Hk:
        raise RuntimeError(f"q's heads ({Hq}) must be a multiple of the KV heads ({Hk})")
    if window < 0 or sinks < 0:
        raise RuntimeError("window and sinks must be >= 0 (0: none)")
    if out is None:
        out = q.new_empty((T, width))
    else:
        _check(out, "out", dev, _FP16)
        if out.dim() == 0 or out.shape[0] != T or out.numel() != T * width:
            raise RuntimeError(f"out must be ({T}, {width})")
    if workspace is None:
        n = _workspace_bytes(cache[6], T, Hq, Hk)
        if torch.cuda.is_current_stream_capturing():
            counters, scratch = _new_workspace(n, q.device)
        else:
            counters = _zeroed_buffer(_counters, q.device, n[0])
            scratch = _stream_scratch(q.device, n[1])
    else:
        counters, scratch = workspace
        _check(counters, "workspace's counters", dev, torch.uint8)
        _check(scratch, "workspace's scratch", dev, torch.uint8)
    _launch(lib.glq_paged_attention, "glq_paged_attention", _attention_params(
        *cache, _ptr(starts), T, q.data_ptr(), out.data_ptr(), Hq, window, counters.data_ptr(),
        scratch.data_ptr(), counters.numel(), scratch.numel(), scale, min(sinks, 0x7FFFFFFF)), dev)
    return out


def _pools(k_pages, v_pages, k_scales, v_scales, name):
    """Pools of one layer or of several: (the C ABI's 5 values, layers, KV heads,
    head width, page size, type, device index)."""
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() not in (4, 5):
        raise RuntimeError(f"{name}: k_pages must be ([layers,] pages, Hk, page, D)")
    dtype, dev = k_pages.dtype, k_pages.get_device()
    if dtype is not _FP8 and dtype is not _FP16:
        raise RuntimeError(f"{name}: k_pages must be float16 or float8_e4m3fn (got {dtype})")
    if dev < 0:
        raise RuntimeError(f"{name}: k_pages must be a GPU tensor (glorcq_amd runs on the GPU only)")
    _check(k_pages, "k_pages", dev, dtype)
    _check(v_pages, "v_pages", dev, dtype)
    *stack, pages, Hk, page, D = k_pages.shape
    blocks = (*stack, pages, Hk, page // BLOCK)
    if v_pages.shape != (*blocks, D, BLOCK):
        raise RuntimeError(f"{name}: v_pages must be {(*blocks, D, BLOCK)}")
    if dtype is _FP16:
        if k_scales is not None or v_scales is not None:
            raise RuntimeError(f"{name}: fp16 pages have no scales")
    else:
        for s, n in ((k_scales, "k_scales"), (v_scales, "v_scales")):
            if s is None:
                raise RuntimeError(f"{name}: 8-bit pages need {n}")
            _check(s, n, dev, _E8M0)
            if s.shape != blocks:
                raise RuntimeError(f"{name}: {n} must be {blocks}")
    return ((k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scales), _ptr(v_scales), pages),
            (stack[0] if stack else 1, Hk, D, page), dtype, dev)


def _numbers(x, name):
    try:
        if isinstance(x, torch.Tensor):
            if x.is_cuda:
                raise RuntimeError(f"{name} must be in host memory")
            x = x.tolist()
        return array("i", x)
    except (TypeError, OverflowError) as e:
        raise RuntimeError(f"{name} must hold page or token numbers: {e}") from None


def paged_copy(k_pages: torch.Tensor, v_pages: torch.Tensor, src, dst,
               k_scales: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
               tokens=None, to=None) -> None:
    """Copies pages in all layers at once, one launch for 256 of them
    (glq_paged_copy): page dst[i] becomes page src[i], the blocks of its first
    tokens[i] tokens (None: all of it).  Pools are one layer's, or those of
    several, one behind the other (layers, pages, ...); `to`: (k_pages, v_pages,
    k_scales, v_scales) of the same layers and heads that get the pages, None:
    the pools themselves.  src, dst and tokens are lists of numbers on the host
    (a captured copy copies the same pages at every replay); a page must not be
    written twice, nor written and read."""
    lib = _lib.load()
    pools, shape, dtype, dev = _pools(k_pages, v_pages, k_scales, v_scales, "pools")
    into = pools
    if to is not None:
        if len(to) != 4:
            raise RuntimeError("to must be (k_pages, v_pages, k_scales, v_scales)")
        into, *like = _pools(*to, "to")
        if like != [shape, dtype, dev]:
            raise RuntimeError("to must have the layers, heads, page size, type and GPU of the pools")
    src, dst = _numbers(src, "src"), _numbers(dst, "dst")
    tokens = None if tokens is None else _numbers(tokens, "tokens")
    n = len(src)
    if len(dst) != n or (tokens is not None and len(tokens) != n):
        raise RuntimeError("src, dst and tokens must be of one length")
    _launch(lib.glq_paged_copy, "glq_paged_copy", _copy_params(
        *pools, *into, *shape, src.buffer_info()[0], dst.buffer_info()[0],
        0 if tokens is None else tokens.buffer_info()[0], n), dev)
