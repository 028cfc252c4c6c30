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

import torch

from .. import _lib
from . import _require, _zeroed_buffer

BLOCK = 16  # tokens of a scale block

# attention workspaces: (device index, stream handle) -> zero-filled uint8 tensor
_workspaces: dict = {}


def paged_cache_tensors(pages: int, kv_heads: int, head_dim: int = 128, page_size: int = 64,
                        dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
    """Zero-filled (k_pages, v_pages, k_scales, v_scales) of one layer's cache
    (the scales None for fp16 pages)."""
    if page_size < BLOCK or page_size > 1024 or page_size & (page_size - 1):
        raise RuntimeError(f"page_size must be a power of two in [16, 1024] (got {page_size})")
    if dtype not in (torch.float16, torch.float8_e4m3fn):
        raise RuntimeError(f"pages are float16 or float8_e4m3fn (got {dtype})")
    blocks = page_size // BLOCK
    size = 1 if dtype == torch.float8_e4m3fn else 2

    def zeros(*shape):  # (fp8 types have no fill of their own everywhere)
        return torch.zeros(*shape[:-1], shape[-1] * size, dtype=torch.uint8,
                           device=device).view(dtype)

    k = zeros(pages, kv_heads, page_size, head_dim)
    v = zeros(pages, kv_heads, blocks, head_dim, BLOCK)
    if size == 2:
        return k, v, None, None
    ks, vs = (torch.zeros(pages, kv_heads, blocks, dtype=torch.uint8, device=device)
              .view(torch.float8_e8m0fnu) for _ in range(2))
    return k, v, ks, vs


def _same_device(dev, named) -> None:
    for t, n in named:
        if t is not None and t.device != dev:
            raise RuntimeError(f"{n} is on {t.device}, the pages on {dev}")


def _cache_view(k_pages, v_pages, k_scales, v_scales, page_table, lengths, starts, T):
    """The C ABI's cache descriptor, checked; (descriptor, heads, head_dim)."""
    _require(k_pages, "k_pages")
    if k_pages.dtype not in (torch.float16, torch.float8_e4m3fn):
        raise RuntimeError(f"k_pages must be float16 or float8_e4m3fn (got {k_pages.dtype})")
    _require(v_pages, "v_pages", k_pages.dtype)
    if k_pages.dim() != 4:
        raise RuntimeError("k_pages must be (pages, Hk, page, D)")
    pages, Hk, page, D = k_pages.shape
    if page < BLOCK or page > 1024 or page & (page - 1):
        raise RuntimeError(f"a page holds a power of two of tokens in [16, 1024] (got {page})")
    if tuple(v_pages.shape) != (pages, Hk, page // BLOCK, D, BLOCK):
        raise RuntimeError(f"v_pages must be ({pages}, {Hk}, {page // BLOCK}, {D}, {BLOCK})")
    if k_pages.dtype == torch.float16:
        if k_scales is not None or v_scales is not None:
            raise RuntimeError("fp16 pages have no scales")
    else:
        for s, n in ((k_scales, "k_scales"), (v_scales, "v_scales")):
            if s is None:
                raise RuntimeError(f"8-bit pages need {n}")
            _require(s, n, torch.float8_e8m0fnu)
            if tuple(s.shape) != (pages, Hk, page // BLOCK):
                raise RuntimeError(f"{n} must be ({pages}, {Hk}, {page // BLOCK})")
    if not isinstance(page_table, torch.Tensor) or not page_table.is_cuda \
            or page_table.dtype != torch.int32 or page_table.dim() != 2 \
            or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise RuntimeError("page_table must be a GPU int32 tensor (B, n) of contiguous rows")
    _require(lengths, "lengths", torch.int32)
    B, n = page_table.shape
    if tuple(lengths.shape) != (B,):
        raise RuntimeError(f"lengths must be ({B},)")
    if starts is not None:
        _require(starts, "starts", torch.int32)
        if tuple(starts.shape) != (B + 1,):
            raise RuntimeError(f"starts must be ({B + 1},)")
    elif T % B if B else T:
        raise RuntimeError(f"{T} rows do not divide over {B} sequences (give starts)")
    _same_device(k_pages.device, ((v_pages, "v_pages"), (k_scales, "k_scales"),
                                  (v_scales, "v_scales"), (page_table, "page_table"),
                                  (lengths, "lengths"), (starts, "starts")))
    stride = page_table.stride(0) if B > 1 else n
    if stride < n:
        raise RuntimeError("page_table rows overlap")
    return _lib.PagedCache(
        k_pages.data_ptr(), v_pages.data_ptr(), _lib.ptr(k_scales), _lib.ptr(v_scales),
        page_table.data_ptr(), lengths.data_ptr(), B, n, stride, pages, Hk, D, page), Hk, D


def _rows(t, name, width):
    """(T, ...) rows of `width` values, each contiguous: (T, row stride)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float16:
        raise RuntimeError(f"{name} must be a GPU float16 tensor")
    if t.dim() == 3 and t.shape[1] * t.shape[2] == width:  # (T, heads, D)
        if t.numel() and t.shape[1] > 1 and t.stride(1) != t.shape[2]:
            raise RuntimeError(f"{name}'s heads must be contiguous within a row")
    elif t.dim() != 2 or t.shape[1] != width:
        raise RuntimeError(f"{name} must be (T, {width}) (got {tuple(t.shape)})")
    if t.stride(-1) != 1 and t.numel():
        raise RuntimeError(f"{name} must have contiguous rows")
    T = t.shape[0]
    return T, t.stride(0) if T > 1 else width


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor,
                 starts: torch.Tensor | None = None, k_scales: torch.Tensor | None = None,
                 v_scales: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, q: torch.Tensor | None = None,
                 q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
                 eps: float = 1e-6, q_out: torch.Tensor | None = None):
    """Writes the new tokens' k (T, Hk*D) and v into their positions' pages,
    one launch (glq_paged_append): each k head normalized (k_norm_w (D,), None:
    not) and rotated (cos/sin (T or 1, D), None: not) in fp32 and rounded once
    to the pages' type; with q (T, Hq*D) -- or item-major (n, T, R), a batched
    GEMV's output over R-row slices -- its heads likewise, returned as q_out
    (T, Hq, D) fp16 (else None).  Rows of k, v and q may be slices of a wider
    matrix.  8-bit pages: a block's scale is the smallest power of two that
    takes its values to e4m3's 448; tokens that a block already had are scaled
    along when it grows.  Infinities and NaN are stored as NaN."""
    lib = _lib.load()
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() != 4:
        raise RuntimeError("k_pages must be (pages, Hk, page, D)")
    width = k_pages.shape[1] * k_pages.shape[3]
    T, k_stride = _rows(k, "k", width)
    Tv, v_stride = _rows(v, "v", width)
    if Tv != T:
        raise RuntimeError(f"k has {T} rows, v {Tv}")
    view, Hk, D = _cache_view(k_pages, v_pages, k_scales, v_scales, page_table, lengths, starts, T)
    for w, n in ((q_norm_w, "q_norm_w"), (k_norm_w, "k_norm_w")):
        if w is not None:
            _require(w, n, torch.float16)
            if tuple(w.shape) != (D,):
                raise RuntimeError(f"{n} must be ({D},)")
    if (cos is None) != (sin is None):
        raise RuntimeError("cos and sin come together")
    cs_stride = 0
    if cos is not None:
        _require(cos, "cos", torch.float16)
        _require(sin, "sin", torch.float16)
        if cos.shape[-1] != D or sin.shape != cos.shape or cos.numel() // D not in (1, T):
            raise RuntimeError(f"cos and sin must hold 1 or {T} rows of {D}")
        cs_stride = D if cos.numel() // D > 1 else 0
    Hq = item_rows = q_stride = 0
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() not in (2, 3):
            raise RuntimeError("q must be (T, Hq*D), (T, Hq, D) or item-major (n, T, R)")
        if q.dim() == 3 and q.shape[2] != D and q.shape[1] == T:  # item-major
            _require(q, "q", torch.float16)
            item_rows = q.shape[2]
            if item_rows % D:
                raise RuntimeError(f"q's items must be of whole heads ({D})")
            Hq = q.shape[0] * item_rows // D
        else:
            Hq = q.shape[1:].numel() // D
            Tq, q_stride = _rows(q, "q", Hq * D)
            if Tq != T:
                raise RuntimeError(f"k has {T} rows, q {Tq}")
        if Hq == 0 or Hq % Hk:
            raise RuntimeError(f"q's heads ({Hq}) must be a multiple of the KV heads ({Hk})")
        if q_out is None:
            q_out = torch.empty(T, Hq, D, dtype=torch.float16, device=k.device)
        else:
            _require(q_out, "q_out", torch.float16)
            if q_out.numel() != T * Hq * D:
                raise RuntimeError(f"q_out must be ({T}, {Hq}, {D})")
    elif q_out is not None or q_norm_w is not None:
        raise RuntimeError("q_out and q_norm_w need a q")
    dev = k_pages.device
    _same_device(dev, ((k, "k"), (v, "v"), (q, "q"), (cos, "cos"), (sin, "sin"),
                       (q_norm_w, "q_norm_w"), (k_norm_w, "k_norm_w"), (q_out, "q_out")))
    with torch.cuda.device(dev):
        _lib.check(lib.glq_paged_append(
            ctypes.byref(view), _lib.ptr(starts), T, k.data_ptr(), k_stride, v.data_ptr(),
            v_stride, _lib.ptr(q), Hq, q_stride, item_rows, _lib.ptr(q_norm_w),
            _lib.ptr(k_norm_w), float(eps), _lib.ptr(cos), _lib.ptr(sin), cs_stride,
            _lib.ptr(q_out), _lib.stream_handle(dev)), "glq_paged_append")
    return q_out


def paged_attention_workspace(q: torch.Tensor, k_pages: torch.Tensor,
                              page_table: torch.Tensor) -> torch.Tensor:
    """A zeroed workspace for paged_attention at these shapes (keep it for the
    calls that follow: every call leaves its counters zero, and calls that
    share it must not overlap)."""
    D = k_pages.shape[3]
    n = _workspace_bytes(page_table.shape[0], q.shape[0], q.shape[1:].numel() // D,
                         k_pages.shape[1], D)
    return torch.zeros(n, dtype=torch.uint8, device=k_pages.device)


def _workspace_bytes(B, T, Hq, Hk, D) -> int:
    n = _lib.load().glq_paged_attention_workspace_bytes(B, T, Hq, Hk, D)
    if n < 0:
        raise RuntimeError("invalid paged attention shapes")
    return max(int(n), 256)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, scale: float,
                    starts: torch.Tensor | None = None, k_scales: torch.Tensor | None = None,
                    v_scales: torch.Tensor | None = None, window: int = 0,
                    out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the new tokens' q (T, Hq, D) fp16 (paged_append's
    result) over their sequences' pages -> (T, Hq*D) fp16 (glq_paged_attention).
    The token at position p attends to (p - window, p], or [0, p] with window
    0.  `out`: rows behind starts[B] keep what they held.  `workspace`: from
    paged_attention_workspace; None takes one of the stream's, or under graph
    capture one of the call's own, so that graphs may be replayed on several
    streams."""
    lib = _lib.load()
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() != 4:
        raise RuntimeError("k_pages must be (pages, Hk, page, D)")
    _require(q, "q", torch.float16)
    D = k_pages.shape[3]
    if q.dim() not in (2, 3) or (q.dim() == 3 and q.shape[2] != D) or q.shape[1:].numel() % D:
        raise RuntimeError(f"q must be (T, Hq, {D}) or (T, Hq*{D})")
    T, Hq = q.shape[0], q.shape[1:].numel() // D
    view, Hk, D = _cache_view(k_pages, v_pages, k_scales, v_scales, page_table, lengths, starts, T)
    if Hq == 0 or Hq % Hk:
        raise RuntimeError(f"q's heads ({Hq}) must be a multiple of the KV heads ({Hk})")
    if window < 0:
        raise RuntimeError("window must be >= 0 (0: none)")
    dev = k_pages.device
    if out is None:
        out = torch.empty(T, Hq * D, dtype=torch.float16, device=dev)
    else:
        _require(out, "out", torch.float16)
        if out.numel() != T * Hq * D or out.shape[0] != T:
            raise RuntimeError(f"out must be ({T}, {Hq * D})")
    _same_device(dev, ((q, "q"), (out, "out"), (workspace, "workspace")))
    with torch.cuda.device(dev):
        if workspace is None:
            n = _workspace_bytes(view.seqs, T, Hq, Hk, D)
            if torch.cuda.is_current_stream_capturing():
                workspace = torch.zeros(n, dtype=torch.uint8, device=dev)
            else:
                workspace = _zeroed_buffer(_workspaces, dev, n)
        else:
            _require(workspace, "workspace", torch.uint8)
        _lib.check(lib.glq_paged_attention(
            ctypes.byref(view), _lib.ptr(starts), T, q.data_ptr(), Hq, float(scale), int(window),
            out.data_ptr(), workspace.data_ptr(), workspace.numel(), _lib.stream_handle(dev)),
            "glq_paged_attention")
    return out
