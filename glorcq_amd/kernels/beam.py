"""Selection of beam search: the best continuations of each prompt over its
beams and the vocabulary.  No reference counterpart (its generation is greedy,
inference/graph_wrapper.py:69-149)."""

from __future__ import annotations

import ctypes
import struct

import torch

from .. import _lib
from . import _zeroed_buffer, workspace as _stream_scratch
from .paged import _check, _launch, _new_workspace

_FORMAT = "2P5q5P2q2i"
_params = struct.Struct(_FORMAT).pack
assert struct.calcsize(_FORMAT) == ctypes.sizeof(_lib.BeamSelectParams)
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
# counters: (device index, stream handle) -> zero-filled uint8 tensor
_counters: dict = {}
_ws_bytes: dict = {}


def beam_select(logits: torch.Tensor, scores: torch.Tensor, num: int):
    """The `num` best continuations of each prompt (glq_beam_select): logits
    (B * K, V) or (B, K, V) fp16, bf16 or fp32, whose rows may be slices of
    wider ones, scores (B, K) fp32 -> (scores (B, num) fp32, parents (B, num)
    int64, tokens (B, num) int64), by

        scores[b, k] + logits[b, k, v] - log(sum_u exp(logits[b, k, u]))

    in falling order, the lowest (k, v) first among equal ones; sums and
    comparisons are fp64.  Logits and scores of -inf come last, NaN (and +inf,
    which makes it) first.  K <= 64, num <= 128."""
    lib = _lib.load()
    if not isinstance(logits, torch.Tensor) or logits.dim() not in (2, 3) or not logits.is_cuda:
        raise RuntimeError("logits must be a GPU tensor (B * K, V) or (B, K, V)")
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None:
        raise RuntimeError(f"logits must be float16, bfloat16 or float32 (got {logits.dtype})")
    dev = logits.get_device()
    _check(scores, "scores", dev, torch.float32)
    if scores.dim() != 2:
        raise RuntimeError("scores must be (B, K)")
    B, K = scores.shape
    V = logits.shape[-1]
    if logits.shape[:-1] != (B * K,) and logits.shape[:-1] != (B, K):
        raise RuntimeError(f"logits must hold {B} x {K} rows (got {tuple(logits.shape)})")
    row = logits.stride(-2) if (B * K if logits.dim() == 2 else K) > 1 else \
        logits.stride(0) if B > 1 else V
    if (logits.stride(-1) != 1 and V > 1) or row < V or \
            (logits.dim() == 3 and B > 1 and K > 1 and logits.stride(0) != K * row):
        raise RuntimeError("logits must have contiguous rows, the same distance apart")
    need = _ws_bytes.get((B, K, V, num))
    if need is None:
        need = (max(lib.glq_beam_select_counter_bytes(B, K), 1),
                max(lib.glq_beam_select_scratch_bytes(B, K, V, num), 1))
        _ws_bytes[(B, K, V, num)] = need
    n = max(num, 0)
    out = scores.new_empty((B, n))
    parents, tokens = torch.empty((2, B, n), dtype=torch.int64, device=scores.device)
    if torch.cuda.is_current_stream_capturing():
        counters, scratch = _new_workspace(need, scores.device)
    else:
        counters = _zeroed_buffer(_counters, scores.device, need[0])
        scratch = _stream_scratch(scores.device, need[1])
    _launch(lib.glq_beam_select, "glq_beam_select", _params(
        logits.data_ptr(), scores.data_ptr(), B, K, V, row, num, out.data_ptr(),
        parents.data_ptr(), tokens.data_ptr(), counters.data_ptr(), scratch.data_ptr(),
        counters.numel(), scratch.numel(), dtype, 0), dev)
    return out, parents, tokens
