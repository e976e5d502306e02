"""Beam search's selection over beams and vocabulary on the GPU (include/logkv_beam.h).

No reference counterpart: the reference decodes greedily or by sampling.  ``LogKVBeams``
(logkv_b200.decode) calls it and lets the caches' rows follow.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_native = None   # (beam call, function addresses) of the host binding, once a call has gone through
MAX_K, MAX_WIDTH = 128, 256   # LOGKV_BEAM_MAX_K, LOGKV_BEAM_MAX_WIDTH


def beam_select(logits, scores, k: int, *, keep_places: bool = False):
    """The k best continuations of every request: (scores [N, k] float32, rows [N, k] int64, tokens [N, k]
    int64).

    logits [N, W, V] (float32 or bf16; any strides of N and W) are the next-token logits of W beams per
    request, ``scores`` [N, W] float32 their log-probabilities so far.  A continuation (w, v) scores
    scores[w] + log_softmax(logits[w])[v]; best first, ties to the lower (w, v).  ``rows`` are flat beam
    rows n * W + w.  Logits of -inf are never chosen; a beam whose score is not finite, or that has a NaN
    or +inf logit or no finite one, offers nothing; places without a continuation get score -inf, token
    0 and row n * W + min(place, W - 1).

    Scores are ordered as float64 sums order them, within a beam by the logits themselves: beams whose
    scores come closer than float32 sums of exponentials tell apart are summed again in float64 (equal
    beams above all, which tie exactly; 115 us a beam of 151936).  Mask with -inf: finite masks are right
    too, but where few tokens are left the masked ones' ties are searched bit by bit, up to 70 times slower.

    ``keep_places`` (k == W): a beam's best continuation is put into the beam's own place and the others
    into the free places in order of score, so that as few rows as possible move when the caches follow
    (``LogStructuredKVCache.reorder_batch(rows.view(-1))``).

    k <= 128, W <= 256, N * W <= 65535.  The scratch is allocated per call, so calls on different streams,
    or captured graphs, never share it.  Forward-only.
    """
    global _native
    if _native is not None:      # checks, allocations and launch in the host binding; None: not covered there
        y = _native[0](_native[1], _native[2], logits, scores, k, keep_places)
        if y is not None:
            if type(y) is int:
                _lib.check(y, "logkv_beam_select")
            return y
    if logits.dim() != 3:
        raise ValueError(f"logits must be [N, W, V], got {tuple(logits.shape)}")
    N, W, V = logits.shape
    if logits.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"logits dtype {logits.dtype} is not supported (float32 or bfloat16)")
    if scores.shape != (N, W) or scores.dtype != torch.float32:
        raise ValueError(f"scores must be float32 [{N}, {W}], got {scores.dtype} {tuple(scores.shape)}")
    k = int(k)
    if not 1 <= k <= min(MAX_K, W * V):
        raise ValueError(f"k must be in [1, min({MAX_K}, W * V = {W * V})], got {k}")
    if keep_places and k != W:
        raise ValueError(f"keep_places takes as many continuations as beams (k = {k}, W = {W})")
    if W > MAX_WIDTH or N * W > 65535 or W * V >= (1 << 31) - 32:
        raise ValueError(f"beam shape outside the supported range (N={N}, W={W}, V={V})")
    if (logits.requires_grad or scores.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError("beam_select is forward-only")
    dev = logits.device
    if dev.type != "cuda" or scores.device != dev:
        raise ValueError("logits and scores must be CUDA tensors on one device")
    out_scores = scores.new_empty((N, k))
    out_rows, out_tokens = scores.new_empty((N, k), dtype=torch.int64), scores.new_empty((N, k), dtype=torch.int64)
    if N == 0:
        return out_scores, out_rows, out_tokens
    with _lib.on_device(dev):
        if V > 1 and logits.stride(2) != 1:
            logits = logits.contiguous()
        scores = scores.contiguous()
        lib = _lib.lib()
        _native = (_lib.host().beam, _lib.address("logkv_beam_select"), _lib.address("logkv_beam_workspace_bytes"))
        n = lib.logkv_beam_workspace_bytes(N, W, V, k)
        ws = scores.new_empty((n + 7) >> 3, dtype=torch.float64)
        args = _lib.BeamArgs(logits.data_ptr(), scores.data_ptr(), out_scores.data_ptr(), out_rows.data_ptr(),
                             out_tokens.data_ptr(), logits.stride(0), logits.stride(1),
                             _lib.DTYPE_CODES[logits.dtype], N, W, V, k, keep_places)
        _lib.check(lib.logkv_beam_select(ctypes.byref(args), ws.data_ptr(), n, _lib.stream_ptr(dev)),
                   "logkv_beam_select")
    return out_scores, out_rows, out_tokens
