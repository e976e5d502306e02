"""Penalties of repeated tokens, biases and grammar masks on next-token logits (include/logkv_logits.h).

No reference counterpart.  ``LogKVBeams`` (logkv_b200.decode) calls it in front of ``beam_select``.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_native = None    # (logits call, function address) of the host binding, once a call has gone through
MAX_BIAS = 1024   # LOGKV_LOGITS_MAX_BIAS
_INTS = (torch.int32, torch.int64)


def _number(name: str, value, lead, dev, positive: bool = False):
    """(float, None) of a scalar, or (0.0, [rows] float32 tensor)."""
    if isinstance(value, torch.Tensor) and value.dim():
        if value.shape != lead or value.dtype != torch.float32 or value.device != dev:
            raise ValueError(f"{name} must be a number or float32 {list(lead)} on {dev}, got {value.dtype} "
                             f"{tuple(value.shape)} on {value.device}")
        return 1.0, value.contiguous()
    try:
        held = ctypes.c_float(float(value)).value    # as the kernel has it
    except OverflowError:
        held = math.inf
    if not math.isfinite(held) or (positive and held <= 0):
        raise ValueError(f"{name} must be finite{' and positive' if positive else ''} in float32, got {str(value)[:40]}")
    return held, None


def _count(name: str, value, lead, dev):
    """(int, None) of a host number, or (0, [rows] integer tensor)."""
    if isinstance(value, torch.Tensor):
        if value.shape != lead or value.dtype not in _INTS or value.device != dev:
            raise ValueError(f"{name} must be an integer or int32 or int64 {list(lead)} on {dev}, got {value.dtype} "
                             f"{tuple(value.shape)} on {value.device}")
        return 0, value.contiguous()
    value = int(value)
    if value < 0:
        raise ValueError(f"{name} must not be negative, got {value}")
    return min(value, 2 ** 31 - 1), None


def _table(name: str, t, lead, dev, dtypes, shared: bool):
    """(rows x entries tensor with its entries next to each other, row stride) of [*lead, n], or [n] when `shared`."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.device != dev:
        raise ValueError(f"{name} must be a tensor of {' or '.join(str(d) for d in dtypes)} on {dev}")
    if shared and t.dim() == 1:
        return t.contiguous(), 0
    if t.dim() != len(lead) + 1 or t.shape[:-1] != lead:
        raise ValueError(f"{name} must be [{', '.join(str(n) for n in lead)}, n]{' or [n]' if shared else ''}, got "
                         f"{tuple(t.shape)}")
    t = t.flatten(0, -2)
    if t.size(1) > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _rows_overlap(x) -> bool:
    """Whether two rows of x ([..., V], V elements next to each other) have an element in common."""
    if not x.numel():
        return False
    V, reach = x.size(-1), x.size(-1)
    dims = sorted((s, n) for n, s in zip(x.shape[:-1], x.stride()) if n > 1)
    for s, n in dims:                    # rows inside one another, as a tensor's usually are
        if s < reach:
            break
        reach += (n - 1) * s
    else:
        return False
    at = torch.zeros(1, dtype=torch.int64, device="cpu")
    for s, n in dims:                    # otherwise where each of them starts
        at = (at[:, None] + s * torch.arange(n, device="cpu")).flatten()
    return bool((at.sort().values.diff() < V).any())


def adjust_logits(logits, *, history=None, lengths=None, prompt=0, repetition=1.0, presence=0.0, frequency=0.0,
                  bias=None, mask=None, out=None):
    """Next-token logits with penalties for repeated tokens, biases and a grammar mask, in this order.

    logits [N, W, V] (W beams per request) or [rows, V], float32 or bf16, any strides but the vocabulary's.  With
    c(v) the times that v occurs in a row's ``history`` behind its prompt:
      x / repetition where x > 0, else x * repetition      for v anywhere in the history;
      x - (frequency * c(v) + presence)                    for c(v) > 0;
      x + the sum of v's biases;  -inf where the mask says so.
    In float32, rounded once; what nothing touches is copied bit by bit.

    ``history`` [N, W, L] (or [rows, L]; int32 or int64) are the rows' tokens so far, of which ``lengths`` count (an
    int or integers [N, W]; None: all L) and the first ``prompt`` (likewise) are the prompt's; tokens outside
    [0, V) are passed over.  ``repetition`` (positive), ``presence`` and ``frequency`` are numbers or float32 [N, W].
    ``bias`` is (tokens, values): up to 1024 tokens [N, W, K] with float32 values, or [K] for all rows; a token's
    entries add up.  ``mask`` [N, W, ceil(V / 32)] int32 (or [ceil(V / 32)] for all rows) holds a bit per token, bit
    v % 32 of word v // 32, 0 for a banned one.  A row may be banned altogether: beam_select then takes nothing of it.

    Returns logits of the same shape and dtype, contiguous; ``out`` may be given, and may be ``logits`` itself.
    V <= 2^30, N * W <= 65535.  Forward-only.
    """
    global _native
    if _native is not None and out is None:   # checks, allocation and launch in the host binding; None: not covered there
        tokens, values = (None, None) if bias is None else bias
        y = _native[0](_native[1], logits, history, lengths, prompt, repetition, presence, frequency, tokens, values, mask)
        if y is not None:
            if type(y) is int:
                _lib.check(y, "logkv_adjust_logits")
            return y
    if logits.dim() not in (2, 3):
        raise ValueError(f"logits must be [N, W, V] or [rows, V], got {tuple(logits.shape)}")
    lead, V, dev = logits.shape[:-1], logits.size(-1), logits.device
    if logits.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"logits dtype {logits.dtype} is not supported (float32 or bfloat16)")
    rows = lead.numel()
    if V < 1 or V > 1 << 30 or rows > 65535:
        raise ValueError(f"logits shape outside the supported range ({rows} rows, V={V})")
    if torch.is_grad_enabled() and (logits.requires_grad or any(
            isinstance(t, torch.Tensor) and t.requires_grad for t in (repetition, presence, frequency, *(bias or ())))):
        raise NotImplementedError("adjust_logits is forward-only")
    a = _lib.LogitsArgs()
    a.repetition, reps = _number("repetition", repetition, lead, dev, True)
    a.presence, press = _number("presence", presence, lead, dev)
    a.frequency, freqs = _number("frequency", frequency, lead, dev)
    hist = lens = prompts = tokens = values = None
    if history is not None:
        hist, a.history_stride = _table("history", history, lead, dev, _INTS, False)
        L = hist.size(1)
        if L > 1 << 30:
            raise ValueError(f"a history of {L} tokens: at most 2^30")
        a.history_len, a.history_wide = L, hist.dtype == torch.int64
        a.length, lens = _count("lengths", L if lengths is None else lengths, lead, dev)
        a.prompt, prompts = _count("prompt", prompt, lead, dev)
        if lens is None and a.length > L:
            raise ValueError(f"lengths must be at most the history's {L} tokens, got {a.length}")
    elif lengths is not None:
        raise ValueError("lengths without a history")
    if bias is not None:
        tokens, values = bias
        tokens, a.bias_tokens_stride = _table("bias tokens", tokens, lead, dev, _INTS, True)
        values, a.bias_values_stride = _table("bias values", values, lead, dev, (torch.float32,), True)
        if tokens.size(-1) != values.size(-1) or tokens.dim() != values.dim():
            raise ValueError(f"bias tokens and values must have one shape, got {tuple(bias[0].shape)} and "
                             f"{tuple(bias[1].shape)}")
        if tokens.size(-1) > MAX_BIAS:
            raise ValueError(f"{tokens.size(-1)} biased tokens: at most {MAX_BIAS}")
        a.bias_count, a.bias_wide = tokens.size(-1), tokens.dtype == torch.int64
    if mask is not None:
        mask, a.mask_stride = _table("mask", mask, lead, dev, (torch.int32,), True)
        if mask.size(-1) != (V + 31) // 32:
            raise ValueError(f"mask must hold {(V + 31) // 32} words a row, got {mask.size(-1)}")
    if out is logits and _rows_overlap(logits):
        raise ValueError("logits adjusted in place must not share memory between rows")
    if dev.type != "cuda":
        raise ValueError("logits must be a CUDA tensor")
    if out is None:
        out = logits.new_empty(logits.shape)
    elif out is not logits and (out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev
                                or not out.is_contiguous()):
        raise ValueError(f"out must be logits itself, or contiguous {list(logits.shape)} {logits.dtype} on {dev}")
    elif out is not logits and out.untyped_storage().data_ptr() == logits.untyped_storage().data_ptr() and rows:
        raise ValueError("out must be logits itself or have memory of its own")
    if not rows:
        return out
    with _lib.on_device(dev):
        x = logits
        if V > 1 and x.stride(-1) != 1:
            if out is logits:
                raise ValueError("logits adjusted in place must have their vocabulary contiguous")
            x = x.contiguous()
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        a.logits, a.out, a.dtype, a.rows, a.vocab = x.data_ptr(), out.data_ptr(), _lib.DTYPE_CODES[x.dtype], rows, V
        a.width = lead[-1]
        a.w_stride, a.out_w_stride = x.stride(-2), out.stride(-2)
        if len(lead) == 2:
            a.n_stride, a.out_n_stride = x.stride(0), out.stride(0)
        a.history, a.lengths, a.prompts = ptr(hist), ptr(lens), ptr(prompts)
        a.lengths_wide = lens is not None and lens.dtype == torch.int64
        a.prompts_wide = prompts is not None and prompts.dtype == torch.int64
        a.repetitions, a.presences, a.frequencies = ptr(reps), ptr(press), ptr(freqs)
        a.bias_tokens, a.bias_values, a.mask = ptr(tokens), ptr(values), ptr(mask)
        _native = (_lib.host().logits, _lib.address("logkv_adjust_logits"))
        _lib.check(_lib.lib().logkv_adjust_logits(ctypes.byref(a), _lib.stream_ptr(dev)), "logkv_adjust_logits")
    return out
