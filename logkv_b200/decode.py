"""Token-by-token decoding over one layer's cache, as the reference's attention module runs it.

The reference commits decode tokens in pairs (litgpt/model.py:1219-1247, :1330-1352): a token
with no pending token attends over the frozen cache plus itself (causal) and becomes pending;
the next token's single query attends over the cache plus [pending, itself] (``causal_tail=0``)
and the pair is committed with ``add_recent``, which flushes ``semantic_flush_granularity``
tokens when the window overflows (the first pair after a full window does).  ``LogKVDecoder``
keeps the pending token in preallocated two-token buffers, so a step allocates nothing.

``LogKVBeams`` runs beam search over such decoders, one per layer: it selects every step's
continuations and lets the rows of the beams that go on be taken over, in the decoders and their
caches.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import log_kv_chunk_attention
from .beam import beam_select


class LogKVDecoder:
    """Decode steps (one token per batch row) over ``cache``, with the reference's pending pairing."""

    def __init__(self, cache, scale: float):
        self.cache, self.scale = cache, float(scale)
        B, G = cache.batch_size, cache.n_groups
        dt, dev = cache.level_k.dtype, cache.level_k.device
        self._k = torch.zeros(B, G, 2, cache.k_dim, dtype=dt, device=dev)
        self._v = torch.zeros(B, G, 2, cache.v_dim, dtype=dt, device=dev)
        self._kr = torch.zeros(B, G, 2, cache.k_dim, dtype=dt, device=dev)
        self._pos = torch.zeros(B, 2, dtype=torch.int64, device=dev)
        self._ends = torch.zeros(B, 2, dtype=torch.uint8, device=dev)
        self._ends_host = None
        self._has_pos = False
        self.pending = False

    def reset(self) -> None:
        """Forget the pending token (the reference clears it with the cache, model.py:1180-1182)."""
        self.pending = False

    def reorder(self, index, *, window_from=None) -> None:
        """Row b takes over the old row index[b]: the cache's rows (``LogStructuredKVCache.reorder_batch``,
        same arguments) and the pending token's.  A pending token's span-end flags must be on the device
        (``span_ends_device``): host lists cannot follow a device index."""
        self._check_reorder(window_from)
        cache = self.cache
        index = cache._row_index(index)
        cache.reorder_batch(index, window_from=window_from)
        if not self.pending:
            return
        bufs = (self._k, self._v, self._kr, self._pos, self._ends)
        rows = (_lib.Rows * len(bufs))(*[_lib.Rows(t.data_ptr(), t.numel() * t.element_size() // cache.batch_size)
                                         for t in bufs])
        dev = self._k.device
        with _lib.on_device(dev):
            _lib.check(_lib.lib().logkv_reorder_rows(
                rows, len(bufs), cache.batch_size, index.data_ptr(), index.dtype == torch.int64,
                cache._read.status_ptr, _lib.stream_ptr(dev)), "logkv_reorder_rows")

    def _check_reorder(self, window_from=None) -> None:
        """Raise if reorder would be refused (but for its index)."""
        if self.pending and self._ends_host is not None:
            raise RuntimeError("reordering a pending token needs its span-end flags on the device (span_ends_device)")
        self.cache._check_reorder(window_from)

    def step(self, q, k, v, *, k_raw, input_pos=None, span_ends=None, span_ends_device=None, out=None):
        """One token: q [B, H, 1, D], k / v / k_raw [B, G, 1, D]; returns the attention output
        [B, H, 1, D].  ``input_pos`` ([1] or [B, 1]) and the span-end flags (``span_ends`` host
        rows of one flag, or ``span_ends_device`` uint8 [B, 1]) follow add_recent's contract."""
        if q.size(2) != 1 or k.size(2) != 1:
            raise ValueError("decode steps take one token per batch row")
        slot = 1 if self.pending else 0
        self._k[:, :, slot:slot + 1].copy_(k)
        self._v[:, :, slot:slot + 1].copy_(v)
        self._kr[:, :, slot:slot + 1].copy_(k_raw)
        if input_pos is not None:
            pos = input_pos.reshape(1, 1) if input_pos.dim() == 1 else input_pos
            self._pos[:, slot:slot + 1].copy_(pos)
        if slot == 0:
            self._has_pos = input_pos is not None
            self._ends_host = [list(r) for r in span_ends] if span_ends is not None else None
        elif (input_pos is not None) != self._has_pos:
            raise ValueError("input_pos must be given for both tokens of a pair or for neither")
        if span_ends_device is not None:
            self._ends[:, slot:slot + 1].copy_(span_ends_device)
        if not self.pending:
            y = log_kv_chunk_attention(self.cache, q, k, v, self.scale, 0.0, reuse_prefix=True, out=out)
            self.pending = True
            return y
        y = log_kv_chunk_attention(self.cache, q, self._k, self._v, self.scale, 0.0, causal_tail=0,
                                   reuse_prefix=True, out=out)
        ends = [a + list(b) for a, b in zip(self._ends_host, span_ends)] \
            if (self._ends_host is not None and span_ends is not None) else None
        if ends is None:
            ends = [[False, False] for _ in range(self.cache.batch_size)]
        self.cache.add_recent(self._k, self._v, k_raw=self._kr, input_pos=self._pos if self._has_pos else None,
                              span_ends=ends, span_ends_device=self._ends if span_ends_device is not None else None)
        self.pending = False
        return y


class LogKVBeams:
    """Beam search over ``decoders`` (one LogKVDecoder per layer) whose batch rows are `requests` x
    `beams`, a request's beams next to each other.

    After the prompt, ``fork()`` gives every beam its request's first row; then each step is the
    decoders' ``step`` for the beams' last tokens, the model's logits, and ``advance``.
    """

    def __init__(self, decoders, requests: int, beams: int):
        self.decoders = list(decoders)
        if not self.decoders or requests < 1 or beams < 1:
            raise ValueError("at least one decoder, request and beam")
        for d in self.decoders:
            if d.cache.batch_size != requests * beams:
                raise ValueError(f"a decoder's cache has {d.cache.batch_size} rows, not {requests} x {beams}")
        self.requests, self.beams = int(requests), int(beams)
        dev = self.decoders[0].cache.level_k.device
        self.scores = torch.full((self.requests, self.beams), float("-inf"), dtype=torch.float32, device=dev)
        self.scores[:, 0] = 0.0
        self._forked = None

    def fork(self) -> None:
        """Every beam takes over its request's first row; the scores start again (only that beam alive)."""
        for d in self.decoders:      # refused before any row has moved
            d._check_reorder()
        dev = self.scores.device
        first = torch.arange(self.requests, device=dev).mul_(self.beams).repeat_interleave(self.beams)
        for d in self.decoders:
            d.reorder(first)
        self.scores.fill_(float("-inf"))
        self.scores[:, 0] = 0.0
        # Until a cache's next flush (or reset) its rows of one request differ in the window behind this fill only.
        self._forked = [(d.cache._ladder_epoch, d.cache.recent_count) for d in self.decoders]

    def advance(self, logits):
        """Select the next tokens from the logits [requests, beams, V] (or [requests * beams, V]) of the
        beams' last tokens and let the rows follow.  Returns (tokens, rows), each [requests * beams]:
        the token of every row and the old row it continues; ``scores`` holds their scores.  The best
        continuation of a beam stays in the beam's row, so rows are in no order of score."""
        if logits.dim() == 2:
            logits = logits.view(self.requests, self.beams, -1)
        if logits.shape[:2] != (self.requests, self.beams):
            raise ValueError(f"logits must be [{self.requests}, {self.beams}, V], got {tuple(logits.shape)}")
        window = [None] * len(self.decoders)
        for i, d in enumerate(self.decoders):      # refused before any row has moved
            forked = self._forked[i] if self._forked else (None, 0)
            window[i] = forked[1] if forked[0] == d.cache._ladder_epoch else None
            d._check_reorder(window[i])
        scores, rows, tokens = beam_select(logits, self.scores, self.beams, keep_places=True)
        rows = rows.view(-1)
        for d, w in zip(self.decoders, window):
            d.reorder(rows, window_from=w)
        self.scores = scores
        return tokens.view(-1), rows
