"""Token-by-token decoding over one layer's cache, as the reference's attention module runs it.

The reference commits decode tokens in pairs (litgpt/model.py:1219-1247, :1330-1352): a token
with no pending token attends over the frozen cache plus itself (causal) and becomes pending;
the next token's single query attends over the cache plus [pending, itself] (``causal_tail=0``)
and the pair is committed with ``add_recent``, which flushes ``semantic_flush_granularity``
tokens when the window overflows (the first pair after a full window does).  ``LogKVDecoder``
keeps the pending token in preallocated two-token buffers, so a step allocates nothing.

``LogKVBeams`` runs beam search over such decoders, one per layer: its steps read what a request's beams
share once, and it selects every step's continuations and lets the rows of the beams that go on be taken
over, in the decoders and their caches.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, rotary
from .attention import _MAX_QUERY_ROWS, log_kv_chunk_attention, log_kv_shared_attention
from .beam import beam_select
from .logits import adjust_logits


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

    def step(self, q, k, v, *, k_raw, input_pos=None, span_ends=None, span_ends_device=None, out=None, shared=None):
        """One token: q [B, H, 1, D], k / v / k_raw [B, G, 1, D]; returns the attention output
        [B, H, 1, D].  ``input_pos`` ([1] or [B, 1]) and the span-end flags (``span_ends`` host
        rows of one flag, or ``span_ends_device`` uint8 [B, 1]) follow add_recent's contract.
        ``shared`` (beams, window_from): the rows share a prefix as log_kv_shared_attention has it."""
        if q.size(2) != 1 or k.size(2) != 1:
            raise ValueError("decode steps take one token per batch row")
        slot = self._slot(shared)
        self._k[:, :, slot:slot + 1].copy_(k)
        self._v[:, :, slot:slot + 1].copy_(v)
        self._kr[:, :, slot:slot + 1].copy_(k_raw)
        if input_pos is not None:
            pos = input_pos.reshape(1, 1) if input_pos.dim() == 1 else input_pos
            self._pos[:, slot:slot + 1].copy_(pos)
        self._keep(slot, input_pos, span_ends)
        if span_ends_device is not None:
            self._ends[:, slot:slot + 1].copy_(span_ends_device)
        return self._finish(slot, q, k, v, span_ends, span_ends_device, out, shared)

    def step_raw(self, q, k_raw, v, *, input_pos=None, layout: str = "half", span_ends=None, span_ends_device=None,
                 out=None, shared=None):
        """``step`` of unrotated queries and keys, q [B, H, 1, D] and k_raw / v [B, G, 1, D] in the cache dtype, any
        strides: one kernel rotates them at ``input_pos`` ([1] or [B, 1] integers; None: the position that continues
        the sequence) and puts the token into the pending slot.  ``layout`` is log_kv_rotate's, all else step's."""
        mode = rotary.check_layout(layout)
        cache = self.cache
        slot = self._slot(shared)
        at = slice(slot, slot + 1)
        call = rotary.native(cache)
        if call is not None and q.dim() == 4 and q.size(2) == 1 and (slot == 0 or (input_pos is not None) == self._has_pos):
            # A call like one before: checks and launch in the host binding; None: not covered there.
            turned = call.append(call.fn, call.rope, call.status, self._k, self._kr, self._v, self._pos, self._ends, k_raw,
                                 v, input_pos, span_ends_device, cache.token_count + slot, slot, mode, q)
            if turned is not None:
                if type(turned) is int:
                    _lib.check(turned, "logkv_rotate")
                self._keep(slot, input_pos, span_ends)
                return self._finish(slot, turned, self._k[:, :, at], self._v[:, :, at], span_ends, span_ends_device, out,
                                    shared)
        B, G, D, dt, dev = cache.batch_size, cache.n_groups, cache.k_dim, self._k.dtype, self._k.device
        if q.dim() != 4 or q.size(1) < 1 or q.size(1) % G or q.shape != (B, q.size(1), 1, D) or q.dtype != dt:
            raise ValueError(f"q must be [{B}, H, 1, {D}] in the cache dtype, H a multiple of {G}")
        for name, t in (("k_raw", k_raw), ("v", v)):
            if t.shape != (B, G, 1, D) or t.dtype != dt:
                raise ValueError(f"{name} must be [{B}, {G}, 1, {D}] in the cache dtype, got {tuple(t.shape)} {t.dtype}")
        if q.device != dev or k_raw.device != dev or v.device != dev:
            raise ValueError(f"q, k_raw and v must be on the cache's device {dev}")
        if torch.is_grad_enabled() and (q.requires_grad or k_raw.requires_grad or v.requires_grad):
            raise NotImplementedError("logkv_b200 attention is forward-only")
        positions = rotary.check_positions(cache, input_pos, 1)
        ends = span_ends_device
        if ends is not None:
            if tuple(ends.shape) != (B, 1):
                raise ValueError("AlphaLogKV span boundaries must match the input batch and token count")
            ends = ends.to(device=dev, dtype=torch.uint8)
        self._keep(slot, positions, span_ends)
        k, v1 = self._k[:, :, at], self._v[:, :, at]
        with _lib.on_device(dev):
            turned = q.new_empty((B, q.size(1), 1, D))
            rotary.launch(cache, [(rotary.last_contiguous(q), turned),
                                  (rotary.last_contiguous(k_raw), k, self._kr[:, :, at]),
                                  (rotary.last_contiguous(v), None, v1)], positions, cache.token_count + slot, mode,
                          positions_out=None if positions is None else self._pos[:, at], ends=ends,
                          ends_out=None if ends is None else self._ends[:, at])
        return self._finish(slot, turned, k, v1, span_ends, span_ends_device, out, shared)

    def _slot(self, shared) -> int:
        """The slot of the next token; raises if the attention would refuse ``shared``."""
        if shared is not None:
            beams, window_from = shared
            if beams < 1 or self.cache.batch_size % beams or not 0 <= window_from <= self.cache.recent_count:
                raise ValueError(f"shared must be (beams, window_from) with beams a divisor of {self.cache.batch_size} "
                                 f"and window_from in [0, {self.cache.recent_count}], got {shared}")
        return 1 if self.pending else 0

    def _keep(self, slot: int, input_pos, span_ends) -> None:
        """What the host keeps of a pair's tokens."""
        if slot == 0:
            self._has_pos = input_pos is not None
            self._ends_host = [list(r) for r in span_ends] if span_ends is not None else None
        elif (input_pos is not None) != self._has_pos:
            raise ValueError("input_pos must be given for both tokens of a pair or for neither")

    def _attend(self, q, k, v, causal_tail, out, shared):
        if shared is None:
            return log_kv_chunk_attention(self.cache, q, k, v, self.scale, 0.0, causal_tail=causal_tail,
                                          reuse_prefix=True, out=out)
        return log_kv_shared_attention(self.cache, q, k, v, self.scale, beams=shared[0], window_from=shared[1],
                                       causal_tail=causal_tail, out=out)

    def _finish(self, slot: int, q, k, v, span_ends, span_ends_device, out, shared):
        """Attention of the token in `slot`, and the pair's commit."""
        if slot == 0:
            y = self._attend(q, k, v, None, out, shared)
            self.pending = True
            return y
        y = self._attend(q, self._k, self._v, 0, out, shared)
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

    After the prompt, ``fork()`` gives every beam its request's first row; then each step is ``step`` of every
    layer (or the decoders' own) for the beams' last tokens, the model's logits, and ``advance``.

    ``penalties``: {"repetition": .., "presence": .., "frequency": ..} (any of them, as adjust_logits takes them)
    for tokens that a beam repeats; the beams' tokens so far are then kept here and follow the beams.
    """

    def __init__(self, decoders, requests: int, beams: int, *, penalties: dict | None = None):
        self.decoders = list(decoders)
        if not self.decoders or requests < 1 or beams < 1:
            raise ValueError("at least one decoder, request and beam")
        for d in self.decoders:
            if d.cache.batch_size != requests * beams:
                raise ValueError(f"a decoder's cache has {d.cache.batch_size} rows, not {requests} x {beams}")
        if penalties is not None and set(penalties) - {"repetition", "presence", "frequency"}:
            raise ValueError(f"penalties are repetition, presence and frequency, got {sorted(penalties)}")
        self.requests, self.beams = int(requests), int(beams)
        self.penalties = None if penalties is None else dict(penalties)
        dev = self.decoders[0].cache.level_k.device
        self.scores = torch.full((self.requests, self.beams), float("-inf"), dtype=torch.float32, device=dev)
        self.scores[:, 0] = 0.0
        self._forked = None
        self._tokens = None          # [rows, capacity] int32: the prompt's and the beams' tokens (with penalties)
        self._prompt = self._length = 0

    def fork(self, prompt=None) -> None:
        """Every beam takes over its request's first row; the scores start again (only that beam alive).
        ``prompt`` ([requests, L] integers on the device, shorter ones padded with -1): the tokens that a
        repetition penalty counts besides the beams' own."""
        rows = self.requests * self.beams
        if prompt is not None:
            if self.penalties is None:
                raise ValueError("a prompt is kept for penalties only")
            if prompt.dim() != 2 or prompt.size(0) != self.requests or prompt.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"prompt must be integers [{self.requests}, L], got {prompt.dtype} {tuple(prompt.shape)}")
            if prompt.device != self.scores.device:
                raise ValueError(f"prompt must be on {self.scores.device}, got {prompt.device}")
        for d in self.decoders:      # refused before any row has moved
            d._check_reorder()
        dev = self.scores.device
        first = torch.arange(self.requests, device=dev).mul_(self.beams).repeat_interleave(self.beams)
        for d in self.decoders:
            d.reorder(first)
        self.scores.fill_(float("-inf"))
        self.scores[:, 0] = 0.0
        if self.penalties is not None:
            self._prompt = self._length = 0 if prompt is None else prompt.size(1)
            self._tokens = torch.empty(rows, (self._length + 256) // 4 * 4, dtype=torch.int32, device=dev)
            if prompt is not None:
                self._tokens[:, :self._length] = prompt.repeat_interleave(self.beams, 0)
        # Until a cache's next flush (or reset) its rows of one request differ in the window behind this fill only.
        self._forked = [(d.cache._ladder_epoch, d.cache.recent_count) for d in self.decoders]

    def _window_from(self, i: int):
        """The window rows that decoder i's rows of a request share with the packed prefix, None: not even that."""
        forked = self._forked[i] if self._forked else (None, 0)
        return forked[1] if forked[0] == self.decoders[i].cache._ladder_epoch else None

    def step(self, layer: int, q, k_raw, v, *, input_pos=None, layout: str = "half", span_ends_device=None, out=None):
        """``LogKVDecoder.step_raw`` of layer ``layer`` for the beams' last tokens: q [rows, H, 1, D], k_raw and v
        [rows, G, 1, D], unrotated.  Until the cache's next flush after ``fork`` the keys that a request's beams
        share are read once for all of them."""
        d, w = self.decoders[layer], self._window_from(layer)
        shared = (self.beams, w) if w is not None and self.beams > 1 else None
        rf = q.size(1) // d.cache.n_groups if q.dim() == 4 else 1
        if shared is None and rf and (rf & (rf - 1) or rf > _MAX_QUERY_ROWS[d._k.dtype]):
            shared = (1, 0)      # heads per group that log_kv_chunk_attention does not take
        return d.step_raw(q, k_raw, v, input_pos=input_pos, layout=layout, span_ends_device=span_ends_device, out=out,
                          shared=shared)

    def advance(self, logits, *, bias=None, mask=None):
        """Select the next tokens from the logits [requests, beams, V] (or [requests * beams, V]) of the
        beams' last tokens and let the rows follow.  Returns (tokens, rows), each [requests * beams]:
        the token of every row and the old row it continues; ``scores`` holds their scores.  The best
        continuation of a beam stays in the beam's row, so rows are in no order of score.

        The logits are adjusted first where there are penalties, a ``bias`` or a grammar ``mask`` (adjust_logits';
        leading dimensions [requests, beams] or none).  With penalties a step cannot be captured in a graph: the
        number of tokens so far is the host's."""
        if logits.dim() == 2:
            logits = logits.view(self.requests, self.beams, -1)
        if logits.shape[:2] != (self.requests, self.beams):
            raise ValueError(f"logits must be [{self.requests}, {self.beams}, V], got {tuple(logits.shape)}")
        if self.penalties is not None and self._tokens is None:
            raise RuntimeError("fork() before advance() with penalties")
        if self.penalties is not None and _lib.capture_id(self.scores.device):
            raise RuntimeError("advance() with penalties cannot be captured")
        window = [self._window_from(i) for i in range(len(self.decoders))]
        for d, w in zip(self.decoders, window):      # refused before any row has moved
            d._check_reorder(w)
        if self.penalties is not None:
            past = self._tokens[:, :self._length].unflatten(0, (self.requests, self.beams))
            logits = adjust_logits(logits, history=past, prompt=self._prompt, bias=bias, mask=mask, **self.penalties)
        elif bias is not None or mask is not None:
            logits = adjust_logits(logits, bias=bias, mask=mask)
        scores, rows, tokens = beam_select(logits, self.scores, self.beams, keep_places=True)
        rows, tokens = rows.view(-1), tokens.view(-1)
        for d, w in zip(self.decoders, window):
            d.reorder(rows, window_from=w)
        if self.penalties is not None:
            self._follow(rows, tokens)
        self.scores = scores
        return tokens, rows

    def _follow(self, rows, tokens) -> None:
        """The beams' tokens so far take over the rows they continue, and the new ones are put behind them."""
        t = self._tokens
        with _lib.on_device(t.device):
            one = (_lib.Rows * 1)(_lib.Rows(t.data_ptr(), t.size(1) * 4))
            _lib.check(_lib.lib().logkv_reorder_rows(
                one, 1, t.size(0), rows.data_ptr(), rows.dtype == torch.int64, self.decoders[0].cache._read.status_ptr,
                _lib.stream_ptr(t.device)), "logkv_reorder_rows")
        if self._length == t.size(1):
            self._tokens = t.new_empty(t.size(0), 2 * t.size(1))
            self._tokens[:, :self._length] = t
        self._tokens[:, self._length] = tokens
        self._length += 1
