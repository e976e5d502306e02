"""Rotary positions on the GPU (include/logkv_rotary.h): queries and keys rotated with a cache's tables.

The reference's model rotates in PyTorch before it calls its cache (litgpt/model.py); here one kernel makes what
attention and the cache take: rotated queries, rotated keys and the unrotated keys in the cache's order.
``LogStructuredKVCache.add_recent_rotated`` and ``LogKVDecoder.step_raw`` use the same kernel to bring unrotated
rows into the window and the pending slot.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _lib

LAYOUTS = {"half": 0, "interleaved": 1}


def check_layout(layout: str) -> int:
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    return LAYOUTS[layout]


def check_positions(cache, input_pos, T: int):
    """Positions of T tokens ([T] or [B, T] integers) on the cache's device, int32 or int64; host values are
    checked against the tables.  None: None."""
    if input_pos is None:
        return None
    B, dev = cache.batch_size, cache.recent_pos.device
    p = input_pos if isinstance(input_pos, torch.Tensor) else torch.as_tensor(input_pos)
    if p.dtype != torch.int32 and p.dtype != torch.int64 and p.numel():
        raise ValueError(f"input_pos must hold integers (int32 or int64), got {p.dtype}")
    if p.shape != (T,) and p.shape != (B, T):
        raise ValueError(f"input_pos must be [{T}] or [{B}, {T}], got {tuple(p.shape)}")
    if p.device != dev:
        if p.device.type != "cpu":
            raise ValueError(f"input_pos must be on {dev}, got {p.device}")
        if cache.rope_n_elem and bool(((p < 0) | (p >= cache.cos_cache.size(0))).any()):
            raise ValueError(f"input_pos must lie in the rotary tables, [0, {cache.cos_cache.size(0)})")
        p = p.to(dev)
    return p


def last_contiguous(t):
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def part(src, rotated=None, raw=None) -> _lib.RotatePart:
    """One tensor of a call ([B, heads, T, D] views); without ``rotated`` a plain copy into ``raw``."""
    x = _lib.RotatePart()
    x.src, x.heads, x.rotate = src.data_ptr(), src.size(1), rotated is not None
    x.src_strides[:] = src.stride()[:3]
    if rotated is not None:
        x.rotated = rotated.data_ptr()
        x.rotated_strides[:] = rotated.stride()[:3]
    if raw is not None:
        x.raw = raw.data_ptr()
        x.raw_strides[:] = raw.stride()[:3]
    return x


def launch(cache, parts, positions, pos0: int, interleaved: int, *, positions_out=None, ends=None, ends_out=None) -> None:
    """logkv_rotate of ``parts`` (their tensors [B, heads, T, D]) on the current stream of the cache's device;
    positions_out [B, T] int64 and ends / ends_out [B, T] uint8, unit token stride."""
    from .attention import _rope
    first = parts[0][0]
    a = _lib.RotateArgs()
    for i, p in enumerate(parts):
        a.parts[i] = part(*p)
    a.n_parts, a.batch, a.tokens, a.dim = len(parts), first.size(0), first.size(2), first.size(3)
    a.dtype, a.interleaved, a.pos0 = _lib.DTYPE_CODES[first.dtype], interleaved, int(pos0)
    if positions is not None:
        a.positions, a.positions_wide = positions.data_ptr(), positions.dtype == torch.int64
        s = positions.stride()
        a.position_strides[:] = s if len(s) == 2 else (0, s[0])
    if positions_out is not None:
        a.positions_out, a.positions_out_stride = positions_out.data_ptr(), positions_out.stride(0)
    if ends_out is not None:
        a.ends, a.ends_out = ends.data_ptr(), ends_out.data_ptr()
        a.ends_stride, a.ends_out_stride = ends.stride(0), ends_out.stride(0)
    status = getattr(cache, "_read_status", None)   # a foreign cache has none
    a.status = None if status is None else status.data_ptr()
    rope = _rope(cache)
    if status is not None and native(cache) is None and _contiguous(cache):
        cache._rotary = _Native(cache, rope)
    _lib.check(_lib.lib().logkv_rotate(ctypes.byref(rope), ctypes.byref(a), _lib.stream_ptr(cache.recent_k.device)),
               "logkv_rotate")


def _contiguous(cache) -> bool:
    """Whether the tables can be read where they are; strided ones are copied in every call."""
    b = cache._buffers
    return b["cos_cache"].is_contiguous() and b["sin_cache"].is_contiguous()


class _Native:
    """The host binding's calls with their arguments that do not change for a cache."""

    def __init__(self, cache, rope):
        host = _lib.host()
        self.rotate, self.append, self.fn = host.rotate, host.append, _lib.address("logkv_rotate")
        self.tables = rope
        self.rope, self.dtype = ctypes.addressof(self.tables), cache.cos_cache.dtype
        self.status = cache._read_status.data_ptr()


def native(cache):
    """The cache's _Native once a call has gone through and while its tables are what they were; else None."""
    n = getattr(cache, "_rotary", None)
    if n is None:
        return None
    b = cache._buffers
    cos, sin = b["cos_cache"], b["sin_cache"]
    t = n.tables
    same = (t.cos == cos.data_ptr() and t.sin == sin.data_ptr() and t.rows == cos.size(0) and n.dtype is cos.dtype
            and _contiguous(cache))
    return n if same or not cache.rope_n_elem else None


def log_kv_rotate(cache, q, k, input_pos=None, *, layout: str = "half"):
    """Queries and keys rotated at their positions: (q, k, k_raw) as ``log_kv_chunk_attention``,
    ``log_kv_tree_attention``, ``log_kv_shared_attention`` and ``add_recent`` take them (no reference counterpart).

    q [B, H, T, D] and k [B, G, T, D] are a projection's unrotated output in the cache dtype, any strides.
    ``input_pos`` ([T] or [B, T]; int32 or int64) are the tokens' positions, None for those that continue the
    sequence (token_count and on).  Positions on the host are checked here; one in a device tensor that lies outside
    the tables is rotated at the nearest table row and sets bit 16 of ``cache.read_status()``.

    The cache's tables and ``rope_n_elem`` say how (``scaled_rope_tables`` makes them for long contexts): the first
    rope_n_elem features rotate, the others pass.  ``layout`` "half": feature i turns with i + rope_n_elem / 2, and
    k_raw is k itself.  "interleaved": features (2 i, 2 i + 1) turn together, and all three results come in halves,
    the order in which the cache rotates what it keeps; attention does not depend on it.

    Computed in float32 and rounded once (tables are read as they are stored).  Forward-only.
    """
    mode = check_layout(layout)
    call = native(cache)
    if call is not None:     # checks, allocations and launch in the host binding; None: not covered there
        y = call.rotate(call.fn, call.rope, call.status, cache._buffers["recent_k"], q, k, input_pos, cache.token_count,
                        mode)
        if y is not None:
            if type(y) is int:
                _lib.check(y, "logkv_rotate")
            return y
    dev, dt, B, G, D = cache.recent_k.device, cache.recent_k.dtype, cache.batch_size, cache.n_groups, cache.k_dim
    if q.dim() != 4 or q.size(0) != B or q.size(3) != D or q.dtype != dt:
        raise ValueError(f"q must be [B={B}, H, T, {D}] in the cache dtype, got {tuple(q.shape)} {q.dtype}")
    H, T = q.size(1), q.size(2)
    if k.shape != (B, G, T, D) or k.dtype != dt:
        raise ValueError(f"k must be [{B}, {G}, {T}, {D}] in the cache dtype, got {tuple(k.shape)} {k.dtype}")
    if H < 1 or H % G:
        raise ValueError(f"query heads {H} must be a multiple of KV groups {G}")
    if q.device != dev or k.device != dev:
        raise ValueError(f"q and k must be on the cache's device {dev}")
    if (q.requires_grad or k.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError("log_kv_rotate is forward-only")
    p = check_positions(cache, input_pos, T)
    qo, ko = q.new_empty((B, H, T, D)), k.new_empty((B, G, T, D))
    raw = k.new_empty((B, G, T, D)) if mode else k
    if T:
        with _lib.on_device(dev):
            launch(cache, [(last_contiguous(q), qo), (last_contiguous(k), ko, raw if mode else None)], p,
                   cache.token_count, mode)
    return qo, ko, raw


def _entry(name: str, value, infinite: bool = False) -> float:
    """A scaling's entry as a finite number (or one that may be infinite)."""
    try:
        number = float(value)
    except (TypeError, ValueError, OverflowError):
        number = math.nan
    if not math.isfinite(number) and not (infinite and number == math.inf):
        raise ValueError(f"{name} must be a finite number, got {value!r}")
    return number


def scaled_rope_tables(length: int, n_elem: int, *, base: float = 10000.0, scaling: dict | None = None, device=None,
                       dtype=torch.float32):
    """(cos, sin), each [length, n_elem], of the positions 0 .. length - 1 as ``LogStructuredKVCache`` takes them.

    Angles are position * base ** (-2 i / n_elem), taken in float64 and rounded once.  ``scaling`` stretches them for
    contexts longer than the model's own:
      {"kind": "linear", "factor": f}            every angle divided by f;
      {"kind": "base", "factor": f}              base * f ** (n_elem / (n_elem - 2)): the slowest pair divided by f,
                                                 the fastest kept;
      {"kind": "bands", "factor": f, "original": n, "low": a, "high": b}
                                                 pairs that turn less than a times over the original n positions
                                                 divided by f, those that turn more than b times kept, in between
                                                 blended linearly in the number of turns;
      {"kind": "yarn", "factor": f, "original": n, "fast": 32, "slow": 1, "attention": 0.1 ln f + 1}
                                                 blended linearly over the pairs' indices between those that turn
                                                 `fast` and `slow` times, and the tables multiplied by `attention`
                                                 (queries and keys both carry it).
    """
    length, n = int(length), int(n_elem)
    if length < 1 or n < 2 or n % 2:
        raise ValueError(f"length must be positive and n_elem even and positive, got {length} and {n}")
    if dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"table dtype {dtype} is not supported (float32 or bfloat16)")
    s = dict(scaling or {"kind": "none"})
    known = {"none": (), "linear": ("factor",), "base": ("factor",), "bands": ("factor", "original", "low", "high"),
             "yarn": ("factor", "original", "fast", "slow", "attention")}
    kind = s.pop("kind", None)
    if kind not in known or set(s) - set(known[kind]):
        raise ValueError(f"scaling must be one of {sorted(known)} with its own entries, got {scaling}")
    missing = [name for name in known[kind] if name not in s and name not in ("fast", "slow", "attention")]
    if missing:
        raise ValueError(f"scaling {kind!r} needs {missing}")
    entry = lambda name, default: _entry(name, s.get(name, default))  # noqa: E731
    f = entry("factor", 1.0)
    if not (math.isfinite(base) and base > 1 and f >= 1):
        raise ValueError(f"base must be above 1 and factor at least 1, got {base} and {f}")
    original = entry("original", 1.0)
    if original <= 0:
        raise ValueError(f"original must be positive, got {original}")
    i = np.arange(n // 2, dtype=np.float64)
    amplitude = 1.0
    if kind == "base" and n > 2:
        base = base * f ** (n / (n - 2))
    inv = base ** (-2.0 * i / n)
    if kind == "linear" or (kind == "base" and n == 2):
        inv = inv / f
    elif kind == "bands":
        turns = original * inv / (2 * math.pi)
        low, high = entry("low", None), _entry("high", s["high"], infinite=True)   # infinite: no pair is kept
        if not 0 < low < high:
            raise ValueError(f"bands need 0 < low < high, got {low} and {high}")
        keep = np.clip((turns - low) / (high - low), 0.0, 1.0)
        inv = inv * (keep + (1 - keep) / f)
    elif kind == "yarn":
        fast, slow = entry("fast", 32), entry("slow", 1)
        if not 0 < slow < fast:
            raise ValueError(f"yarn needs 0 < slow < fast, got {slow} and {fast}")
        # Index of the pair that turns `t` times over the original positions.
        at = lambda t: n * math.log(original / (t * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), n - 1)
        stretch = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        inv = inv * ((1 - stretch) + stretch / f)
        amplitude = entry("attention", 0.1 * math.log(f) + 1.0)
    inv = torch.from_numpy(inv).to(device or "cpu")
    cos, sin = (torch.empty(length, n, dtype=dtype, device=inv.device) for _ in range(2))
    for at0 in range(0, length, 65536):     # the float64 angles of a part of the positions at a time
        to = min(length, at0 + 65536)
        ang = torch.arange(at0, to, dtype=torch.float64, device=inv.device)[:, None] * inv
        for out, fn in ((cos, torch.cos), (sin, torch.sin)):
            v = (fn(ang) * amplitude).to(dtype)
            out[at0:to, :n // 2], out[at0:to, n // 2:] = v, v
    return cos, sin
