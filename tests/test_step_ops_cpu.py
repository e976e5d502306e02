"""Refusals of a decoding step's operators (rotation, rotated append, logits), checked on the host before anything is
launched, and the tables of scaled rotary positions."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from hypotheses import make_cache


@pytest.fixture(scope="module")
def lib():
    from logkv_b200 import build
    build.build()
    from logkv_b200 import _lib
    return _lib.lib()


@pytest.fixture()
def cache(lib):
    return make_cache(torch.float32, B=2, G=2, D=64, levels=0, R=5, max_seq=500, device="cpu")


def test_rotate_refusals(cache):
    from logkv_b200 import log_kv_rotate as f
    q, k, p = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 3, 64), torch.arange(3)
    for args, kw, match in [
            ((q[:1], k, p), {}, "q must be"), ((q[0], k, p), {}, "q must be"), ((q[..., :32], k, p), {}, "q must be"),
            ((q.bfloat16(), k, p), {}, "q must be"), ((q, k[:, :1], p), {}, "k must be"),
            ((q, k[:, :, :2], p), {}, "k must be"), ((q, k.bfloat16(), p), {}, "k must be"),
            ((q[:, :3], k, p), {}, "multiple"), ((q[:, :0], k, p), {}, "multiple"), ((q, k, p[:2]), {}, "input_pos"),
            ((q, k, p[None]), {}, "input_pos"), ((q, k, p.float()), {}, "integers"),
            ((q, k, p), {"layout": "pairs"}, "layout")]:
        with pytest.raises(ValueError, match=match):
            f(cache, *args, **kw)
    with pytest.raises(NotImplementedError):
        f(cache, q.requires_grad_(), k, p)


def test_host_positions_are_checked_against_the_tables(cache):
    from logkv_b200.rotary import check_positions
    cache.register_buffer("recent_pos", torch.zeros(2, 512, dtype=torch.int64, device="meta"))
    for bad in ([0, 1, 564], [-1, 0, 1]):
        with pytest.raises(ValueError, match="rotary tables"):
            check_positions(cache, bad, 3)
    assert check_positions(cache, [0, 1, 563], 3).shape == (3,)
    assert check_positions(cache, None, 3) is None


def test_rotated_append_refusals(cache):
    k, ends = torch.zeros(2, 2, 3, 64), [[False] * 3] * 2
    f = lambda *a, **kw: cache.add_recent_rotated(*a, **{"span_ends": ends, **kw})  # noqa: E731
    before = (cache.token_count, cache.recent_count)
    for args, kw, match in [
            ((k[0], k), {}, "k_raw must be"), ((k[..., :32], k), {}, "k_raw must be"), ((k, k[:, :, :2]), {}, "v must be"),
            ((k, k.bfloat16()), {}, "v must be"), ((k, k), {"layout": "both"}, "layout"),
            ((k, k), {"input_pos": torch.arange(2)}, "input_pos"), ((k, k), {"input_pos": torch.rand(3)}, "integers"),
            ((k, k), {"span_ends": None}, "span boundaries"), ((k, k), {"span_ends": ends[:1]}, "span boundaries"),
            ((k, k), {"span_ends_device": torch.zeros(2, 2)}, "span boundaries")]:
        with pytest.raises(ValueError, match=match):
            f(*args, **kw)
    long = torch.zeros(2, 2, cache.recent_size + 1, 64)
    with pytest.raises(ValueError, match="recent_size"):
        f(long, long, span_ends=[[False] * long.size(2)] * 2)
    cache.token_count = 499
    with pytest.raises(RuntimeError, match="token overflow"):
        f(k, k)
    cache.token_count = before[0]
    cache._deferred_take = 1
    with pytest.raises(RuntimeError, match="commit_deferred"):
        f(k, k)
    cache._deferred_take = None
    f(k[:, :, :0], k[:, :, :0], span_ends=[[], []])
    assert before == (cache.token_count, cache.recent_count)


def test_shared_attention_refusals(cache):
    from logkv_b200 import log_kv_shared_attention
    q, k = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 3, 64)
    f = lambda q, k, v, **kw: log_kv_shared_attention(cache, q, k, v, 0.125, **{"beams": 2, "window_from": 5, **kw})  # noqa: E731
    for args, kw, match in [
            ((q[:1], k, k), {}, "q must be"), ((q[..., :32], k, k), {}, "q must be"), ((q[0], k, k), {}, "q must be"),
            ((q.bfloat16(), k, k), {}, "q must be"), ((q, k[:, :1], k), {}, "k must be"), ((q, k, k[:, :, :2]), {}, "v shape"),
            ((q, k.bfloat16(), k), {}, "dtype"), ((q[:, :, :2], k, k), {}, "same tokens"), ((q, k[:, :, :2], k[:, :, :2]), {}, "same tokens"),
            ((q[:, :, :2], k, k), {"causal_tail": 2}, "same tokens"), ((q, k, k), {"causal_tail": 2}, "causal_tail"),
            ((q[:, :3], k, k), {}, "multiple"), ((q[:, :0], k, k), {}, "multiple"), ((q, k, k), {"beams": 0}, "beams"),
            ((q, k, k), {"beams": 3}, "beams"), ((q, k, k), {"window_from": 6}, "window_from"),
            ((q, k, k), {"window_from": -1}, "window_from"), ((q, k, k), {"out": torch.zeros(2, 4, 3, 32)}, "out must be")]:
        with pytest.raises(ValueError, match=match):
            f(*args, **kw)
    with pytest.raises(NotImplementedError):
        f(q.clone().requires_grad_(), k, k)


def test_shared_attention_c_abi_checks(lib):
    from logkv_b200 import _lib
    layout = _lib.Layout(16, 8, 128, 12, 7, 125, 4096, 256, 64, 1, 1, 1.0, 2048.0, 1.0)
    a = _lib.SharedArgs()

    def size(lay=layout, cap=10756, **kw):
        base = dict(heads=16, beams=4, q_tokens=1, tokens=1, recent_count=100, window_from=60, causal=1)
        for name, value in {**base, **kw}.items():
            setattr(a, name, value)
        return lib.logkv_shared_attention_workspace_bytes(ctypes.byref(lay), ctypes.byref(a), cap)

    row = 16 * 16 * 132 * 4                              # partial rows of one split
    assert size() > 0 and size() % row == 0 and size(recent_count=4096, window_from=0) > 0
    assert size(beams=16, q_tokens=7, tokens=7) > 0 and size(q_tokens=1, tokens=2, causal=0) > 0
    for bad in (dict(heads=12), dict(heads=0), dict(beams=0), dict(beams=3), dict(q_tokens=0), dict(q_tokens=2),
                dict(tokens=2), dict(recent_count=4097), dict(recent_count=-1), dict(window_from=101), dict(window_from=-1),
                dict(cap=-1), dict(q_tokens=1 << 18, tokens=1 << 18, beams=16)):
        assert size(**bad) == 0, bad
    odd = _lib.Layout(16, 8, 96, 12, 7, 125, 4096, 256, 64, 1, 1, 1.0, 2048.0, 1.0)
    f32 = _lib.Layout(16, 8, 256, 12, 7, 125, 4096, 256, 64, 1, 0, 1.0, 2048.0, 1.0)
    assert size(odd) == 0 and size(f32) == 0
    n = size()
    state, pre = _lib.State(), _lib.Prefix()
    call = lambda bytes_: lib.logkv_shared_attention(ctypes.byref(layout), ctypes.byref(state), ctypes.byref(pre),  # noqa: E731
                                                     ctypes.byref(a), 1 << 20, bytes_, None)
    assert lib.logkv_shared_attention(None, None, None, None, None, 0, None) == -4
    pre.capacity = 10756
    assert call(n) == -4                                 # null pointers
    state.recent_k = state.recent_v = pre.k = pre.v = pre.mass = pre.length = 1 << 20
    a.q = a.k_new = a.v_new = a.out = 1 << 20
    assert call(n - 1) == -3                             # workspace too small
    a.k_strides[1] = 4
    assert call(n) == -4                                 # rows not 16-byte aligned
    a.k_strides[1], a.beams = 0, 3
    assert call(n) == -1


def test_logits_refusals(lib):
    from logkv_b200 import adjust_logits as f
    x, h = torch.zeros(2, 3, 70), torch.zeros(2, 3, 5, dtype=torch.int64)
    m, t, b = torch.zeros(2, 3, 3, dtype=torch.int32), torch.zeros(2, 3, 4, dtype=torch.int32), torch.zeros(2, 3, 4)
    n = torch.zeros(2, 3, dtype=torch.int64)
    for args, kw, match in [
            (x[0, 0], {}, "logits must be"), (x.half(), {}, "dtype"), (x[..., :0], {}, "supported range"),
            (torch.zeros(65536, 1), {}, "supported range"), (x, {"repetition": 0.0}, "positive"),
            (x, {"repetition": -1.0}, "positive"), (x, {"presence": math.inf}, "finite"),
            (x, {"frequency": math.nan}, "finite"), (x, {"repetition": b}, "repetition must be"),
            (x, {"presence": n}, "presence must be"), (x, {"history": h[0]}, "history must be"),
            (x, {"history": h.float()}, "history must be"), (x, {"history": h, "lengths": 6}, "at most"),
            (x, {"history": h, "lengths": -1}, "negative"), (x, {"history": h, "lengths": n[0]}, "lengths must be"),
            (x, {"history": h, "lengths": n.float()}, "lengths must be"), (x, {"lengths": 3}, "without a history"),
            (x, {"history": h, "prompt": -2}, "negative"), (x, {"history": h, "prompt": n[:, :2]}, "prompt must be"),
            (x, {"bias": (t, b[..., :3])}, "one shape"), (x, {"bias": (t[0, 0], b)}, "one shape"),
            (x, {"bias": (b, b)}, "bias tokens must be"), (x, {"bias": (t, b.double())}, "bias values must be"),
            (x, {"bias": (t[0], b[0])}, "bias tokens must be"),
            (x, {"bias": (torch.zeros(1025, dtype=torch.int64), torch.zeros(1025))}, "at most 1024"),
            (x, {"mask": m[..., :2]}, "3 words"), (x, {"mask": m.long()}, "mask must be"), (x, {"mask": m[0]}, "mask must be"),
            (x, {}, "CUDA tensor")]:
        with pytest.raises(ValueError, match=match):
            f(args, **kw)
    for kw in ({}, {"bias": (t, b.clone().requires_grad_())}):
        with pytest.raises(NotImplementedError):
            f(x.clone().requires_grad_() if not kw else x, **kw)


def test_c_abi_checks(lib):
    from logkv_b200 import _lib
    rope, a = _lib.Rope(1 << 20, 1 << 20, 100, 64, 0), _lib.RotateArgs()
    call = lambda: lib.logkv_rotate(ctypes.byref(rope), ctypes.byref(a), None)  # noqa: E731
    assert lib.logkv_rotate(None, ctypes.byref(a), None) == -4
    assert call() == -1                                  # no parts
    a.n_parts, a.batch, a.tokens, a.dim = 1, 1, 1, 64
    assert call() == -4                                  # null pointers
    a.parts[0].src, a.parts[0].heads, a.parts[0].rotate = 1 << 20, 1, 1
    assert call() == -4                                  # nowhere to write
    a.parts[0].rotated = (1 << 20) + 2
    assert call() == -4                                  # a float32 row off 4 bytes
    a.parts[0].rotated = 1 << 21
    a.dtype = 2
    assert call() == -2
    a.dtype, rope.rope_n = 0, 63
    assert call() == -1
    rope.rope_n = 66
    assert call() == -1
    rope.rope_n, rope.rows = 64, 0
    assert call() == -4
    rope.rows, a.positions, a.positions_wide = 100, (1 << 20) + 4, 1
    assert call() == -4
    x = _lib.LogitsArgs()
    call = lambda: lib.logkv_adjust_logits(ctypes.byref(x), None)  # noqa: E731
    assert call() == -1
    x.rows, x.width, x.vocab, x.repetition = 3, 1, 100, 1.0
    assert call() == -4
    x.logits = x.out = 1 << 20
    x.mask = (1 << 20) + 2
    assert call() == -4
    x.mask, x.repetition = None, 0.0
    assert call() == -1
    x.repetition, x.bias_count = 1.0, 1025
    assert call() == -1
    x.bias_count, x.dtype = 0, 5
    assert call() == -2


def test_scaled_tables():
    """Angles against their formulas in 64 bits, rounded once."""
    from logkv_b200 import scaled_rope_tables as f
    n, base, rows = 32, 5e5, 70000
    inv = np.array([base ** (-2 * i / n) for i in range(n // 2)])
    pos = np.array([0, 1, 4097, 65535, 65536, 69999])

    def close(tables, freq, amplitude=1.0):
        cos, sin = tables
        assert cos.shape == sin.shape == (rows, n) and cos.dtype == torch.float32
        ang = pos[:, None] * freq[None]
        for t, want in ((cos, np.cos(ang)), (sin, np.sin(ang))):
            got = t[pos].double().numpy()
            # 2^-24 relative for the rounding; the angle's own float64 rounding moves it by pos 2^-52.
            assert (np.abs(got - np.concatenate([want, want], 1) * amplitude) <= 2.0 ** -24 * amplitude * 1.01).all()

    close(f(rows, n, base=base), inv)
    close(f(rows, n, base=base, scaling={"kind": "linear", "factor": 4}), inv / 4)
    wide = f(rows, n, base=base, scaling={"kind": "base", "factor": 8})
    stretched = np.array([(base * 8 ** (n / (n - 2))) ** (-2 * i / n) for i in range(n // 2)])
    close(wide, stretched)
    assert math.isclose(stretched[-1], inv[-1] / 8, rel_tol=1e-12) and stretched[0] == 1
    bands = np.empty(n // 2)
    for i, w in enumerate(inv):
        turns = 8192 * w / (2 * math.pi)
        bands[i] = w if turns > 4 else w / 8 if turns < 1 else w / 8 + (turns - 1) / 3 * (w - w / 8)
    close(f(rows, n, base=base, scaling={"kind": "bands", "factor": 8, "original": 8192, "low": 1, "high": 4}), bands)
    lo = math.floor(n * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(base)))
    hi = math.ceil(n * math.log(4096 / (2 * math.pi)) / (2 * math.log(base)))
    yarn = np.array([w * (1 - min(max((i - lo) / (hi - lo), 0), 1) * (1 - 1 / 16)) for i, w in enumerate(inv)])
    close(f(rows, n, base=base, scaling={"kind": "yarn", "factor": 16, "original": 4096}), yarn, 0.1 * math.log(16) + 1)
    assert f(10, 8, dtype=torch.bfloat16)[0].dtype == torch.bfloat16
    for kw in ({"scaling": {"kind": "other"}}, {"scaling": {"kind": "linear"}}, {"scaling": {"kind": "linear", "factor": 0.5}},
               {"scaling": {"kind": "linear", "factor": 2, "low": 1}}, {"base": 1.0}, {"dtype": torch.float16},
               {"scaling": {"kind": "bands", "factor": 2, "original": 10, "low": 4, "high": 1}},
               {"scaling": {"kind": "yarn", "factor": 2, "original": 10, "fast": 1, "slow": 4}}):
        with pytest.raises(ValueError):
            f(10, 8, **kw)
    for shape in ((0, 8), (10, 7), (10, 0)):
        with pytest.raises(ValueError):
            f(*shape)
