"""Calls of a decoding step's operators that their other tests do not make."""
from __future__ import annotations

import pytest
import torch

from test_rotary_gpu import BF16, F32, check, make, projected, state
from test_step_calls_cpu import strided_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tables", [F32, BF16])
def test_strided_tables(tables):
    """Tables that are every other column of wider ones, from the start and in place of others: rotated alone, on the
    way into the window and in the packed prefix as contiguous ones are."""
    from logkv_b200 import log_kv_rotate
    from logkv_b200.attention import refresh_prefix
    cos, sin = (t.to("cuda", tables) for t in strided_tables(512, 64))
    wide = [torch.full((512, 128), 7.0, device="cuda", dtype=tables) for _ in range(2)]
    for w, t in zip(wide, (cos, sin)):
        w[:, ::2] = t
    cos, sin = (w[:, ::2] for w in wide)
    a, b = make(F32, tables=tables), make(F32, tables=tables)
    a.cos_cache, a.sin_cache = cos, sin
    pos = torch.randint(0, 512, (2, 9), device="cuda")
    for layout in ("half", "interleaved"):
        for _ in range(2):
            check(a, 4, 9, pos, layout)
    for step, T in enumerate((64, 64, 30, 2)):
        _, k, v = projected(a, 2, T, step)
        ends = torch.zeros(2, T, dtype=torch.uint8, device="cuda")
        at = (torch.arange(T, device="cuda") + a.token_count) % 512
        a.add_recent_rotated(k, v, input_pos=at, span_ends_device=ends)
        b.add_recent_rotated(k, v, input_pos=at, span_ends_device=ends)
        x, y = state(a), state(b)
        for name in x:
            assert torch.equal(x[name], y[name]), (step, name)
    x, y = refresh_prefix(a), refresh_prefix(b)
    assert x.length.max() > 0 and torch.equal(x.length, y.length) and torch.equal(x.pk, y.pk) and torch.equal(x.pv, y.pv)
    q, k, _ = projected(a, 4, 3, 9)
    a.cos_cache, a.sin_cache = b.cos_cache, b.sin_cache           # contiguous ones again
    for _ in range(2):
        assert torch.equal(log_kv_rotate(a, q, k)[0], log_kv_rotate(b, q, k)[0])
    a.cos_cache = b.cos_cache[:1].expand(512, 64)                 # one row for all, at the same address
    check(a, 4, 9, pos, "half")
