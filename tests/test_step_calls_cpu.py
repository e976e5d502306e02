"""Calls of a decoding step's operators that their other tests do not make, as far as the host goes."""
from __future__ import annotations

import ctypes
import os
import re

import pytest
import torch

from hypotheses import make_cache


@pytest.fixture(scope="module")
def lib():
    from logkv_b200 import build
    build.build()
    from logkv_b200 import _lib
    return _lib.lib()


def strided_tables(rows, n):
    """Rotary tables as every other column of a wider one."""
    from logkv_b200 import scaled_rope_tables
    out = []
    for t in scaled_rope_tables(rows, n, base=1e4):
        wide = torch.full((rows, 2 * n), 7.0)
        wide[:, ::2] = t
        out.append(wide[:, ::2])
    return out


def test_strided_tables_keep_their_memory(lib, monkeypatch):
    """The addresses of a rotation's tables are those of tensors that live as long as the addresses do."""
    from logkv_b200 import _lib
    from logkv_b200.attention import _rope
    cos, sin = strided_tables(564, 64)
    cache = make_cache(torch.float32, B=2, G=2, D=64, levels=0, R=5, max_seq=500, device="cpu")
    monkeypatch.setattr(_lib, "ptr", lambda t: t.contiguous().data_ptr())
    cache.cos_cache, cache.sin_cache = cos, sin
    rope = _rope(cache)
    assert rope.cos != rope.sin
    for at, t in ((rope.cos, cos), (rope.sin, sin)):
        held = torch.frombuffer((ctypes.c_float * t.numel()).from_address(at), dtype=torch.float32)
        assert torch.equal(held.view(t.shape), t)


def test_constructor_lays_strided_tables_out(lib):
    from logkv_b200 import LogStructuredKVCache
    cos, sin = strided_tables(600, 64)
    shape = (2, 2, 500, 64)
    cache = LogStructuredKVCache(
        shape, shape, B=32, recent_size=64, device="cpu", dtype=torch.float32, semantic_clusters=True,
        semantic_anchor_mode="mid", allocate_second_order=False, cluster_k_max=4, semantic_flush_granularity=64,
        alpha_exact_tokens=32, alpha_span_max_tokens=8, beta_novelty=True, beta_adaptive_merge=True, cos_cache=cos,
        sin_cache=sin, rope_n_elem=64)
    assert cache.cos_cache.is_contiguous() and cache.sin_cache.is_contiguous()
    assert torch.equal(cache.cos_cache, cos) and torch.equal(cache.sin_cache, sin)


def test_shared_kernels_read_the_prefix_behind_their_wait():
    """What an earlier kernel wrote is visible behind a kernel's own wait (pdl_entry) only: in front of it nothing looks
    at the prefix's length."""
    import logkv_b200
    at = os.path.join(os.path.dirname(logkv_b200.__file__), "csrc", "shared_attention.cu")
    with open(at) as fh:
        kernels = [k.split("\n}\n")[0] for k in fh.read().split("__global__")[1:]]
    assert len(kernels) == 4
    for k in kernels:
        before, entry, after = k.partition("pdl_entry();")
        assert entry and re.search(r"share_prefix_length|share_keys", after)
        assert not re.search(r"share_prefix_length|share_keys|pre\.", before), before


def test_penalties_beyond_float32(lib):
    """Numbers that float32 has no finite (positive) value for are refused like infinities."""
    from logkv_b200 import adjust_logits
    x = torch.zeros(2, 3, 70)
    for name, bad in [("repetition", 1e300), ("repetition", 1e-60), ("repetition", 10 ** 400), ("presence", 1e300),
                      ("presence", -1e39), ("presence", 10 ** 400), ("frequency", -10 ** 400), ("frequency", 3.5e38)]:
        with pytest.raises(ValueError, match="finite"):
            adjust_logits(x, **{name: bad})
    for ok in (3.4e38, 1e-40):
        with pytest.raises(ValueError, match="CUDA tensor"):
            adjust_logits(x, repetition=ok, presence=-ok)


def test_in_place_rows_that_share_memory(lib):
    """Logits adjusted in place whose rows overlap, in whatever way their strides make it, are refused."""
    from logkv_b200 import adjust_logits
    base = torch.zeros(4000)
    for shape, strides in [((3, 2, 70), (70, 70, 1)), ((2, 3, 70), (140, 70, 1)), ((3, 2, 70), (70, 140, 1)),
                           ((3, 70), (69, 1)), ((2, 2, 70), (0, 70, 1)), ((3, 3, 70), (70, 200, 1)), ((2, 70), (0, 1))]:
        x = base.as_strided(shape, strides)
        with pytest.raises(ValueError, match="share memory"):
            adjust_logits(x, out=x)
    for shape, strides in [((3, 2, 70), (140, 70, 1)), ((3, 2, 70), (70, 210, 1)), ((3, 1, 70), (70, 0, 1)),
                           ((1, 3, 70), (0, 75, 1)), ((3, 70), (80, 1)), ((0, 2, 70), (0, 70, 1)), ((2, 2, 1), (2, 1, 1))]:
        x = base.as_strided(shape, strides)
        with pytest.raises(ValueError, match="CUDA tensor"):
            adjust_logits(x, out=x)


def test_scaling_entries_are_checked(lib):
    from logkv_b200 import scaled_rope_tables as f
    bands = {"kind": "bands", "factor": 2, "original": 10, "low": 1, "high": 4}
    yarn = {"kind": "yarn", "factor": 2, "original": 10}
    inf, nan = float("inf"), float("nan")
    for s, name, bads in [(bands, "original", (0, -5, inf, nan, None)), (yarn, "original", (0, -5, inf, nan, None, "x")),
                          (yarn, "attention", (None, inf, nan, "x")), (bands, "low", (None, nan)),
                          (bands, "high", (None, nan)), (yarn, "fast", (None, inf, nan)), (yarn, "slow", (None, nan)),
                          (bands, "factor", (None, inf, "x"))]:
        for bad in bads:
            with pytest.raises(ValueError, match=name):
                f(10, 8, scaling={**s, name: bad})
    all_divided = f(10, 8, scaling={"kind": "linear", "factor": 2})
    assert torch.equal(f(10, 8, scaling={**bands, "high": inf})[0], all_divided[0])
    f(10, 8, scaling=bands), f(10, 8, scaling={**yarn, "attention": 0.9})
