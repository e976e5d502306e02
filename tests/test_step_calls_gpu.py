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


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [64, 1003, 5000])
def test_banned_tokens_of_the_history(dtype, V):
    """A banned token is -inf whatever its row's penalties, its count or its logit are; the others follow the formula."""
    from logkv_b200 import adjust_logits
    inf, nan = float("inf"), float("nan")
    rows = 7
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(rows, V, generator=gen, device="cuda").to(dtype)
    x[:, 5], x[:, 6] = -inf, nan
    h = torch.randint(0, V, (rows, 40), generator=gen, device="cuda")
    h[:, :4] = torch.tensor([3, 5, 6, 9], device="cuda")
    allowed = torch.rand(rows, V, generator=gen, device="cuda") < 0.5
    allowed[:, 3] = allowed[:, 5] = allowed[:, 6] = False
    allowed[:, 9] = True
    bits = torch.zeros(rows, (V + 31) // 32 * 32, dtype=torch.bool, device="cuda")
    bits[:, :V] = allowed
    mask = (bits.view(rows, -1, 32).long() << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
    rep = torch.tensor([1.0, 2.0, 1.5, 0.5, inf, 1.0, 1.0], device="cuda")
    pres = torch.tensor([-inf, 0.25, inf, 0.0, 0.0, -inf, nan], device="cuda")
    freq = torch.tensor([0.0, -inf, 0.0, 3e38, 0.0, inf, 0.0], device="cuda")
    bias = (torch.tensor([3, 9, 11], device="cuda"), torch.tensor([inf, 0.5, -1.0], device="cuda"))
    for b in (None, bias):
        kw = dict(history=h, repetition=rep, presence=pres, frequency=freq, mask=mask, bias=b)
        got = adjust_logits(x, **kw)
        assert (got[~allowed] == -inf).all()
        for _ in range(2):
            assert torch.equal(adjust_logits(x, **kw).nan_to_num(7.0), got.nan_to_num(7.0))
        y = x.clone()
        adjust_logits(y, out=y, **kw)
        assert torch.equal(y.nan_to_num(7.0), got.nan_to_num(7.0))
        free = adjust_logits(x, **{**kw, "mask": None})
        assert torch.equal(got[allowed].nan_to_num(7.0), free[allowed].nan_to_num(7.0))


def test_append_of_host_span_ends_does_not_wait():
    """Host lists of span ends go to the device without a wait, in the window write and in a flush's."""
    cache = make(BF16)
    chunks = [projected(cache, 2, T, T)[1:] for T in (64, 20, 64)]
    ends = [torch.rand(2, k.size(2), generator=torch.Generator().manual_seed(k.size(2))) < 0.3 for k, _ in chunks]
    other = make(BF16)
    for (k, v), e in zip(chunks, ends):
        other.add_recent_rotated(k, v, span_ends_device=e.cuda())
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for (k, v), e in zip(chunks, ends):
            cache.add_recent_rotated(k, v, span_ends=e.tolist())
    finally:
        torch.cuda.set_sync_debug_mode("default")
    x, y = state(cache), state(other)
    for name in x:
        assert torch.equal(x[name], y[name]), name


def test_captured_append_refuses_host_span_ends():
    """A graph would read the lists' staging memory again at every replay, when it holds something else."""
    cache = make(BF16)
    _, k, v = projected(cache, 2, 2, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        x = k + 1
        with pytest.raises(RuntimeError, match="span_ends_device"):
            cache.add_recent_rotated(k, v, span_ends=[[False, True]] * 2)
    graph.replay()
    assert torch.equal(x, k + 1) and cache.recent_count == cache.token_count == 0
    cache.add_recent_rotated(k, v, span_ends=[[False, True]] * 2)
    assert cache.recent_count == 2 and cache.read_status() == 0


@pytest.mark.parametrize("name", ["prompt", "lengths", "repetition", "presence", "frequency"])
def test_numbers_out_of_range(name):
    """Python integers of any size are refused like others, and a prompt longer than the history is the whole of it."""
    from logkv_b200 import adjust_logits
    x = torch.randn(3, 100, device="cuda")
    h = torch.randint(0, 100, (3, 9), device="cuda")
    kw = dict(history=h, repetition=1.5, frequency=0.25)
    want = adjust_logits(x, prompt=9, **kw)
    if name == "prompt":
        assert torch.equal(adjust_logits(x, prompt=10 ** 400, **kw), want)
        return
    for bad in (10 ** 400, -10 ** 400):
        with pytest.raises(ValueError):
            adjust_logits(x, prompt=9, **{**kw, name: bad})


@pytest.mark.parametrize("name", ["beams", "window_from"])
def test_shared_numbers_out_of_range(name):
    from logkv_b200 import log_kv_shared_attention
    cache = make(BF16, B=4)
    q, k, v = (t.contiguous() for t in projected(cache, 4, 1, 3))
    f = lambda **kw: log_kv_shared_attention(cache, q, k, v, 0.125, **{"beams": 2, "window_from": 0, **kw})  # noqa: E731
    f()
    for bad in (10 ** 30, -10 ** 30):
        with pytest.raises(ValueError):
            f(**{name: bad})


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype,D,beams", [(BF16, 64, 2), (BF16, 64, 12), (BF16, 128, 3), (F32, 64, 2)])
def test_one_feature_of_a_new_value_that_is_not_finite(dtype, D, beams, bad):
    """One query token, or new tokens that all queries see: that feature of the row's outputs alone is not finite.
    Several query tokens in order: the outputs of those that see the token are NaN, the others as without it."""
    from logkv_b200 import log_kv_shared_attention
    cache = make(dtype, B=2 * beams, D=D, window=64)
    n = 40
    _, k, v = projected(cache, 4, n, 1)
    cache.add_recent_rotated(k[:1].expand(2 * beams, -1, -1, -1), v[:1].expand(2 * beams, -1, -1, -1),
                             span_ends_device=torch.zeros(2 * beams, n, dtype=torch.uint8, device="cuda"))
    call = lambda q, k, v, tail: log_kv_shared_attention(cache, q, k, v, 0.125, beams=beams, window_from=n - 7,  # noqa: E731
                                                         causal_tail=tail)
    row, feature, token = 1, D - 3, 1
    for T, Tk, tail in ((1, 1, None), (1, 2, 0), (2, 3, 0), (3, 3, None)):
        q, k, v = (t.contiguous() for t in projected(cache, 4, Tk, 2))
        q = q[:, :, :T].contiguous()
        want = call(q, k, v, tail)
        assert torch.isfinite(want).all()
        v[row, 1, min(token, Tk - 1), feature] = bad
        got = call(q, k, v, tail)
        spoiled = torch.zeros_like(got, dtype=torch.bool)      # heads 2 and 3 are the second group's
        if tail is None and T > 1:
            spoiled[row, 2:, token:] = True
            assert torch.isnan(got[spoiled]).all()
        else:
            spoiled[row, 2:, :, feature] = True
            assert not torch.isfinite(got[spoiled]).any()
        assert torch.equal(got[~spoiled], want[~spoiled])
    assert cache.read_status() == 0
