"""Rotary positions (log_kv_rotate) against their 64-bit form, and rows appended with the rotation on the way
(add_recent_rotated) against rotating and appending them."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def make(dtype=F32, B=2, G=2, D=64, n=None, rows=512, window=64, tables=F32, granularity=None, scaling=None):
    from logkv_b200 import LogStructuredKVCache, scaled_rope_tables
    n = D if n is None else n
    cos, sin = scaled_rope_tables(rows, n, base=1e4, scaling=scaling, dtype=tables) if n else (torch.zeros(rows, 0),) * 2
    shape = (B, G, 4096, D)
    return LogStructuredKVCache(
        shape, shape, B=32, recent_size=window, device="cuda", dtype=dtype, semantic_clusters=True,
        semantic_anchor_mode="mid", allocate_second_order=False, cluster_k_max=4,
        semantic_flush_granularity=granularity or window, alpha_exact_tokens=32, alpha_span_max_tokens=8,
        beta_novelty=True, beta_adaptive_merge=True, cos_cache=cos, sin_cache=sin, rope_n_elem=n)


def projected(cache, heads, T, seed, fused=True, odd=False):
    """q, k, v as slices of one projection's [B, T, heads, D] output; `odd`: rows that start off 16 bytes."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, G, D, dt = cache.batch_size, cache.n_groups, cache.k_dim, cache.level_k.dtype
    wide = (heads + 2 * G) * D + (1 if odd else 0)
    x = torch.randn(B, T, wide, generator=gen, device="cuda").to(dt)
    x = x[..., wide - (heads + 2 * G) * D:].unflatten(-1, (heads + 2 * G, D)).transpose(1, 2)
    q, k, v = x[:, :heads], x[:, heads:heads + G], x[:, heads + G:]
    return (q, k, v) if fused else (q.contiguous(), k.contiguous(), v.contiguous())


def reference(cache, x, pos, interleaved):
    """(64-bit result, bound on a kernel's distance from it, raw halves).

    x c is exact inside the fused product and sum, the other product is rounded once (2^-24 of it), the sum once,
    and the result once to the storage type (u of it)."""
    n, u = cache.rope_n_elem, torch.finfo(x.dtype).eps / 2
    h = n // 2
    raw = torch.cat([x[..., 0:n:2], x[..., 1:n:2], x[..., n:]], -1) if interleaved else x
    y = raw.double().clone()
    bound = torch.zeros_like(y)
    at = pos.long().expand(x.size(0), -1)
    cos, sin = (t.double()[at][:, None] for t in (cache.cos_cache, cache.sin_cache))
    a, b = raw[..., :h].double(), raw[..., h:n].double()
    y[..., :h] = a * cos[..., :h] - b * sin[..., :h]
    y[..., h:n] = b * cos[..., h:] + a * sin[..., h:]
    bound[..., :h], bound[..., h:n] = (b * sin[..., :h]).abs(), (a * sin[..., h:]).abs()
    bound = 1.001 * (2.0 ** -24 * (bound + y.abs()) + (u if x.dtype == BF16 else 0.0) * y.abs()) + 1e-44
    bound[..., n:] = 0
    return y, bound, raw


def check(cache, heads, T, pos, layout, seed=0, **kw):
    from logkv_b200 import log_kv_rotate
    q, k, _ = projected(cache, heads, T, seed, **kw)
    qo, ko, raw = log_kv_rotate(cache, q, k, pos, layout=layout)
    at = pos if pos is not None else cache.token_count + torch.arange(T, device="cuda")
    at = at.to("cuda")
    at = at if at.dim() == 2 else at[None]
    for x, got in ((q, qo), (k, ko)):
        want, bound, halves = reference(cache, x, at, layout == "interleaved")
        assert got.shape == x.shape and got.dtype == x.dtype
        assert ((got.double() - want).abs() <= bound).all()
    assert torch.equal(raw, halves)
    if layout == "half":
        assert raw is k
    assert cache.read_status() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,D,n", [(BF16, 128, 128), (BF16, 64, 16), (BF16, 64, 24), (BF16, 80, 80), (BF16, 64, 10),
                                       (BF16, 256, 2), (F32, 64, 64), (F32, 64, 8), (F32, 36, 20), (F32, 128, 6)])
def test_rotation(dtype, D, n, layout):
    cache = make(dtype, D=D, n=n)
    for T, shape in ((1, "row"), (7, "all"), (130, "row")):
        base = torch.randint(0, 512 - T, (2, 1), generator=torch.Generator().manual_seed(T)) + torch.arange(T)
        pos = (base if shape == "row" else base[0]).to("cuda", torch.int32 if T == 7 else torch.int64)
        check(cache, 6, T, pos, layout, seed=T)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rotation_of_odd_strides_and_tables(dtype):
    for tables in (F32, BF16):
        cache = make(dtype, B=3, G=1, D=64, n=32, tables=tables)
        pos = torch.tensor([[511, 0, 3], [1, 1, 1], [5, 400, 2]], device="cuda")
        check(cache, 5, 3, pos, "half", odd=True)
        check(cache, 5, 3, pos, "interleaved", odd=True)
        check(cache, 1, 3, pos[0].int(), "half", fused=False)
        check(cache, 2, 3, pos.T.contiguous().T, "half")           # strided positions
        check(cache, 2, 3, torch.tensor([9, 8, 7]), "half")        # positions on the host
        cache.token_count = 17
        check(cache, 2, 3, None, "half")
    none = make(dtype, n=0)
    from logkv_b200 import log_kv_rotate
    q, k, _ = projected(none, 4, 5, 1)
    qo, ko, _ = log_kv_rotate(none, q, k, torch.arange(5))
    assert torch.equal(qo, q) and torch.equal(ko, k)
    assert log_kv_rotate(none, q[:, :, :0], k[:, :, :0])[0].shape == (2, 4, 0, 64)


def test_rotation_of_many_rows():
    """More items than one wave, with every head of a token in one thread."""
    cache = make(BF16, B=4, G=4, D=128, rows=4096)
    pos = torch.randint(0, 4096, (4, 3001), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    check(cache, 20, 3001, pos, "half")
    check(cache, 20, 3001, pos, "interleaved")


def test_attention_does_not_depend_on_the_layout():
    """An interleaved checkpoint's scores are those of its features sorted into halves."""
    from logkv_b200 import log_kv_rotate
    cache = make(F32, D=64, n=48)
    q, k, _ = projected(cache, 2, 9, 5)
    pos = torch.arange(9, device="cuda") * 50
    order = torch.cat([torch.arange(0, 48, 2), torch.arange(1, 48, 2), torch.arange(48, 64)]).cuda()
    a = log_kv_rotate(cache, q, k, pos, layout="interleaved")
    b = log_kv_rotate(cache, q[..., order], k[..., order], pos)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_positions_outside_the_tables():
    from logkv_b200 import log_kv_rotate
    cache = make(F32, rows=100)
    q, k, _ = projected(cache, 2, 4, 2)
    pos = torch.tensor([3, 100, -1, 1 << 40], device="cuda")
    got = log_kv_rotate(cache, q, k, pos)
    want = log_kv_rotate(cache, q, k, torch.tensor([3, 99, 0, 99]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert cache.read_status() == 1 << 16


def state(cache):
    out = dict(cache.named_buffers())
    out.update(ends=cache._recent_ends, span_len=cache._span_len, span_count=cache._span_count)
    return {name: t.clone() for name, t in out.items() if t is not None}


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,n,gran", [(BF16, 64, 64), (F32, 24, 16), (BF16, 20, 64)])
def test_append_equals_rotating_and_appending(dtype, n, gran, layout):
    """Chunks that fit, pairs, a chunk whose flush is the window's next one and one that flushes several times."""
    from logkv_b200 import log_kv_rotate
    a, b = (make(dtype, n=n, granularity=gran) for _ in range(2))
    start = torch.tensor([[0], [40]], device="cuda")
    for step, T in enumerate((40, 2, 22, 1, 64, 2, 30)):
        _, k, v = projected(a, 2, T, step)
        gen = torch.Generator().manual_seed(step)
        ends = torch.rand(2, T, generator=gen) < 0.2
        pos = None if step == 1 else start + torch.arange(T, device="cuda")
        kw = dict(span_ends=ends.tolist()) if step % 2 else dict(span_ends_device=ends.cuda())
        a.add_recent_rotated(k, v, input_pos=pos, layout=layout, **kw)
        _, kr, raw = log_kv_rotate(b, torch.cat([k, k], 1), k, pos, layout=layout)
        b.add_recent(kr, v, k_raw=raw, input_pos=pos, span_ends=ends.tolist())
        start = start + T
        assert a.recent_count == b.recent_count and a.token_count == b.token_count
        assert a._ladder_epoch == b._ladder_epoch
        x, y = state(a), state(b)
        for name in x:
            assert torch.equal(x[name], y[name]), (step, name)
    assert a.read_status() == b.read_status() == 0
    assert a._flush_cursor > 0


def test_append_records_the_op_log():
    from logkv_b200 import log_kv_rotate
    a, b = make(F32), make(F32)
    for c in (a, b):
        c.begin_op_log()
    for step, T in enumerate((64, 64, 10)):
        _, k, v = projected(a, 2, T, step)
        ends = [[False] * T] * 2
        _, kr, raw = log_kv_rotate(b, torch.cat([k, k], 1), k)
        a.add_recent_rotated(k, v, span_ends=ends, record_op_log=True)
        b.add_recent(kr, v, k_raw=raw, span_ends=ends, record_op_log=True)
    for x, y in zip(a.take_op_log(), b.take_op_log()):
        assert torch.equal(x, y)


def test_capture_and_replay():
    """Captured with the buffers' first contents, replayed on others; nothing of the capture stays."""
    from logkv_b200 import log_kv_rotate
    cache = make(BF16, D=128)
    q, k, v = (t.contiguous() for t in projected(cache, 4, 3, 1))
    pos = torch.tensor([[1, 2, 3], [7, 8, 9]], device="cuda")
    ends = torch.zeros(2, 3, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        log_kv_rotate(cache, q, k, pos)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = log_kv_rotate(cache, q, k, pos, layout="interleaved")
            cache.add_recent_rotated(k, v, input_pos=pos, span_ends_device=ends)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (2, 3):
        for t, new in zip((q, k, v), projected(cache, 4, 3, seed)):
            t.copy_(new)
        pos += 100
        ends.bitwise_xor_(1)
        graph.replay()
        want = log_kv_rotate(cache, q, k, pos, layout="interleaved")
        for x, y in zip(out, want):
            assert torch.equal(x, y)
        assert torch.equal(cache.recent_k[:, :, :3], log_kv_rotate(cache, q, k, pos)[1])
        assert torch.equal(cache.recent_k_raw[:, :, :3], k) and torch.equal(cache.recent_v[:, :, :3], v)
        assert torch.equal(cache.recent_pos[:, :3], pos) and torch.equal(cache._recent_ends[:, :3], ends)
        assert not cache.recent_k[:, :, 3:].any()


def test_two_streams():
    """Calls on two streams at once, each with its own inputs."""
    from logkv_b200 import log_kv_rotate
    cache = make(F32)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ins = [projected(cache, 2, 100, s) for s in range(2)]
    pos = torch.arange(100, device="cuda")
    want = [log_kv_rotate(cache, q, k, pos) for q, k, _ in ins]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = log_kv_rotate(cache, *ins[i][:2], pos)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_repeated_calls_are_checked_like_the_first():
    """The host binding takes calls that fit; everything else is refused or done as the first call is."""
    from logkv_b200 import log_kv_rotate as f
    cache = make(F32, rows=100, window=16)
    q, k, v = projected(cache, 4, 3, 1)
    p, ends = torch.arange(3, device="cuda"), torch.zeros(2, 3, dtype=torch.uint8, device="cuda")
    want = f(cache, q, k, p)
    cache.add_recent_rotated(k, v, input_pos=p, span_ends_device=ends)
    assert cache._rotary is not None
    for args, kw, match in [
            ((q[:1], k, p), {}, "q must be"), ((q[0], k, p), {}, "q must be"), ((q.bfloat16(), k, p), {}, "q must be"),
            ((q, k[:, :1], p), {}, "k must be"), ((q, k[:, :, :2], p), {}, "k must be"), ((q[:, :3], k, p), {}, "multiple"),
            ((q, k, p[:2]), {}, "input_pos"), ((q, k, p.float()), {}, "integers"), ((q, k, [0, 1, 100]), {}, "tables"),
            ((q, k, p), {"layout": "pairs"}, "layout"), ((q.cpu(), k, p), {}, "device"), ((q, k.cpu(), p), {}, "device")]:
        with pytest.raises(ValueError, match=match):
            f(cache, *args, **kw)
    with pytest.raises(NotImplementedError):
        f(cache, q.clone().requires_grad_(), k, p)
    with pytest.raises((RuntimeError, ValueError)):
        f(cache, q.contiguous().to_sparse(), k, p)
    with torch.no_grad():
        assert torch.equal(f(cache, q.clone().requires_grad_(), k, p)[0], want[0])
    assert torch.equal(f(cache, q, k, [0, 1, 2])[0], want[0]) and torch.equal(f(cache, q, k, p.int())[1], want[1])
    last = q.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    assert torch.equal(f(cache, last, k, p)[0], want[0])
    assert cache.recent_count == 3
    bad = lambda *a, **kw: cache.add_recent_rotated(*a, **{"span_ends_device": ends, **kw})  # noqa: E731
    for args, kw, match in [((k[0], v), {}, "k_raw must be"), ((k, v[:, :, :2]), {}, "v must be"), ((k.bfloat16(), v), {}, "k_raw must be"),
                            ((k, v), {"input_pos": p[:2]}, "input_pos"), ((k, v), {"span_ends_device": ends[:1]}, "span boundaries"),
                            ((k, v.cpu()), {}, "device"), ((k, v), {"layout": 1}, "layout")]:
        with pytest.raises(ValueError, match=match):
            bad(*args, **kw)
    assert cache.recent_count == cache.token_count == 3
    bad(k, v, span_ends_device=ends.bool())
    cache.token_count = 4095
    with pytest.raises(RuntimeError, match="token overflow"):
        bad(k, v)
    cache.token_count = 6
    other = cache.cos_cache.flip(0).contiguous()          # other tables take over at once
    cache.cos_cache, cache.sin_cache = other, cache.sin_cache.flip(0).contiguous()
    assert torch.equal(f(cache, q, k, 99 - p)[0], want[0])
    for dtype in (BF16, F32):                             # of another type, too
        cache.cos_cache, cache.sin_cache = cache.cos_cache.to(dtype), cache.sin_cache.to(dtype)
        for _ in range(2):
            check(cache, 4, 3, p, "half")
    assert cache.read_status() == 0
