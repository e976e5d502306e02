"""Attention of rows that share a prefix (log_kv_shared_attention) against its 64-bit form, and the decoding steps that
use it (LogKVDecoder.step_raw, LogKVBeams.step and advance)."""
from __future__ import annotations

import pytest
import torch

from hypotheses import make_cache

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
NAN = float("nan")


def forked(dtype=BF16, N=2, W=3, w0=40, R=60, seed=0, **kw):
    """A cache of N x W rows, those of a request equal up to window row w0."""
    cache = make_cache(dtype, B=N * W, R=R, seed=seed, **kw)
    cache.reorder_batch(torch.arange(N, device="cuda").mul_(W).repeat_interleave(W))
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    for t in (cache.recent_k, cache.recent_v):
        t[:, :, w0:R] = torch.randn(t[:, :, w0:R].shape, generator=gen, device="cuda").to(dtype)
    return cache


def fresh(cache, rf, T, Tk, seed=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, G, D = cache.batch_size, cache.n_groups, cache.k_dim
    mk = lambda h, t: torch.randn(B, t, h, D, generator=gen, device="cuda").to(cache.level_k.dtype).transpose(1, 2)  # noqa: E731
    return mk(G * rf, T), mk(G, Tk), mk(G, Tk)


def run(cache, q, k, v, W, w0, causal=True, scale=None, **kw):
    from logkv_b200 import log_kv_shared_attention
    scale = cache.k_dim ** -0.5 if scale is None else scale
    return log_kv_shared_attention(cache, q, k, v, scale, beams=W, window_from=w0, causal_tail=None if causal else 0, **kw)


def reference(cache, q, k, v, causal, scale=None):
    """(64-bit attention of every row over its own prefix, window and new tokens, bound on a kernel's distance).

    The bound is that of the tree attention's tests: probabilities reach the value product in the storage type (bf16:
    half a step, u, of each), the output is rounded once; scores are float32 dot products of D + 2 terms, and the sums
    over S keys are off by at most (S + 32) 2^-24, once in the numerator and once in the denominator."""
    rs = cache._read
    B, H, T, D = q.shape
    G, R, Tk = cache.n_groups, cache.recent_count, k.size(2)
    rf, f64 = H // G, torch.float64
    scale = D ** -0.5 if scale is None else scale
    want = torch.zeros(B, H, T, D, dtype=f64, device=q.device)
    bound = torch.zeros_like(want)
    u = torch.finfo(q.dtype).eps / 2
    p_round = u if q.dtype == BF16 else 0.0
    qx = float(torch.tensor(1.0 / scale, dtype=q.dtype))
    late = torch.ones(T, Tk, dtype=torch.bool, device=q.device).triu(1) if causal else None
    for b in range(B):
        for g in range(G):
            n = int(rs.length[b, g])
            key = torch.cat([rs.pk[b, g, :n], cache.recent_k[b, g, :R], k[b, g]]).to(f64)
            val = torch.cat([rs.pv[b, g, :n], cache.recent_v[b, g, :R], v[b, g]]).to(f64)
            mass = torch.zeros(key.size(0), dtype=f64, device=q.device)
            mass[:n] = rs.mass[b, g, :n].to(f64)
            qq = q[b, g * rf:(g + 1) * rf].to(f64)
            z = scale * (qq @ key.T + qx * mass)
            reach = scale * (qq.abs() @ key.abs().T + qx * mass).amax()
            if causal:
                z[..., n + R:] = z[..., n + R:].masked_fill(late, float("-inf"))
            p = torch.softmax(z, -1)
            o, a = p @ val, p @ val.abs()
            e = 2 * (D + 4) * 2.0 ** -24 * reach + 2 * (key.size(0) + 32) * 2.0 ** -24
            want[b, g * rf:(g + 1) * rf] = o
            bound[b, g * rf:(g + 1) * rf] = (p_round + e) * a + u * o.abs() * (1 + p_round) + 2.0 ** -40
    return want, bound


def check(cache, q, k, v, got, causal=True, scale=None):
    want, bound = reference(cache, q, k, v, causal, scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max()
    assert cache.read_status() == 0


@pytest.mark.parametrize("dtype,D,rf,T,Tk,N,W,w0,R,levels", [
    (BF16, 64, 2, 1, 1, 1, 1, 40, 60, 3), (BF16, 64, 2, 1, 1, 2, 3, 0, 0, 0), (BF16, 128, 2, 1, 2, 2, 4, 60, 60, 3),
    (BF16, 128, 1, 1, 1, 3, 16, 17, 33, 2), (BF16, 128, 5, 1, 2, 1, 7, 0, 200, 3), (BF16, 64, 3, 2, 2, 2, 5, 100, 131, 0),
    (BF16, 64, 8, 3, 3, 1, 11, 64, 64, 3), (BF16, 32, 4, 1, 1, 2, 9, 30, 61, 3), (BF16, 16, 2, 5, 5, 2, 3, 3, 5, 1),
    (BF16, 256, 2, 1, 2, 1, 4, 90, 100, 2), (BF16, 64, 2, 2, 5, 2, 3, 9, 30, 2), (F32, 32, 2, 3, 40, 1, 2, 9, 30, 2), (BF16, 128, 2, 40, 40, 1, 3, 50, 77, 2), (BF16, 64, 1, 1, 1, 1, 130, 9, 10, 1),
    (F32, 64, 2, 1, 1, 2, 3, 40, 60, 3), (F32, 128, 3, 1, 2, 1, 5, 0, 100, 2), (F32, 32, 7, 2, 2, 2, 2, 16, 16, 0),
    (F32, 16, 1, 9, 9, 1, 4, 0, 0, 0), (F32, 64, 2, 33, 33, 1, 2, 20, 50, 1)])
def test_against_64_bits(dtype, D, rf, T, Tk, N, W, w0, R, levels):
    """One row to many per prefix; shared parts and own parts that are empty, end inside a tile or on its edge; one
    query over a pending token and itself, and causal ones."""
    cache = forked(dtype, N, W, w0, R, D=D, levels=levels, seed=D + W)
    q, k, v = fresh(cache, rf, T, Tk)
    check(cache, q, k, v, run(cache, q, k, v, W, w0, causal=T == Tk), causal=T == Tk)
    if T == Tk and T < 10:
        check(cache, q, k, v, run(cache, q, k, v, W, w0, causal=False), causal=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,W,G", [(1, 2, 1), (1, 33, 8), (20, 2, 1), (24, 2, 8), (5, 40, 2)])
def test_lane_counts(dtype, N, W, G):
    """From one shared lane (its keys split over all SMs) to more lanes than SMs (one split each)."""
    cache = forked(dtype, N, W, 150, 200, G=G, D=64, seed=N)
    q, k, v = fresh(cache, 2, 1, 2)
    check(cache, q, k, v, run(cache, q, k, v, W, 150, causal=False), causal=False)


@pytest.mark.parametrize("dtype,D,rf,T,w0", [(BF16, 256, 2, 1, 100), (BF16, 128, 9, 2, 100), (BF16, 64, 9, 2, 60), (BF16, 32, 3, 2, 119),
                                             (BF16, 16, 1, 1, 0), (F32, 128, 2, 1, 100), (F32, 64, 9, 2, 110), (F32, 16, 1, 5, 90)])
def test_own_lanes_side_by_side(dtype, D, rf, T, w0):
    """More own lanes than CTAs run at once: one or two warps to a lane, lanes of several row tiles, a last CTA that is
    not full."""
    for N, W, G in ((33, 3, 4), (37, 5, 3)):
        cache = forked(dtype, N, W, w0, 120, G=G, D=D, levels=1, seed=D + N)
        q, k, v = fresh(cache, rf, T, T)
        check(cache, q, k, v, run(cache, q, k, v, W, w0))


@pytest.mark.parametrize("dtype,D,N,W,rf", [(BF16, 128, 20, 3, 8), (BF16, 64, 20, 2, 30), (BF16, 128, 30, 2, 2), (F32, 64, 20, 2, 2)])
def test_long_splits(dtype, D, N, W, rf):
    """One or two splits per lane, many key tiles each (the stages are used over and over), long own parts."""
    cache = forked(dtype, N, W, 1200, 1999, G=8, D=D, recent=2048, max_seq=8192, seed=21)
    q, k, v = fresh(cache, rf, 1, 1)
    check(cache, q, k, v, run(cache, q, k, v, W, 1200))


@pytest.mark.parametrize("dtype,rf", [(BF16, 2), (BF16, 8), (F32, 2)])
def test_equals_chunk_attention(dtype, rf):
    """Each side is off by its own bound; with one beam, and with everything the row's own, too."""
    from logkv_b200 import log_kv_chunk_attention
    cache = forked(dtype, 2, 4, 33, 90, D=128, seed=6)
    q, k, v = fresh(cache, rf, 1, 2)
    chunk = log_kv_chunk_attention(cache, q, k, v, 128 ** -0.5, 0.0, causal_tail=0)
    _, bound = reference(cache, q, k, v, False)
    for W, w0 in ((4, 33), (2, 33), (1, 90), (1, 0), (4, 0)):
        got = run(cache, q, k, v, W, w0, causal=False)
        assert ((got.double() - chunk.double()).abs() <= 2 * bound).all()


@pytest.mark.parametrize("dtype,rf", [(BF16, 2), (BF16, 8), (F32, 3)])
def test_shared_keys_are_read_from_the_first_row(dtype, rf):
    """What the other rows hold of the prefix and of the shared window may be anything; what a row holds behind it,
    or brings as new tokens, is nobody else's."""
    W, w0, R = 4, 37, 70
    cache = forked(dtype, 2, W, w0, R, D=64, seed=7)
    q, k, v = fresh(cache, rf, 1, 1)
    clean = run(cache, q, k, v, W, w0)
    other = torch.arange(2 * W, device="cuda") % W != 0
    saved = [(t, t.clone()) for t in (cache._read.pk, cache._read.pv, cache._read.mass, cache.recent_k, cache.recent_v)]
    for t, _ in saved[:3]:
        t[other] = NAN
    for t in (cache.recent_k, cache.recent_v):
        part = t[:, :, :w0]
        part[other] = NAN
    assert torch.equal(run(cache, q, k, v, W, w0), clean)
    for t, old in saved:
        t.copy_(old)
    for name in ("window", "new"):
        for bad in (NAN, float("inf")):
            t = cache.recent_v if name == "window" else v
            old = t.clone()
            t[5, 1, 60 if name == "window" else 0] = bad
            got = run(cache, q, k, v, W, w0)
            hit = torch.zeros(2 * W, 2 * rf, dtype=torch.bool, device="cuda")
            hit[5, rf:] = True
            assert not got[hit].isfinite().any()
            assert torch.equal(got[~hit], clean[~hit])
            t.copy_(old)
    # The window behind the fill, the prefix behind its length.
    cache.recent_k[:, :, R:], cache.recent_v[:, :, R:] = NAN, NAN
    for b in range(2 * W):
        for g in range(2):
            cache._read.pk[b, g, int(cache._read.length[b, g]):] = NAN
            cache._read.pv[b, g, int(cache._read.length[b, g]):] = NAN
            cache._read.mass[b, g, int(cache._read.length[b, g]):] = NAN
    assert torch.equal(run(cache, q, k, v, W, w0), clean)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F32, 64)])
def test_later_tokens_are_not_seen(dtype, D):
    """A new token with a non-finite V or K spoils the causal rows that see it and no other."""
    cache = forked(dtype, 1, 3, 20, 33, D=D, seed=8)
    T = 21
    q, k, v = fresh(cache, 2, T, T)
    clean = run(cache, q, k, v, 3, 20)
    for bad, where in ((NAN, "v"), (float("-inf"), "v"), (NAN, "k")):
        t = (k if where == "k" else v).clone()
        t[1, 0, 9, D // 2] = bad
        got = run(cache, q, t if where == "k" else k, t if where == "v" else v, 3, 20)
        hit = torch.zeros(3, 4, T, dtype=torch.bool, device="cuda")
        hit[1, :2, 9:] = True
        assert got[hit].isnan().all()
        assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("dtype,W", [(BF16, 4), (BF16, 12), (F32, 4)])
def test_large_scores(dtype, W):
    """Scores far apart: the running maximum keeps moving, and one part's weight underflows beside the other's."""
    cache = forked(dtype, 1, W, 200, 256, D=64, seed=9)
    cache.recent_k *= (1 + torch.arange(cache.recent_k.size(2), device="cuda") / 16.0)[:, None].to(dtype)
    q, k, v = fresh(cache, 2, 1, 1)
    check(cache, q, k, v, run(cache, q, k, v, W, 200))
    check(cache, q, k * 50, v, run(cache, q, k * 50, v, W, 200))


def test_layouts_of_inputs():
    """Strided, sliced, expanded and misaligned inputs; `out`."""
    cache = forked(BF16, 2, 3, 10, 30, D=64, seed=10)
    q, k, v = fresh(cache, 2, 2, 2)
    want = run(cache, q, k, v, 3, 10)
    assert torch.equal(run(cache, q.contiguous(), k.contiguous(), v.contiguous(), 3, 10), want)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(run(cache, odd, k, v, 3, 10), want)
    last = q.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    assert torch.equal(run(cache, last, k, v, 3, 10), want)
    out = torch.zeros_like(want)
    assert run(cache, q, k, v, 3, 10, out=out) is out and torch.equal(out, want)
    one = k[:, :, :1].expand(-1, -1, 2, -1)
    assert torch.equal(run(cache, q, one, v, 3, 10), run(cache, q, one.contiguous(), v, 3, 10))
    assert run(cache, q[:, :, :0], k[:, :, :0], v[:, :, :0], 3, 10).shape == (6, 4, 0, 64)


def test_streams_graphs_and_repeats():
    """Two captured graphs and eager calls on two streams, at once; every result the same as alone."""
    cache = forked(BF16, 2, 12, 300, 400, D=128, recent=512, seed=11)
    ins = [fresh(cache, 2, 1, 2, seed=s) for s in (1, 2)]
    want = [run(cache, *i, 12, 300, causal=False) for i in ins]
    small = [run(cache, *i, 4, 300, causal=False) for i in ins]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for s, i in zip(streams, ins):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            run(cache, *i, 12, 300, causal=False)
            with torch.cuda.graph(g, stream=s):
                outs.append((run(cache, *i, 12, 300, causal=False), run(cache, *i, 4, 300, causal=False)))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        eager = []
        for s, g, i in zip(streams, graphs, ins):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(run(cache, *i, 12, 300, causal=False))
        torch.cuda.synchronize()
        for n in range(2):
            assert torch.equal(outs[n][0], want[n]) and torch.equal(outs[n][1], small[n]) and torch.equal(eager[n], want[n])


def test_refusals():
    cache = forked(BF16, 2, 3, 10, 30, D=64)
    q, k, v = fresh(cache, 2, 1, 1)
    for W, w0, match in ((0, 10, "beams"), (4, 10, "beams"), (3, 31, "window_from"), (3, -1, "window_from")):
        with pytest.raises(ValueError, match=match):
            run(cache, q, k, v, W, w0)
    odd = make_cache(BF16, D=24, levels=0, R=4)
    with pytest.raises(ValueError, match="supported range"):
        run(odd, *fresh(odd, 1, 1, 1), 1, 0)


# ---------------------------------------------------------------- decoding steps
def tables_match(cache, T, pos):
    return torch.full((cache.batch_size, T), pos, device="cuda")


@pytest.mark.parametrize("layout,given", [("half", True), ("interleaved", True), ("half", False)])
def test_step_raw_equals_rotating_and_stepping(layout, given):
    """Cache and pending token bit for bit, over commits and flushes."""
    from logkv_b200 import log_kv_rotate
    from logkv_b200.decode import LogKVDecoder
    a, b = (LogKVDecoder(make_cache(BF16, B=3, G=2, D=64, R=20, recent=32, granularity=16, seed=4), 0.125) for _ in range(2))
    for d in (a, b):
        d.cache.token_count = 700
    for step in range(30):
        q, k, v = fresh(a.cache, 2, 1, 1, seed=step)
        ends = (torch.arange(3, device="cuda") + step) % 4 == 0
        ends = ends.to(torch.uint8).view(3, 1)
        pos = torch.tensor([[700], [500], [600]], device="cuda") + step if given else None
        at = pos if given else torch.full((3, 1), b.cache.token_count + int(b.pending), device="cuda")
        x = a.step_raw(q, k, v, input_pos=pos, layout=layout, span_ends_device=ends)
        qr, kr, raw = log_kv_rotate(b.cache, q, k, at, layout=layout)
        y = b.step(qr, kr, v, k_raw=raw, input_pos=pos, span_ends_device=ends)
        assert torch.equal(x, y), step
        for name in ("_k", "_v", "_kr", "_ends") + (("_pos",) if given else ()):
            assert torch.equal(getattr(a, name), getattr(b, name)), (step, name)
        for (name, s), (_, t) in zip(a.cache.named_buffers(), b.cache.named_buffers()):
            assert torch.equal(s, t), (step, name)
    assert a.cache._flush_cursor > 0
    q, k, v = fresh(a.cache, 2, 1, 1)
    for args, kw, match in (((q[:, :3], k, v), {}, "q must be"), ((q, k[:2], v), {}, "k_raw must be"),
                            ((q, k, v.float()), {}, "v must be"), ((q, k, v), {"layout": "x"}, "layout"),
                            ((q, k, v), {"shared": (2, 0)}, "shared must be"), ((q, k, v), {"shared": (3, 99)}, "shared must be")):
        with pytest.raises(ValueError, match=match):
            a.step_raw(*args, **kw)


@pytest.mark.parametrize("D,rf,steps", [(64, 2, 50), (128, 8, 12), (64, 3, 12), (64, 5, 50)])
def test_beam_steps(D, rf, steps):
    """LogKVBeams.step and advance with penalties, biases and masks, against the same steps without sharing over
    rows copied by indexing; long enough in the first case that the window flushes in between."""
    from logkv_b200 import adjust_logits, beam_select, log_kv_rotate
    from logkv_b200.decode import LogKVBeams, LogKVDecoder
    N, W, V = 2, 4, 203
    mk = lambda: LogKVDecoder(make_cache(BF16, B=N * W, G=2, D=D, K=4, levels=2, R=20, recent=32, granularity=16, seed=22),  # noqa: E731
                              D ** -0.5)
    ours, theirs = mk(), mk()
    penalties = dict(repetition=1.3, presence=0.2, frequency=0.1)
    beams = LogKVBeams([ours], N, W, penalties=penalties)
    prompt = torch.tensor([[5, 9, 200], [7, -1, -1]], device="cuda")
    beams.fork(prompt)
    theirs.reorder(torch.arange(N, device="cuda").mul_(W).repeat_interleave(W))
    past = [prompt[i // W].tolist() for i in range(N * W)]
    gen = torch.Generator(device="cuda").manual_seed(5)
    heads = torch.randn(2 * rf * D, V, generator=gen, device="cuda") * 0.3
    mask = torch.full(((V + 31) // 32,), -1, dtype=torch.int32, device="cuda")
    mask[0] = -1 << 4
    bias = (torch.tensor([11, 12, 11], device="cuda"), torch.tensor([1.0, -2.0, 0.5], device="cuda"))
    scores = beams.scores.clone()
    shared = []
    for step in range(steps):
        q, k, v = fresh(ours.cache, rf, 1, 1, seed=step)
        pos = tables_match(ours.cache, 1, 500 + step)
        ends = torch.zeros(N * W, 1, dtype=torch.uint8, device="cuda")
        shared.append(beams._window_from(0) is not None)
        x = beams.step(0, q, k, v, input_pos=pos, span_ends_device=ends)
        qr, kr, raw = log_kv_rotate(theirs.cache, q, k, pos)
        if rf & (rf - 1):      # beyond log_kv_chunk_attention: one row at a time with nothing shared
            y = theirs.step(qr, kr, v, k_raw=raw, input_pos=pos, span_ends_device=ends, shared=(1, 0))
        else:
            y = theirs.step(qr, kr, v, k_raw=raw, input_pos=pos, span_ends_device=ends)
        # Both sides are within a few 2^-8 of the largest value: rounded probabilities, one rounding of the output.
        top = max(float(t.abs().max()) for t in (v, ours.cache.recent_v, ours.cache._read.pv))
        assert ((x.float() - y.float()).abs() <= 4.2 * 2.0 ** -8 * top).all(), step
        logits = x.float().reshape(N * W, -1) @ heads
        tokens, rows = beams.advance(logits, bias=bias, mask=mask)
        width = max(len(p) for p in past)
        hist = torch.tensor(past, device="cuda").view(N, W, width)
        adjusted = adjust_logits(logits.view(N, W, V), history=hist, prompt=3, bias=bias, mask=mask, **penalties)
        s, r, t = beam_select(adjusted, scores, W, keep_places=True)
        assert torch.equal(s, beams.scores) and torch.equal(r.view(-1), rows) and torch.equal(t.view(-1), tokens)
        scores = s.clone()
        assert (t[s > -float("inf")] >= 4).all()
        past = [past[i] + [j] for i, j in zip(rows.tolist(), tokens.tolist())]
        assert torch.equal(beams._tokens[:, :beams._length].cpu(), torch.tensor(past, dtype=torch.int32))
        theirs.reorder(rows)
        for (name, s1), (_, t1) in zip(ours.cache.named_buffers(), theirs.cache.named_buffers()):
            if name not in ("recent_k", "recent_v", "recent_k_raw", "recent_pos"):
                assert torch.equal(s1, t1), (step, name)
            else:
                R = ours.cache.recent_count
                s1, t1 = (z[:, :R] if z.dim() == 2 else z[:, :, :R] for z in (s1, t1))
                assert torch.equal(s1, t1), (step, name)
    assert all(shared) if steps == 12 else shared[0] and not shared[-1]
    assert (ours.cache._flush_cursor > 0) == (steps == 50)


def test_beams_keep_more_tokens_than_they_began_with():
    from logkv_b200.decode import LogKVBeams, LogKVDecoder
    d = LogKVDecoder(make_cache(BF16, B=2, G=1, D=16, levels=0, R=3), 0.25)
    beams = LogKVBeams([d], 1, 2, penalties={"presence": 5.0})
    with pytest.raises(RuntimeError, match="fork"):
        beams.advance(torch.zeros(2, 50, device="cuda"))
    beams.fork()
    gen = torch.Generator(device="cuda").manual_seed(1)
    seen = []
    for _ in range(300):
        seen.append(beams.advance(torch.randn(2, 900, generator=gen, device="cuda")))
    assert beams._tokens.size(1) == 512 and beams._length == 300
    chain = 0
    for i in range(299, -1, -1):           # the first row's tokens, followed back through the rows it came from
        assert int(beams._tokens[0, i]) == int(seen[i][0][chain])
        chain = int(seen[i][1][chain])
    for kw in ({"penalties": {"temperature": 1.0}},):
        with pytest.raises(ValueError):
            LogKVBeams([d], 1, 2, **kw)
    with pytest.raises(ValueError, match="penalties only"):
        LogKVBeams([d], 1, 2).fork(torch.zeros(1, 3, dtype=torch.int64, device="cuda"))
    for bad in (torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(1, 3, device="cuda"), torch.zeros(1, 3, dtype=torch.int64)):
        with pytest.raises(ValueError, match="prompt must be"):
            beams.fork(bad)


def test_repeated_calls_are_checked_like_the_first():
    """The host binding takes calls that fit; everything else is refused or done as the first call is."""
    cache = forked(F32, 2, 3, 10, 30, D=64)
    q, k, v = fresh(cache, 2, 2, 2)
    want = run(cache, q, k, v, 3, 10)
    assert cache._read.native_shared is not None and torch.equal(run(cache, q, k, v, 3, 10), want)
    f = lambda q, k, v, W=3, w0=10, **kw: run(cache, q, k, v, W, w0, **kw)  # noqa: E731
    for args, kw, match in [
            ((q[:1], k, v), {}, "q must be"), ((q[0], k, v), {}, "q must be"), ((q.bfloat16(), k, v), {}, "q must be"),
            ((q, k[:, :1], v), {}, "k must be"), ((q, k, v[:, :, :1]), {}, "v shape"), ((q, k, v.bfloat16()), {}, "dtype"),
            ((q[:, :, :1], k, v), {}, "same tokens"), ((q[:, :3], k, v), {}, "multiple"), ((q.cpu(), k, v), {}, "device"),
            ((q, k, v), {"W": 4}, "beams"), ((q, k, v), {"W": 0}, "beams"), ((q, k, v), {"w0": 31}, "window_from"),
            ((q, k, v), {"w0": -1}, "window_from")]:
        with pytest.raises(ValueError, match=match):
            f(*args, **kw)
    from logkv_b200 import log_kv_shared_attention
    with pytest.raises(ValueError, match="causal_tail"):
        log_kv_shared_attention(cache, q, k, v, 0.125, beams=3, window_from=10, causal_tail=1)
    with pytest.raises(NotImplementedError):
        f(q.clone().requires_grad_(), k, v)
    last = q.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    assert torch.equal(f(last, k, v), want)
    wide = log_kv_shared_attention(cache, q, k, v, 0.125, beams=torch.tensor(3), window_from=10.0)
    assert torch.equal(wide, want)
    # A flush makes the prefix anew, and the cache's rows are then what they are.
    cache.recent_count = 20
    check(cache, q, k, v, run(cache, q, k, v, 3, 10))
    cache.add_recent(torch.randn_like(cache.recent_k[:, :, :256]), torch.randn_like(cache.recent_k[:, :, :256]),
                     k_raw=torch.randn_like(cache.recent_k[:, :, :256]), span_ends=[[False] * 256] * 6)
    assert cache._flush_cursor == 1
    check(cache, q, k, v, run(cache, q, k, v, 1, 0))


@pytest.mark.parametrize("shared", [None, (2, 12)])
def test_captured_pair_of_steps(shared):
    """Two steps (a pending token, then the pair's commit) captured once and replayed on other tokens, against the same
    steps run at once."""
    from logkv_b200.decode import LogKVDecoder
    mk = lambda: LogKVDecoder(make_cache(BF16, B=4, G=2, D=64, R=20, recent=64, seed=4), 0.125)  # noqa: E731
    a, b = mk(), mk()
    for d in (a, b):
        d.reorder(torch.tensor([0, 0, 2, 2], device="cuda"))
    ins = [[t.contiguous() for t in fresh(a.cache, 2, 1, 1, seed=s)] + [torch.full((4, 1), 90 + s, device="cuda"),
                                                                       torch.zeros(4, 1, dtype=torch.uint8, device="cuda")]
           for s in (0, 1)]

    def two(d, ins):
        return [d.step_raw(q, k, v, input_pos=p, span_ends_device=e, shared=shared) for q, k, v, p, e in ins]

    two(mk(), ins)           # everything that a first call sets up
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        from logkv_b200.attention import refresh_prefix
        refresh_prefix(a.cache)
        with torch.cuda.graph(graph, stream=side):
            out = two(a, ins)
    torch.cuda.current_stream().wait_stream(side)
    for i, (q, k, v, p, e) in enumerate(ins):
        for old, new in zip((q, k, v), fresh(a.cache, 2, 1, 1, seed=10 + i)):
            old.copy_(new)
        p += 7
        e.fill_(1)
    graph.replay()
    want = two(b, ins)
    for x, y in zip(out, want):
        assert torch.equal(x, y)
    for (name, s), (_, t) in zip(a.cache.named_buffers(), b.cache.named_buffers()):
        assert torch.equal(s, t), name
    assert torch.equal(a.cache._recent_ends, b.cache._recent_ends) and a.cache.recent_count == b.cache.recent_count == 22
