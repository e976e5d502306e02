"""Tree attention of drafted tokens over the cache against its 64-bit form, at the sizes and trees
where it can go wrong."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hypotheses import make_cache, random_tree, tree_reference, visible

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def drafts(cache, rf, T, seed=1):
    """q, k, v of T drafted tokens as a projection leaves them ([B, T, heads, D], heads seen first)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda h: torch.randn(cache.batch_size, T, h, cache.k_dim, generator=gen,  # noqa: E731
                               device="cuda").to(cache.level_k.dtype).transpose(1, 2)
    return mk(cache.n_groups * rf), mk(cache.n_groups), mk(cache.n_groups)


def check(cache, q, k, v, p, out, scale=None):
    scale = cache.k_dim ** -0.5 if scale is None else scale
    want, bound = tree_reference(cache, q, k, v, scale, visible(p))
    torch.cuda.synchronize()
    err = (out.double() - want).abs()
    worst = (err / bound).max().item()
    assert torch.isfinite(out).all()
    assert worst <= 1.0, (worst, err.max().item())


def run(cache, q, k, v, p, **kw):
    from logkv_b200 import log_kv_tree_attention
    out = log_kv_tree_attention(cache, q, k, v, cache.k_dim ** -0.5,
                                torch.from_numpy(p).to("cuda", torch.int32), **kw)
    torch.cuda.synchronize()
    assert int(cache._read.status.item()) == 0
    return out


@pytest.mark.parametrize("dtype,D,rf,T,R,levels", [
    (BF16, 128, 2, 1, 100, 3), (BF16, 128, 2, 7, 100, 3), (BF16, 128, 1, 16, 1, 2), (BF16, 128, 1, 17, 0, 3),
    (BF16, 128, 3, 11, 256, 3), (BF16, 128, 2, 64, 100, 4), (BF16, 128, 5, 61, 77, 3), (BF16, 128, 8, 33, 129, 1),
    (BF16, 128, 2, 65, 64, 0), (BF16, 128, 1, 256, 100, 3), (BF16, 128, 7, 130, 31, 3), (BF16, 64, 2, 5, 100, 3),
    (BF16, 64, 4, 40, 255, 3), (BF16, 64, 3, 100, 0, 0), (BF16, 64, 16, 16, 90, 3), (BF16, 32, 2, 9, 100, 3),
    (BF16, 32, 3, 50, 63, 3), (BF16, 16, 4, 21, 100, 3), (BF16, 16, 1, 1, 0, 0), (BF16, 256, 2, 20, 100, 3),
    (BF16, 256, 1, 3, 17, 0), (BF16, 128, 8, 256, 200, 3), (BF16, 64, 12, 256, 0, 2), (BF16, 32, 3, 256, 100, 3),
    (F32, 128, 3, 256, 100, 3), (BF16, 128, 17, 1, 40, 3), (F32, 32, 9, 2, 40, 3),
    (F32, 64, 2, 1, 100, 3), (F32, 64, 3, 13, 100, 3), (F32, 128, 2, 40, 65, 3), (F32, 128, 5, 7, 0, 0),
    (F32, 32, 4, 33, 256, 2), (F32, 16, 2, 70, 31, 3), (F32, 16, 1, 2, 0, 3)])
def test_tree_matches_64_bits(dtype, D, rf, T, R, levels):
    cache = make_cache(dtype, B=2, G=2, D=D, levels=levels, R=R, seed=T)
    q, k, v = drafts(cache, rf, T)
    p = random_tree(np.random.RandomState(T), 2, T, absent=T // 4)
    check(cache, q, k, v, p, run(cache, q, k, v, p))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,G", [(1, 1), (1, 8), (17, 1), (40, 8)])
def test_tree_lane_counts(dtype, B, G):
    """From one lane (its keys split over all SMs) to more lanes than SMs (one split each)."""
    cache = make_cache(dtype, B=B, G=G, D=64, R=200, seed=B)
    q, k, v = drafts(cache, 2, 24)
    p = random_tree(np.random.RandomState(3), B, 24, absent=5)
    check(cache, q, k, v, p, run(cache, q, k, v, p))


@pytest.mark.parametrize("dtype,D,T,rf", [(BF16, 128, 40, 2), (BF16, 64, 60, 2), (BF16, 128, 200, 1), (BF16, 32, 10, 2),
                                          (BF16, 128, 8, 2), (F32, 64, 20, 2)])
def test_long_splits(dtype, D, T, rf):
    """One split per lane, many key tiles each (the stages are used over and over)."""
    cache = make_cache(dtype, B=40, G=8, D=D, R=1999, recent=2048, seed=21)
    q, k, v = drafts(cache, rf, T)
    p = random_tree(np.random.RandomState(22), 40, T, absent=5)
    check(cache, q, k, v, p, run(cache, q, k, v, p))


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 32), (F32, 64)])
def test_special_trees(dtype, D):
    """A chain (every token sees all before it), a star (none sees another), a batch row without any
    token, a subtree under an absent token."""
    T = 70
    cache = make_cache(dtype, B=4, D=D, R=50, seed=5)
    q, k, v = drafts(cache, 2, T)
    p = np.full((4, T), -1, np.int64)
    p[0] = np.arange(T) - 1
    p[2] = -2
    p[3] = np.arange(T) - 1
    p[3, 20] = -2
    out = run(cache, q, k, v, p)
    check(cache, q, k, v, p, out)
    assert (out[2] == 0).all() and (out[3, :, 20:] == 0).all() and (out[3, :, :20] != 0).any()


def test_chain_of_256_equals_chunk_attention():
    """A chain of drafts is the causal tail of chunk attention; each side is off by its own bound."""
    from logkv_b200 import log_kv_chunk_attention
    cache = make_cache(BF16, B=1, D=128, R=120, seed=6)
    q, k, v = drafts(cache, 2, 256)
    p = np.arange(256)[None] - 1
    got = run(cache, q, k, v, p)
    with torch.no_grad():
        chunk = log_kv_chunk_attention(cache, q, k, v, 128 ** -0.5, 0.0)
    _, bound = tree_reference(cache, q, k, v, 128 ** -0.5, visible(p))
    assert ((got.double() - chunk.double()).abs() <= 2 * bound).all()


@pytest.mark.parametrize("dtype,D,T", [(BF16, 128, 40), (BF16, 64, 6), (BF16, 32, 40), (F32, 64, 40)])
def test_values_in_masked_places(dtype, D, T):
    """Absent tokens may hold anything; a token with a non-finite V or K spoils the rows that see it and
    no other row."""
    cache = make_cache(dtype, B=3, D=D, R=33, seed=7)
    q, k, v = drafts(cache, 3, T)
    p = random_tree(np.random.RandomState(8), 3, T)
    p[:, -3:] = -2
    clean = run(cache, q, k, v, p)
    bad_q, bad_k, bad_v = q.clone(), k.clone(), v.clone()
    bad_q[:, :, -3:] = float("nan")
    bad_k[:, :, -3:] = float("inf")
    bad_v[:, :, -3:] = float("nan")
    assert torch.equal(run(cache, bad_q, bad_k, bad_v, p), clean)
    see = torch.from_numpy(visible(p)).cuda()
    for value, where in ((float("nan"), "v"), (float("-inf"), "v"), (float("nan"), "k")):
        bad = (k if where == "k" else v).clone()
        bad[0, 1, 2, D // 2] = value                # token 2 of row 0, group 1
        out = run(cache, q, bad if where == "k" else k, bad if where == "v" else v, p)
        hit = torch.zeros(3, 6, T, dtype=torch.bool, device="cuda")
        hit[0, 3:] = see[0, :, 2]
        assert out[hit].isnan().all()
        assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores(dtype):
    """Scores far apart (the running maximum keeps moving; most probabilities underflow)."""
    cache = make_cache(dtype, B=1, D=64, R=256, seed=9)
    cache.recent_k *= (1 + torch.arange(cache.recent_k.size(2), device="cuda") / 16.0)[:, None].to(dtype)
    q, k, v = drafts(cache, 2, 30)
    k = k * 20
    p = random_tree(np.random.RandomState(10), 1, 30)
    check(cache, q, k, v, p, run(cache, q, k, v, p))


def test_layouts_of_inputs():
    """Strided, misaligned and expanded inputs, shared and 64-bit parents, a given output."""
    from logkv_b200 import log_kv_tree_attention
    cache = make_cache(BF16, B=3, D=64, R=40, seed=11)
    q, k, v = drafts(cache, 2, 19)
    p = random_tree(np.random.RandomState(12), 1, 19, absent=4)
    p3 = np.repeat(p, 3, 0)
    want = run(cache, q, k, v, p3)
    scale = 64 ** -0.5
    dev = torch.from_numpy(p[0]).cuda()
    out = torch.full_like(want, 7.0).contiguous()
    assert log_kv_tree_attention(cache, q, k, v, scale, dev, out=out) is out
    assert torch.equal(out, want)
    assert torch.equal(log_kv_tree_attention(cache, q, k, v, scale, p[0].tolist()), want)
    assert torch.equal(log_kv_tree_attention(cache, q, k, v, scale, torch.from_numpy(p3).cuda().t().contiguous().t()), want)
    assert torch.equal(log_kv_tree_attention(cache, q, k, v, scale, dev.to(torch.int32).expand(3, 19)), want)
    odd = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731  (2-byte offset)
    assert torch.equal(log_kv_tree_attention(cache, odd(q), odd(k.contiguous()), v.contiguous(), scale, dev), want)
    one = k[:, :1].expand(-1, 2, -1, -1)
    assert torch.equal(log_kv_tree_attention(cache, q, one, v, scale, dev),
                       log_kv_tree_attention(cache, q, one.contiguous(), v, scale, dev))


def test_bad_parents_on_the_device():
    """Device values that are no parent count as absent and set bit 18 of the read status."""
    from logkv_b200 import log_kv_tree_attention
    cache = make_cache(BF16, B=2, D=64, R=40, seed=13)
    q, k, v = drafts(cache, 2, 21)
    p = random_tree(np.random.RandomState(14), 2, 21)
    p[0, 5], p[1, 3], p[1, 9] = 5, 1 << 40, -7
    out = log_kv_tree_attention(cache, q, k, v, 64 ** -0.5, torch.from_numpy(p).cuda())
    assert int(cache._read.status.item()) == 1 << 18
    check(cache, q, k, v, p, out)


def test_no_tokens_and_refusals():
    from logkv_b200 import log_kv_tree_attention as f
    cache = make_cache(BF16, B=2, D=64, R=40, seed=15)
    q, k, v = drafts(cache, 2, 4)
    assert f(cache, q[:, :, :0], k[:, :, :0], v[:, :, :0], 0.125, []).shape == (2, 4, 0, 64)
    with pytest.raises(ValueError, match="device"):
        f(cache, q.cpu(), k, v, 0.125, [-1, 0, 1, 2])
    with pytest.raises(ValueError, match="out must be"):
        f(cache, q, k, v, 0.125, [-1, 0, 1, 2], out=torch.empty(2, 4, 4, 64, device="cuda"))


def test_streams_and_graphs():
    """Calls on two streams at once, and two captured graphs replayed at once on new inputs."""
    from logkv_b200 import log_kv_tree_attention
    caches = [make_cache(BF16, B=2, D=128, R=200, seed=s) for s in (16, 17)]
    sets = [[t.contiguous() for t in drafts(c, 2, 30, seed=s)] for s, c in enumerate(caches)]
    p = random_tree(np.random.RandomState(18), 2, 30, absent=6)
    dev = torch.from_numpy(p).cuda()
    scale = 128 ** -0.5
    for c, (q, k, v) in zip(caches, sets):
        check(c, q, k, v, p, log_kv_tree_attention(c, q, k, v, scale, dev))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(log_kv_tree_attention(caches[i % 2], *sets[i % 2], scale, dev))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        check(caches[i % 2], *sets[i % 2], p, o)
    # Two graphs over the same cache (and so the same packed prefix).
    c = caches[0]
    graphs, outs = [], []
    for s, (q, k, v) in zip(streams, sets):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(log_kv_tree_attention(c, q, k, v, scale, dev))
        graphs.append(g)
    for q, k, v in sets:
        for t in (q, k, v):
            t.normal_()
    torch.cuda.synchronize()
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (q, k, v), o in zip(sets, outs):
        check(c, q, k, v, p, o)


def test_runs_agree_bit_for_bit():
    cache = make_cache(BF16, B=1, D=128, R=256, levels=4, seed=19)
    q, k, v = drafts(cache, 2, 50)
    p = random_tree(np.random.RandomState(20), 1, 50)
    first = run(cache, q, k, v, p)
    for _ in range(5):
        assert torch.equal(run(cache, q, k, v, p), first)


def test_two_threads_at_once():
    """Two host threads on streams of their own, over one cache, tree attention and beam selection."""
    import threading
    from logkv_b200 import beam_select, log_kv_tree_attention
    cache = make_cache(BF16, B=2, G=4, D=128, R=200, seed=23)
    p = random_tree(np.random.RandomState(24), 2, 40, absent=6)
    dev = torch.from_numpy(p).cuda()
    sets = [drafts(cache, 2, 40, seed=s) for s in (25, 26)]
    x = torch.randn(3, 4, 20000, device="cuda")
    r = torch.zeros(3, 4, device="cuda")
    want = [run(cache, *s, p) for s in sets]
    best = beam_select(x, r, 6)
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                a = log_kv_tree_attention(cache, *sets[i], 128 ** -0.5, dev)
                b = beam_select(x, r, 6)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(a, want[i]) or not all(torch.equal(s, t) for s, t in zip(b, best)):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_repeated_calls_are_checked_like_the_first():
    """Once a call of a shape has gone through, the host binding takes over: same results, same refusals."""
    from logkv_b200 import log_kv_tree_attention as f
    cache = make_cache(BF16, B=2, D=64, R=40, seed=27)
    q, k, v = drafts(cache, 2, 9)
    p = random_tree(np.random.RandomState(28), 2, 9, absent=2)
    dev = torch.from_numpy(p).cuda()
    first = f(cache, q, k, v, 0.125, dev)
    assert cache._read.native is not None
    for parents in (dev, dev.int(), torch.from_numpy(p), p.tolist()):
        assert torch.equal(f(cache, q, k, v, 0.125, parents), first)
    assert torch.equal(f(cache, q, k, v, 0.125, dev, out=torch.empty_like(first)), first)
    bad = p.copy()
    bad[0, 3] = 5
    for args, match in [((q[:1], k, v, 0.125, dev), "q must be"), ((q.float(), k, v, 0.125, dev), "q must be"),
                        ((q, k[:, :1], v, 0.125, dev), "k must be"), ((q, k, v[:, :, :8], 0.125, dev), "v shape"),
                        ((q[:, :3], k, v, 0.125, dev), "multiple"), ((q.cpu(), k, v, 0.125, dev), "device"),
                        ((q, k, v, 0.125, dev[:, :8]), "parents must be"), ((q, k, v, 0.125, dev.float()), "integers"),
                        ((q, k, v, 0.125, torch.from_numpy(bad)), "earlier token")]:
        with pytest.raises(ValueError, match=match):
            f(cache, *args)
    with pytest.raises(NotImplementedError):
        f(cache, q.detach().requires_grad_(), k, v, 0.125, dev)
    # A flush changes the ladder: the prefix is packed again before the next call.
    cache._ladder_epoch += 1
    cache.level_w.mul_(2)
    again = f(cache, q, k, v, 0.125, dev)
    assert cache._read.epoch == cache._ladder_epoch and not torch.equal(again, first)
    check(cache, q, k, v, p, again, scale=0.125)


def test_first_calls_of_a_process_in_two_threads():
    """The first calls of a process, from two threads at once, look up the driver's tensor-map encoder: the
    same bits as later calls."""
    import os
    import subprocess
    import sys
    import textwrap
    here = os.path.dirname(os.path.abspath(__file__))
    code = """
        import threading, torch
        import numpy as np
        from hypotheses import make_cache, random_tree
        from test_tree_attention_gpu import BF16, drafts
        from logkv_b200 import log_kv_tree_attention
        caches = [make_cache(BF16, B=2, G=2, D=128, R=200, seed=s) for s in (1, 2)]
        sets = [drafts(c, 2, 40) for c in caches]
        p = torch.from_numpy(random_tree(np.random.RandomState(3), 2, 40)).cuda()
        start, out = threading.Barrier(2), [None, None]
        def work(i):
            start.wait()
            out[i] = log_kv_tree_attention(caches[i], *sets[i], 0.1, p)
        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        [t.start() for t in threads], [t.join() for t in threads]
        for i in range(2):
            assert torch.equal(out[i], log_kv_tree_attention(caches[i], *sets[i], 0.1, p))
    """
    subprocess.run([sys.executable, "-c", textwrap.dedent(code)], check=True, timeout=300,
                   cwd=here, env={**os.environ, "PYTHONPATH": os.path.dirname(here)})


def test_another_stream_waits_for_the_prefix():
    """The first call after a flush packs the prefix, on its stream; a call on another stream that waits for
    the flush alone still reads the packed prefix.  So does chunk attention, and a reorder moves it."""
    from logkv_b200 import log_kv_chunk_attention, log_kv_tree_attention
    cache, same = (make_cache(BF16, B=2, G=2, D=64, R=40, seed=29) for _ in range(2))
    q, k, v = drafts(cache, 2, 9)
    p = torch.arange(-1, 8, device="cuda")
    tree = lambda c: log_kv_tree_attention(c, q, k, v, 0.125, p)  # noqa: E731
    chunk = lambda c: log_kv_chunk_attention(c, q, k, v, 0.125, 0.0)  # noqa: E731
    for c in (cache, same):
        tree(c)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        for call in (tree, chunk):
            for c in (cache, same):          # a flush, as far as the read side can tell
                c.level_w.mul_(2)
                c._ladder_epoch += 1
            want = call(same)
            torch.cuda.synchronize()
            with torch.cuda.stream(a):
                torch.cuda._sleep(100_000_000)
                tree(cache)
            with torch.cuda.stream(b):
                got = call(cache)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        cache._ladder_epoch += 1
        cache.level_w.mul_(2)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            torch.cuda._sleep(100_000_000)
            tree(cache)
        with torch.cuda.stream(b):
            cache.reorder_batch([1, 0])
        torch.cuda.synchronize()
        moved = tree(cache)
        cache._ladder_epoch += 1
        assert torch.equal(moved, tree(cache))


def test_a_captured_pack_is_its_graphs_own():
    """A call that is captured while the prefix is out of date packs it when its graph runs: calls outside
    that graph, and other graphs, pack it themselves."""
    from logkv_b200 import log_kv_chunk_attention, log_kv_tree_attention
    q, k, v = drafts(make_cache(BF16, B=2, G=2, D=64, R=40, seed=30), 2, 9)
    p = torch.arange(-1, 8, device="cuda")
    tree = lambda c: log_kv_tree_attention(c, q, k, v, 0.125, p)  # noqa: E731
    chunk = lambda c: log_kv_chunk_attention(c, q, k, v, 0.125, 0.0)  # noqa: E731
    for call in (tree, chunk):
        cache, same = (make_cache(BF16, B=2, G=2, D=64, R=40, seed=31) for _ in range(2))
        with torch.no_grad():
            for c in (cache, same):
                call(c)
                c.level_w.mul_(2)            # a flush, as far as the read side can tell
                c._ladder_epoch += 1
            want = call(same)
            graphs, outs = [], []
            for _ in range(2):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    call(cache)
                    outs.append(call(cache))
                graphs.append(g)
            graphs[1].replay()               # not the one captured first
            torch.cuda.synchronize()
            assert torch.equal(outs[1], want)
            for c in (cache, same):
                c.level_w.mul_(2)
                c._ladder_epoch += 1
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call(cache)
            want = call(same)
            assert torch.equal(call(cache), want)    # outside, before any replay
            graphs[0].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want)
