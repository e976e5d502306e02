"""Batch rows taken over in place (reorder_batch) and accepted paths committed (add_recent_path),
against the same done with torch indexing, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from fixtures import config, make_stream
from hypotheses import make_cache, random_tree
from test_flush_gpu import make_cache as stream_cache
from test_flush_gpu import push_chunk

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
ROWS = ["level_k", "level_v", "level_w", "level_p_lo", "level_p_hi", "level_sum_wp", "level_order", "pad_mask",
        "level_count", "centroid", "n_eff", "n_total", "p_hi_c", "level0_phase", "alive", "s_h", "recent_k",
        "recent_k_raw", "recent_v", "recent_pos", "_recent_ends", "alpha_k_raw", "alpha_v", "alpha_pos", "alpha_valid",
        "_span_len", "_span_closed", "_span_count", "_row_count"]


def state(cache):
    return {n: getattr(cache, n).clone() for n in ROWS}


def same(got, want, what=""):
    for n in ROWS:
        assert torch.equal(got[n], want[n]), (what, n)


def maps(B, rs):
    yield np.arange(B)
    yield rs.permutation(B)                       # cycles
    yield np.roll(np.arange(B), 1)                # one cycle through every row
    yield np.zeros(B, np.int64)                   # one row taken over by all
    yield np.full(B, B - 1)
    yield rs.randint(0, B, B)
    keep = rs.permutation(B)[:max(1, B // 2)]     # rows that go on keep their places
    idx = np.arange(B)
    idx[~np.isin(idx, keep)] = rs.choice(keep, B - keep.size)
    yield idx


@pytest.mark.parametrize("dtype,B,G,D,levels,R", [(BF16, 1, 2, 64, 3, 100), (BF16, 2, 2, 64, 3, 101), (F32, 3, 1, 16, 2, 7),
                                                  (BF16, 5, 3, 128, 4, 256), (F32, 8, 2, 64, 0, 0), (BF16, 19, 1, 32, 3, 1),
                                                  (BF16, 70, 1, 16, 2, 33), (BF16, 300, 1, 16, 1, 5), (F32, 33, 2, 32, 3, 255)])
def test_reorder_equals_indexing(dtype, B, G, D, levels, R):
    from logkv_b200.attention import refresh_prefix
    cache = make_cache(dtype, B=B, G=G, D=D, levels=levels, R=R, seed=B)
    cache.s_h.uniform_(1, 2)
    cache._span_closed.random_(0, 2)
    rs = np.random.RandomState(B)
    for i, idx in enumerate(maps(B, rs)):
        read = refresh_prefix(cache)
        old = state(cache)
        pk, pv, mass, rows = (t.clone() for t in (read.pk, read.pv, read.mass, read.length))
        dev = torch.from_numpy(idx).cuda()
        cache.reorder_batch(dev.to(torch.int32) if i % 2 else dev)
        torch.cuda.synchronize()
        same(state(cache), {n: t[dev] for n, t in old.items()}, i)
        assert refresh_prefix(cache) is read and torch.equal(read.length, rows[dev])
        for b in range(B):
            for g in range(G):
                n = int(read.length[b, g])
                for a, z in ((read.pk, pk), (read.pv, pv), (read.mass, mass)):
                    assert torch.equal(a[b, g, :n], z[idx[b], g, :n])
    assert int(cache._read.status.item()) == 0


@pytest.mark.parametrize("dtype,B", [(BF16, 6), (F32, 3)])
def test_reorder_of_the_window_tail(dtype, B):
    cache = make_cache(dtype, B=B, G=2, D=64, R=131, seed=3)
    rs = np.random.RandomState(4)
    for w0 in (0, 1, 57, 130, 131):
        old, idx = state(cache), rs.randint(0, B, B)
        dev = torch.from_numpy(idx).cuda()
        cache.reorder_batch(idx.tolist(), window_from=w0)
        torch.cuda.synchronize()
        for n in ROWS:
            want = old[n].clone()
            if n in ("recent_pos", "_recent_ends"):
                want[:, w0:131] = old[n][dev][:, w0:131]
            elif n.startswith("recent_"):
                want[:, :, w0:131] = old[n][dev][:, :, w0:131]
            assert torch.equal(getattr(cache, n), want), (w0, n)


def test_rows_behind_the_window_stay():
    cache = make_cache(BF16, B=3, G=2, D=64, R=20, seed=5)
    for n in ("recent_k", "recent_v", "recent_k_raw"):
        getattr(cache, n)[:, :, 20:] = torch.randn_like(getattr(cache, n)[:, :, 20:])
    old = {n: getattr(cache, n)[:, :, 20:].clone() for n in ("recent_k", "recent_v", "recent_k_raw")}
    cache.reorder_batch([2, 0, 1])
    for n, t in old.items():
        assert torch.equal(getattr(cache, n)[:, :, 20:], t)


def test_bad_indices_on_the_device():
    cache = make_cache(BF16, B=4, G=2, D=64, R=20, seed=6)
    old = state(cache)
    cache.reorder_batch(torch.tensor([1, -1, 1 << 40, 0], device="cuda"))
    torch.cuda.synchronize()
    same(state(cache), {n: t[torch.tensor([1, 1, 2, 0], device="cuda")] for n, t in old.items()})
    assert int(cache._read.status.item()) == 1 << 19


@pytest.mark.parametrize("name", ["fp32_beta", "bf16_beta", "bf16_unified", "fp32_beta_g2k"])
def test_streams_swapped_half_way(name):
    """Rows swapped between flushes and then fed each other's stream: every buffer as if each had been
    in its place from the start, and attention over the moved prefix too."""
    from logkv_b200 import log_kv_chunk_attention
    cfg = config(name) if not name.endswith("unified") else next(
        c for c in __import__("streams").UNIFIED_CONFIGS if c["name"] == name)
    stream = make_stream(cfg)
    a, b = stream_cache(cfg, stream), stream_cache(cfg, stream)
    swap = lambda ch: {k: (v[::-1].copy() if isinstance(v, np.ndarray) and v.ndim > 1 else  # noqa: E731
                           v[::-1] if k == "span_ends" else v) for k, v in ch.items()}
    q = torch.randn(2, 4, 2, cfg["dim"], device="cuda").to(a.level_k.dtype)
    k = torch.randn(2, cfg["groups"], 2, cfg["dim"], device="cuda").to(a.level_k.dtype)
    for i, chunk in enumerate(stream["chunks"]):
        push_chunk(a, cfg, swap(chunk) if i >= 7 else chunk)
        push_chunk(b, cfg, swap(chunk))
        if i == 6:
            log_kv_chunk_attention(a, q, k, k, 0.25)      # packs the prefix before the swap
            a.reorder_batch([1, 0])
            with torch.no_grad():
                assert torch.equal(log_kv_chunk_attention(a, q, k, k, 0.25), log_kv_chunk_attention(b, q, k, k, 0.25))
    torch.cuda.synchronize()
    same(state(a), state(b))


def test_reorder_in_graphs_and_streams():
    from logkv_b200.attention import refresh_prefix
    caches = [make_cache(BF16, B=4, G=2, D=64, R=50, seed=s) for s in (7, 8)]
    idx = [torch.tensor([1, 2, 3, 0], device="cuda"), torch.tensor([0, 0, 2, 2], device="cuda")]
    for c in caches:
        refresh_prefix(c)
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    for c, i, s in zip(caches, idx, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.reorder_batch(i)
        graphs.append(g)
    old = [state(c) for c in caches]
    idx[1].copy_(torch.tensor([3, 2, 1, 0]))               # the index is read when the graph runs
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, o, i in zip(caches, old, idx):
        same(state(c), {n: t[i][i][i] for n, t in o.items()})


def test_reorder_refusals():
    cache = make_cache(BF16, B=2, G=2, D=64, R=20, seed=9)
    cache._read = None
    g = torch.cuda.CUDAGraph()
    index = torch.tensor([1, 0], device="cuda")
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="attended over"):
            cache.reorder_batch(index)
        index.add_(0)
    cache.begin_op_log()
    with pytest.raises(RuntimeError, match="op-log"):
        cache.reorder_batch(index)


# ---------------------------------------------------------------- accepted paths
def drafted(cache, T, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, G, D = cache.batch_size, cache.n_groups, cache.k_dim
    mk = lambda: torch.randn(B, T, G, D, generator=gen, device="cuda").to(cache.level_k.dtype).transpose(1, 2)  # noqa: E731
    return mk(), mk(), mk()


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F32, 16)])
def test_path_equals_gather_then_append(dtype, D):
    """Paths of 1 to 24 tokens until the window has been flushed several times."""
    a, b = (make_cache(dtype, B=3, G=2, D=D, levels=2, R=60, recent=64, granularity=16, seed=10) for _ in range(2))
    rs = np.random.RandomState(11)
    for i in range(40):
        T, n = rs.randint(1, 40), rs.randint(1, 25)
        k, v, kr = drafted(a, T, i)
        path = torch.from_numpy(rs.randint(0, T, (3, n)) if i % 3 else np.repeat(rs.randint(0, T, (1, n)), 3, 0))
        ends = rs.rand(3, T) < 0.3
        depth = torch.from_numpy(np.arange(T)).cuda() + a.token_count if i % 2 else None
        pos = None if depth is None else depth.expand(3, T).contiguous()
        how = path.cuda() if i % 3 == 1 else path[0].cuda().int() if i % 3 == 0 else path.tolist()
        kw = dict(span_ends=ends.tolist()) if i % 2 else dict(span_ends_device=torch.from_numpy(ends).cuda())
        a.add_recent_path(k, v, how, k_raw=kr, input_pos=pos, **kw)
        at = path.cuda()[:, None, :, None].expand(3, 2, n, D)
        b.add_recent(k.gather(2, at), v.gather(2, at), k_raw=kr.gather(2, at),
                     input_pos=None if pos is None else pos.gather(1, path.cuda()),
                     span_ends=np.take_along_axis(ends, path.numpy(), 1).tolist())
        assert (a.recent_count, a.token_count, a._ladder_epoch) == (b.recent_count, b.token_count, b._ladder_epoch)
    torch.cuda.synchronize()
    same(state(a), state(b))


def test_bad_path_on_the_device():
    from logkv_b200.attention import refresh_prefix
    a, b = (make_cache(BF16, B=2, G=2, D=64, R=5, seed=12) for _ in range(2))
    refresh_prefix(a)
    k, v, kr = drafted(a, 6, 1)
    ends = [[False] * 6] * 2
    a.add_recent_path(k, v, torch.tensor([[1, 6, 2], [0, -1, 5]], device="cuda"), k_raw=kr, span_ends=ends)
    b.add_recent_path(k, v, [[1, 0, 2], [0, 0, 5]], k_raw=kr, span_ends=ends)
    same(state(a), state(b))
    assert int(a._read.status.item()) == 1 << 19


def test_speculative_step_end_to_end():
    """Drafting, tree attention, commit of the accepted path, the next attention: the outputs of the
    accepted tokens equal attention over a cache that committed them one after the other, each within
    its own bound."""
    from hypotheses import tree_reference, visible
    from logkv_b200 import log_kv_tree_attention
    a, b = (make_cache(BF16, B=2, G=2, D=64, levels=2, R=60, recent=64, granularity=32, seed=13) for _ in range(2))
    rs = np.random.RandomState(14)
    scale, T = 0.125, 12
    for step in range(6):
        k, v, kr = drafted(a, T, 100 + step)
        q = torch.randn(2, 6, T, 64, device="cuda").bfloat16()
        p = random_tree(rs, 2, T)
        paths = []
        for row in p:
            leaf = int(rs.randint(0, T))
            chain = []
            while leaf >= 0:
                chain.append(leaf)
                leaf = int(row[leaf])
            paths.append(chain[::-1])
        n = min(len(x) for x in paths)
        paths = np.array([x[:n] for x in paths])
        out = log_kv_tree_attention(a, q, k, v, scale, torch.from_numpy(p).cuda())
        _, bound = tree_reference(a, q, k, v, scale, visible(p))
        at = torch.from_numpy(paths).cuda()
        ends = (rs.rand(2, T) < 0.3)
        # The same tokens as a chain over the other cache.
        pick = lambda t: t.gather(2, at[:, None, :, None].expand(2, t.size(1), n, 64))  # noqa: E731
        chain = log_kv_tree_attention(b, pick(q), pick(k), pick(v), scale, list(range(-1, n - 1)))
        assert ((pick(out).double() - chain.double()).abs() <= 2 * pick(bound)).all()
        a.add_recent_path(k, v, at, k_raw=kr, span_ends=ends.tolist())
        b.add_recent(pick(k), pick(v), k_raw=pick(kr), span_ends=np.take_along_axis(ends, paths, 1).tolist())
        torch.cuda.synchronize()
        same(state(a), state(b), step)


def test_read_status_tells_of_bad_device_values():
    """The public status word has the bits of every call, those before the first attention too, until the
    cache is reset."""
    from logkv_b200 import log_kv_tree_attention
    cache = make_cache(BF16, B=2, G=2, D=64, R=5, seed=15)
    assert cache.read_status() == 0
    k, v, kr = drafted(cache, 6, 1)
    path = torch.tensor([[1, 6, 2], [0, -1, 5]], device="cuda")
    cache.add_recent_path(k, v, path, k_raw=kr, span_ends=[[False] * 6] * 2)
    assert cache.read_status() == 1 << 19
    log_kv_tree_attention(cache, k, k, v, 0.125, torch.tensor([-1, 0, 2, 0, 1, -1], device="cuda"))
    assert cache.read_status() == 1 << 19 | 1 << 18
    cache.reset_parameters()
    assert cache.read_status() == 0
    cache.reorder_batch(torch.tensor([1, 2], device="cuda"))
    assert cache.read_status() == 1 << 19


def test_path_without_drafted_tokens():
    """Nothing drafted: refused before anything is counted, with a path on the device too."""
    cache = make_cache(BF16, B=2, G=2, D=64, R=5, seed=16)
    k = torch.empty(2, 2, 0, 64, dtype=BF16, device="cuda")
    for path in ([0], torch.zeros(1, dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError, match="drafted"):
            cache.add_recent_path(k, k, path, k_raw=k, span_ends=[[], []])
    assert cache.token_count == cache.recent_count == 5
