"""Caches with directly written state and plain 64-bit forms, shared by the tests of the operators
that decode several hypotheses (tree attention, path commits, beam selection, row reorder)."""
from __future__ import annotations

import numpy as np
import torch


def make_cache(dtype=torch.bfloat16, B=2, G=2, D=64, K=4, levels=3, R=100, P=32, recent=256, max_seq=4096, seed=0,
               granularity=None, device="cuda"):
    """A cache with `levels` ladder levels of random occupancy, an exact pool (when levels > 0) and R
    window rows; entries past a level's count and window rows past R hold an empty cache's values."""
    from logkv_b200.cache import LogStructuredKVCache
    from logkv_b200.workload import rope_tables
    cos, sin = rope_tables(max_seq + 64, D, base=1e6)
    cache = LogStructuredKVCache(
        (B, G, max_seq, D), (B, G, max_seq, D), B=32, recent_size=recent, device=device, dtype=dtype,
        semantic_clusters=True, semantic_anchor_mode="mid", allocate_second_order=False, cluster_k_max=K,
        semantic_flush_granularity=granularity or recent, alpha_exact_tokens=P, alpha_span_max_tokens=8,
        beta_novelty=True, beta_adaptive_merge=True, cos_cache=torch.from_numpy(cos), sin_cache=torch.from_numpy(sin),
        rope_n_elem=D)
    gen = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda t: torch.randn(t.shape, generator=gen, device=device).to(t.dtype)  # noqa: E731
    ints = lambda t, lo, hi: torch.randint(lo, hi, t.shape, generator=gen, device=device).to(t.dtype)  # noqa: E731
    if levels:
        Bs = cache.B_prime
        cache.level_count[..., :levels] = torch.randint(0, Bs + 1, cache.level_count[..., :levels].shape, generator=gen,
                                                        device=device).to(torch.int16)
        occ = torch.arange(Bs, device=device) < cache.level_count[..., None]
        for name in ("level_k", "level_v"):
            t = getattr(cache, name)
            t.copy_(rnd(t) * occ[..., None])
        w = ints(cache.level_w, 1, 60)
        m = ints(cache.level_sum_wp, 0, max_seq)
        cache.level_w.copy_(w * occ)
        cache.level_sum_wp.copy_(w.long() * m * occ)
        cache.level_p_lo.copy_(torch.where(occ, m, cache.level_p_lo))
        cache.level_p_hi.copy_(torch.where(occ, m + 1, cache.level_p_hi))
        cache.level_order.copy_(m * occ)
        for name in ("alpha_k_raw", "alpha_v", "centroid"):
            t = getattr(cache, name)
            t.copy_(rnd(t))
        cache.n_eff.copy_(ints(cache.n_eff, 1, 9))
        cache.n_total.copy_(ints(cache.n_total, 1, 900))
        cache.p_hi_c.copy_(ints(cache.p_hi_c, 0, max_seq))
        cache.alive.fill_(True)
        cache.alpha_pos.copy_(ints(cache.alpha_pos, 0, max_seq))
        cache.alpha_valid.fill_(True)
        cache.alpha_valid[0, P // 2] = False
        cache._row_count.fill_(P)
        cache._alpha_count_dev.fill_(P)
        cache._span_count.fill_(P // 8)
        cache._span_len[:, :P // 8] = 8
    for name in ("recent_k", "recent_v", "recent_k_raw"):
        t = getattr(cache, name)
        t[:, :, :R] = rnd(t[:, :, :R])
    cache.recent_pos[:, :R] = ints(cache.recent_pos[:, :R], 0, max_seq)
    cache._recent_ends[:, :R] = ints(cache._recent_ends[:, :R], 0, 2)
    cache.recent_count = cache.token_count = R
    cache._ladder_epoch += 1
    return cache


def random_tree(rs: np.random.RandomState, B: int, T: int, absent: int = 0) -> np.ndarray:
    """[B, T] parents: half of the tokens anywhere, half near the last ones; up to `absent` tokens
    missing at the end of each row."""
    p = np.zeros((B, T), np.int64)
    for b in range(B):
        for t in range(T):
            p[b, t] = rs.randint(-1, t) if rs.rand() < 0.5 else max(-1, t - 1 - rs.randint(0, 3))
        gone = rs.randint(0, absent + 1) if absent else 0
        p[b, T - gone:] = -2
    return p


def visible(p: np.ndarray) -> np.ndarray:
    """[B, T, T] bool: token t sees token j.  Values that are no parent count as absent."""
    B, T = p.shape
    see = np.zeros((B, T, T), bool)
    for b in range(B):
        for t in range(T):
            chain, at = [], t
            while at >= 0:
                chain.append(at)
                up = p[b, at]
                at = -2 if up < -2 or up >= at else int(up)
            if at == -1:
                see[b, t, chain] = True
    return see


def tree_reference(cache, q, k, v, scale, see: np.ndarray):
    """64-bit tree attention over the cache's packed prefix, window and the drafted tokens, and the
    elementwise bound on a kernel's distance from it.

    The bound: the probabilities reach the value product in the storage type (bf16 caches; half a
    step, u, relative to each, so at most u * A, A = sum p |v|), the output is rounded once (u * |out|);
    scores are float32 dot products of D + 2 terms (each term off by at most 2^-24 of it, twice for the
    scaling, so the exponent by at most e = 2 scale (D + 4) 2^-24 max(|q| . |k|)), and the sums over S
    keys are off by at most (S + 32) 2^-24 relative, once in the numerator and once in the denominator.
    """
    rs = cache._read
    B, H, T, D = q.shape
    G, R = cache.n_groups, cache.recent_count
    rf, f64 = H // G, torch.float64
    want = torch.zeros(B, H, T, D, dtype=f64, device=q.device)
    bound = torch.zeros_like(want)
    u = torch.finfo(q.dtype).eps / 2
    P_round = u if q.dtype == torch.bfloat16 else 0.0
    qx = float(torch.tensor(1.0 / scale, dtype=q.dtype))
    for b in range(B):
        vis = torch.from_numpy(see[b]).to(q.device)
        there = vis.any(1)
        keep = vis.any(0)                       # absent tokens: their values are not read
        kd = torch.where(keep[None, :, None], k[b], torch.zeros_like(k[b])).to(f64)
        vd = torch.where(keep[None, :, None], v[b], torch.zeros_like(v[b])).to(f64)
        for g in range(G):
            n = int(rs.length[b, g])
            key = torch.cat([rs.pk[b, g, :n].to(f64), cache.recent_k[b, g, :R].to(f64), kd[g]])
            val = torch.cat([rs.pv[b, g, :n].to(f64), cache.recent_v[b, g, :R].to(f64), vd[g]])
            mass = torch.zeros(key.size(0), dtype=f64, device=q.device)
            mass[:n] = rs.mass[b, g, :n].to(f64)
            qq = torch.where(there[None, :, None], q[b, g * rf:(g + 1) * rf], torch.zeros_like(q[b, :rf])).to(f64)
            z = scale * (qq @ key.T + qx * mass)
            reach = scale * (qq.abs() @ key.abs().T + qx * mass).amax()
            z[..., n + R:] = z[..., n + R:].masked_fill(~vis, float("-inf"))
            p = torch.softmax(z, -1)
            p = torch.where(there[None, :, None], p, torch.zeros_like(p))
            o = p @ val
            a = p @ val.abs()
            e = 2 * (D + 4) * 2.0 ** -24 * reach + 2 * (key.size(0) + 32) * 2.0 ** -24
            want[b, g * rf:(g + 1) * rf] = o
            bound[b, g * rf:(g + 1) * rf] = (P_round + e) * a + u * o.abs() * (1 + P_round) + 2.0 ** -40
    return want, bound
