"""Workloads of the operators that decode several hypotheses over the LogKV cache.

  tree     attention of a tree of drafted tokens over the cache
           (``logkv_b200.log_kv_tree_attention``);
  beam     selection of the best continuations over beams and vocabulary
           (``logkv_b200.beam_select``);
  reorder  the cache's batch rows taken over by the beams that go on
           (``LogStructuredKVCache.reorder_batch``).

``own`` chooses between the framework's kernels and the plain form: elementary torch operations
in float32 (float64 for the beam scores, whose order decides).  Lengths, trees and row maps are
fixed by a case's ``shape`` number, values by the seed.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def _cache_case(op, name, **kw):
    """A cache of B rows, G KV groups, head dim D, K clusters of `slots` budgeted slots, `exact` pool
    rows, `levels` occupied ladder levels and `recent` window rows (of `window` before a flush)."""
    base = dict(op=op, name=name, dtype="bf16", B=1, G=8, D=128, K=12, slots=128, exact=256, max_seq=32768,
                levels=4, window=2048, recent=2048, shape=1)
    base.update(kw)
    return base


def listed():
    return [
        # One drafted token right after a short prompt: nothing flushed yet, launch latency only.
        _cache_case("tree", "tree_token_short", G=2, rf=4, D=64, K=8, slots=64, exact=64, max_seq=8192, levels=0,
                    window=512, recent=37, T=1, shape=11),
        # One sequence over a 32K-token compressed cache, a short chain of drafts with one branch.
        _cache_case("tree", "tree_b1_t7", rf=2, T=7, shape=12),
        # A small serving batch, ordinary tree.
        _cache_case("tree", "tree_b8_t26", B=8, rf=2, T=26, shape=13),
        # The largest: a full batch with 64-token trees.
        _cache_case("tree", "tree_b32_t64", B=32, rf=2, T=64, shape=14),
        # Odd head grouping and tree sizes, some rows' trees padded with absent tokens.
        _cache_case("tree", "tree_b3_t61_rf5", B=3, G=4, rf=5, D=64, K=8, slots=64, exact=64, max_seq=8192, levels=5,
                    window=1024, recent=777, T=61, absent=9, shape=15),
        # A float32 cache.
        _cache_case("tree", "tree_fp32_b2_t13", dtype="fp32", B=2, G=4, rf=3, D=64, K=8, slots=64, exact=64,
                    max_seq=8192, levels=4, window=512, recent=301, T=13, shape=16),
        # First step of one request: only beam 0 is alive, twice the beams asked for.
        dict(op="beam", name="beam_first_w4", dtype="fp32", N=1, W=4, V=32000, k=8, first=True, keep=False, shape=21),
        # A batch of requests at an odd width and vocabulary, children placed in their parents' rows.
        dict(op="beam", name="beam_n29_w5", dtype="fp32", N=29, W=5, V=50021, k=5, first=False, keep=True, shape=22),
        # The largest: wide beams over a 151936-token vocabulary.
        dict(op="beam", name="beam_n32_w16", dtype="bf16", N=32, W=16, V=151936, k=32, first=False, keep=False,
             shape=23),
        # A small float32 cache, whole rows (a step right after a flush).
        _cache_case("reorder", "reorder_b3_fp32", dtype="fp32", B=3, G=2, D=64, K=8, slots=64, exact=64, max_seq=4096,
                    levels=3, window=512, recent=129, groups_of=3, moved=1, window_from=-1, shape=31),
        # Two requests of four beams over a 32K-token compressed cache, whole rows.
        _cache_case("reorder", "reorder_b8", B=8, groups_of=4, moved=4, window_from=-1, shape=32),
        # Sixteen requests of four beams that share everything up to the fork: the window's tail alone.
        _cache_case("reorder", "reorder_tail_b64", B=64, K=4, slots=32, max_seq=8192, exact=64, levels=1, recent=1423,
                    window=2048, groups_of=4, moved=27, window_from=1200, shape=33),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "beam", "reorder"])
    shape = rng.randrange(1, 1 << 20)
    if op == "beam":
        dtype, W, V = rng.choice(["fp32", "bf16"]), _log_int(rng, 1, 16), _log_int(rng, 500, 151936)
        N = _log_int(rng, 1, max(1, min(64, 70_000_000 // (W * V))))
        keep = rng.random() < 0.3
        k = W if keep else min(W * V, _log_int(rng, 1, 2 * W))
        return dict(op="beam", dtype=dtype, N=N, W=W, V=V, k=k, first=rng.random() < 0.2, keep=keep, shape=shape)
    D, G, K = rng.choice([64, 128]), rng.choice([1, 2, 4, 8]), rng.choice([4, 8, 12])
    slots, levels = rng.choice([32, 64, 128]), rng.randrange(0, 5)
    window = rng.choice([256, 512, 2048])
    c = _cache_case(op, "", dtype=rng.choice(["bf16", "bf16", "fp32"]), G=G, D=D, K=K, slots=slots, exact=64,
                    max_seq=8192, levels=levels, window=window, recent=rng.randrange(0, window + 1), shape=shape)
    del c["name"]
    if op == "tree":
        c["T"], c["rf"] = _log_int(rng, 1, 128 if c["dtype"] == "bf16" else 48), rng.choice([1, 2, 3, 4, 5, 7, 8])
        most = 32 * 8 * 8304 * 128 * 128                       # the largest listed case's work
        each = G * (K * levels * slots + 64 + c["recent"] + c["T"]) * D * max(16, c["rf"] * c["T"])
        each *= 16 if c["dtype"] == "fp32" else 1
        c["B"] = _log_int(rng, 1, max(1, min(32, most // each)))
        c["absent"] = rng.randrange(0, max(1, c["T"] // 4))
    else:
        gof = rng.choice([2, 3, 4, 5, 8])
        row = G * (K * 6 * slots * 2 + 4 * window) * 2 * D * (2 if c["dtype"] == "bf16" else 4)
        c["groups_of"], c["B"] = gof, gof * rng.randrange(1, max(2, min(4, 800_000_000 // (row * gof))))
        c["moved"] = rng.randrange(0, c["B"] - c["B"] // gof + 1)
        c["window_from"] = rng.choice([-1, -1, rng.randrange(0, c["recent"] + 1)])
    return c


# ------------------------------------------------------------------ the cache's state
def _geometry(c):
    """(B', L): slots per level and levels of the cache, after the exact pool has been paid for."""
    e, D, G, K, P, N = 2 if c["dtype"] == "bf16" else 4, c["D"], c["G"], c["K"], c["exact"], c["max_seq"]
    levels = lambda b: max(2, math.ceil(math.log2(N / (K * b) + 1.0)) + 2)  # noqa: E731
    packed = (D + 1 + 7) // 8 * 8
    entry = (2 * D + 2 * packed) * e + 41
    pool = P * (G * (2 * D + 2 * packed) * e + 9)
    for b in range(c["slots"] - 1, 1, -1):
        if G * K * levels(b) * (b * entry + 2) + pool <= G * K * levels(c["slots"]) * (c["slots"] * entry + 2):
            return b, levels(b)
    raise ValueError("no room for the exact pool")


def _counts(c):
    """[B, G, K, L] occupied slots per level: the lower `levels` levels between half and quite full."""
    Bs, L = _geometry(c)
    rs = np.random.RandomState(c["shape"])
    n = np.zeros((c["B"], c["G"], c["K"], L), np.int64)
    used = min(c["levels"], L)
    if used:
        n[..., :used] = rs.randint(Bs // 2, Bs + 1, n[..., :used].shape)
        if c["levels"] >= 4:      # a long context: three levels of four are full
            n[..., 1:used] = np.where(rs.rand(*n[..., 1:used].shape) < 0.9, Bs, n[..., 1:used])
    return n


def _prefix_rows(c):
    """[B, G] rows of the packed prefix: the occupied slots, then the exact pool."""
    return _counts(c).sum((2, 3)) + (c["exact"] if c["levels"] else 0)


def _rope_tables(c):
    n = c["max_seq"] + 64
    inv = 1.0 / (1e6 ** (np.arange(0, c["D"], 2, dtype=np.float64) / c["D"]))
    ang = np.arange(n, dtype=np.float64)[:, None] * inv[None]
    ang = np.concatenate([ang, ang], 1)
    return torch.from_numpy(np.cos(ang).astype(np.float32)).cuda(), torch.from_numpy(np.sin(ang).astype(np.float32)).cuda()


def _buffers(c, gen, whole):
    """The cache's device buffers by name; entries past a level's count hold an empty cache's values.
    `whole`: also the bookkeeping that attention does not read."""
    dt, B, G, D, K, P = DTYPES[c["dtype"]], c["B"], c["G"], c["D"], c["K"], c["exact"]
    Bs, L = _geometry(c)
    cap, n = 2 * c["window"], _counts(c)
    R, P_used = c["recent"], P if c["levels"] else 0
    lc = torch.from_numpy(n).cuda()
    occ = torch.arange(Bs, device="cuda") < lc[..., None]                        # [B, G, K, L, B']

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    def ints(lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda")

    def window(t):
        t[:, :, R:] = 0
        return t

    # Merged masses: most slots hold a few tokens, some hundreds; their positions anywhere before.
    u = torch.rand(occ.shape, generator=gen, device="cuda").clamp_min_(1e-6)
    w = torch.where(occ, (u.log() / math.log(0.9)).floor() + 1, torch.zeros_like(u))
    m = ints(0, c["max_seq"], occ.shape)
    b = {"level_k": normal(B, G, K, L, Bs, D) * occ[..., None], "level_v": normal(B, G, K, L, Bs, D) * occ[..., None],
         "level_w": w, "level_sum_wp": w.long() * m, "level_count": lc.to(torch.int16),
         "recent_k": window(normal(B, G, cap, D)), "recent_v": window(normal(B, G, cap, D)),
         "alpha_k_raw": normal(B, G, P, D), "alpha_v": normal(B, G, P, D), "alpha_pos": ints(0, c["max_seq"], (B, P)),
         "alpha_valid": torch.arange(P, device="cuda").expand(B, P) < P_used}
    if not P_used:
        for name in ("alpha_k_raw", "alpha_v", "alpha_pos"):
            b[name].zero_()
    if whole:
        b["level_p_lo"] = torch.where(occ, m, torch.full_like(m, torch.iinfo(torch.int64).max))
        b["level_p_hi"] = torch.where(occ, m + w.long(), torch.full_like(m, -1))
        b["level_order"] = torch.where(occ, ints(0, c["max_seq"], occ.shape), torch.zeros_like(m))
        b["centroid"] = normal(B, G, K, D, dtype=torch.float32)
        b["n_eff"] = torch.rand(B, G, K, generator=gen, device="cuda")
        b["n_total"] = ints(0, c["max_seq"], (B, G, K)).int()
        b["p_hi_c"] = ints(-1, c["max_seq"], (B, G, K))
        b["level0_phase"] = ints(0, 2, (B, G, K)).int()
        b["alive"] = ints(0, 2, (B, G, K)).bool()
        b["recent_k_raw"] = window(normal(B, G, cap, D))
        b["recent_pos"] = ints(0, c["max_seq"], (B, cap))
        b["recent_pos"][:, R:] = 0
    return b


def _packed(c, b, cos, sin):
    """The packed prefix ([B, G, S, D] keys and values, [B, G, S] log-mass terms): per lane the occupied
    slots (cluster by cluster, top level first) and the exact pool, keys rotated at their positions."""
    dt, B, G, D, K, P = DTYPES[c["dtype"]], c["B"], c["G"], c["D"], c["K"], c["exact"]
    Bs, L = _geometry(c)
    n, rows = _counts(c), _prefix_rows(c)
    S, cap = int(rows.max()), K * L * Bs
    slot = np.arange(cap).reshape(K, L, Bs)[:, ::-1]
    take = np.zeros((B, G, S), np.int64)
    for i in range(B):
        for g in range(G):
            at = slot[np.arange(Bs)[None, None] < n[i, g][:, ::-1, None]]
            take[i, g, :rows[i, g]] = np.concatenate([at, cap + np.arange(rows[i, g] - at.size)])
    take = torch.from_numpy(take).cuda()
    wide = take[..., None].expand(B, G, S, D)
    w = b["level_w"].view(B, G, cap)
    sw = b["level_sum_wp"].view(B, G, cap)
    ww = w.long().clamp_min(1)
    pos = torch.cat([torch.div(2 * sw + ww, 2 * ww, rounding_mode="floor"), b["alpha_pos"][:, None].expand(B, G, P)], 2)
    mass = torch.cat([w.clamp_min(1).log().to(dt).float(), torch.zeros(B, G, P, device="cuda")], 2).gather(2, take)
    x = torch.cat([b["level_k"].view(B, G, cap, D), b["alpha_k_raw"]], 2).gather(2, wide).float()
    v = torch.cat([b["level_v"].view(B, G, cap, D), b["alpha_v"]], 2).gather(2, wide)
    pos = pos.gather(2, take)
    rot = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
    return (x * cos[pos] + rot * sin[pos]).to(dt), v, mass


def _cache(c, b, cos, sin):
    """The framework's cache with these buffers."""
    from logkv_b200 import LogStructuredKVCache
    B, G, D = c["B"], c["G"], c["D"]
    shape = (B, G, c["max_seq"], D)
    cache = LogStructuredKVCache(
        shape, shape, B=c["slots"], recent_size=c["window"], device="cuda", dtype=DTYPES[c["dtype"]],
        semantic_clusters=True, semantic_anchor_mode="mid", allocate_second_order=False, cluster_k_max=c["K"],
        semantic_flush_granularity=c["window"], alpha_exact_tokens=c["exact"],
        alpha_span_max_tokens=min(64, c["exact"]), beta_novelty=True, beta_adaptive_merge=True, cos_cache=cos,
        sin_cache=sin, rope_n_elem=D)
    for name, t in b.items():
        getattr(cache, name).copy_(t)
    cache._row_count.fill_(c["exact"] if c["levels"] else 0)
    cache._alpha_count_dev.fill_(c["exact"] if c["levels"] else 0)
    cache.recent_count = cache.token_count = c["recent"]
    cache._ladder_epoch += 1
    return cache


# ------------------------------------------------------------------ tree
def _parents(c):
    """[B, T] parents: -1 a child of the last committed token, -2 no token (the end of a padded row)."""
    rs = np.random.RandomState(c["shape"] + 1)
    T = c["T"]
    p = np.zeros((c["B"], T), np.int64)
    for i in range(c["B"]):
        for t in range(T):
            p[i, t] = rs.randint(-1, t) if rs.rand() < 0.5 else t - 1 - min(t, rs.randint(0, 3))
        gone = rs.randint(0, c.get("absent", 0) + 1) if c.get("absent", 0) else 0
        p[i, T - gone:] = -2
    return p


def _ancestors(p):
    """[B, T, T] whether token t sees token j (itself and its ancestors), from parents on the device."""
    B, T = p.shape
    up = torch.zeros(B, T, T, device=p.device)
    up.scatter_(2, p.clamp_min(0)[..., None], (p >= 0).float()[..., None])
    see = up + torch.eye(T, device=p.device)
    n = 1
    while n < T:
        see = ((see @ see) > 0).float()
        n *= 2
    gone = (see @ (p < -1).float()[..., None]) > 0
    return (see > 0) & ~gone


def _prepare_tree(c, gen):
    dt, B, G, D, T, R = DTYPES[c["dtype"]], c["B"], c["G"], c["D"], c["T"], c["recent"]
    cos, sin = _rope_tables(c)
    b = _buffers(c, gen, False)
    st = {"scale": D ** -0.5, "parents": torch.from_numpy(_parents(c)).to("cuda", torch.int32)}
    # As a projection leaves them: [B, T, heads, D] seen as [B, heads, T, D].
    for name, heads in (("q", G * c["rf"]), ("k", G), ("v", G)):
        st[name] = torch.randn(B, T, heads, D, generator=gen, device="cuda", dtype=dt).transpose(1, 2)
    if own:
        from logkv_b200.attention import refresh_prefix
        st["cache"] = _cache(c, b, cos, sin)
        refresh_prefix(st["cache"])
    else:
        st["pk"], st["pv"], st["mass"] = _packed(c, b, cos, sin)
        st["rows"] = torch.from_numpy(_prefix_rows(c)).cuda()
        st["rk"], st["rv"] = b["recent_k"][:, :, :R].clone(), b["recent_v"][:, :, :R].clone()
    return st


def _run_tree(st):
    q, k, v, parents, scale = st["q"], st["k"], st["v"], st["parents"], st["scale"]
    if own:
        from logkv_b200 import log_kv_tree_attention
        return log_kv_tree_attention(st["cache"], q, k, v, scale, parents)
    B, H, T, D = q.shape
    G, S, R = k.size(1), st["pk"].size(2), st["rk"].size(2)
    keys = torch.cat([st["pk"], st["rk"], k], 2).float()
    qx = float(torch.tensor(1.0 / scale, dtype=q.dtype))
    z = q.float().reshape(B, G, H // G * T, D) @ keys.transpose(2, 3)
    del keys
    z = z.view(B, G, H // G, T, S + R + T)
    z[..., :S] += (qx * st["mass"])[:, :, None, None]
    z *= scale
    dead = torch.arange(S, device=q.device) >= st["rows"][..., None]
    z[..., :S].masked_fill_(dead[:, :, None, None], -math.inf)
    see = _ancestors(parents.long())
    z[..., S + R:].masked_fill_(~see[:, None, None], -math.inf)
    z = (z - z.amax(-1, keepdim=True)).exp()
    z = z / z.sum(-1, keepdim=True)
    out = z.view(B, G, H // G * T, S + R + T) @ torch.cat([st["pv"], st["rv"], v], 2).float()
    there = see.any(-1)
    out = out.view(B, H, T, D).masked_fill(~there[:, None, :, None], 0.0)
    return out.to(q.dtype)


def _exact_tree(c, seed):
    st = _plain_state(c, seed)
    B, G, T, R, rf, D = c["B"], c["G"], c["T"], c["recent"], c["rf"], c["D"]
    rows, par = _prefix_rows(c), _parents(c)
    out = torch.zeros(B, G * rf, T, D, dtype=torch.float64, device="cuda")
    qx = float(torch.tensor(1.0 / st["scale"], dtype=st["q"].dtype))
    for i in range(B):
        chain = []
        for t in range(T):                                # the tokens that t sees, by walking up
            seen, at = [t], par[i, t]
            while at >= 0:
                seen.append(int(at))
                at = par[i, at]
            chain.append(None if at == -2 else seen)
        for g in range(G):
            n = int(rows[i, g])
            key = torch.cat([st["pk"][i, g, :n], st["rk"][i, g]]).double()
            val = torch.cat([st["pv"][i, g, :n], st["rv"][i, g]]).double()
            bias = torch.zeros(n + R, dtype=torch.float64, device="cuda")
            bias[:n] = qx * st["mass"][i, g, :n].double()
            qs = st["q"][i, g * rf:(g + 1) * rf].double()                       # [rf, T, D]
            old = st["scale"] * (qs @ key.T + bias)
            new = st["scale"] * (qs @ st["k"][i, g].double().T)
            hide = torch.ones(T, T, dtype=torch.bool)
            for t in range(T):
                if chain[t] is not None:
                    hide[t, chain[t]] = False
            new = new.masked_fill(hide.cuda(), -math.inf)
            z = torch.cat([old, new], -1)
            p = torch.softmax(z, -1) @ torch.cat([val, st["v"][i, g].double()])
            gone = torch.tensor([x is None for x in chain], device="cuda")
            out[i, g * rf:(g + 1) * rf] = p.masked_fill(gone[None, :, None], 0.0)
    return out


def _work_tree(c):
    e, B, G, D, T, R = 2 if c["dtype"] == "bf16" else 4, c["B"], c["G"], c["D"], c["T"], c["recent"]
    rows = int(_prefix_rows(c).sum())
    keys = rows + B * G * (R + T)
    see = 0
    for p in _parents(c):
        depth = np.zeros(T, np.int64)
        for t in range(T):
            depth[t] = 0 if p[t] == -2 else 1 if p[t] < 0 else depth[p[t]] + 1
        see += int(depth.sum())
    pairs = c["rf"] * (T * (rows + B * G * R) + G * see)
    return {"bytes": keys * 2 * D * e + rows * 4 + 2 * B * G * c["rf"] * T * D * e + B * T * 4, "flops": 4 * D * pairs}


# ------------------------------------------------------------------ beam
def _prepare_beam(c, gen):
    N, W, V = c["N"], c["W"], c["V"]
    x = torch.randn(N, W, V, generator=gen, device="cuda") * 2.5
    x += 6.0 * (torch.rand(N, W, V, generator=gen, device="cuda") < 3.0 / V)     # a few likely tokens
    x[torch.rand(N, W, V, generator=gen, device="cuda") < 0.01] = -math.inf     # banned tokens
    scores = -3.0 - 2.0 * torch.rand(N, W, generator=gen, device="cuda")
    if c["first"]:
        scores = torch.full((N, W), -math.inf, device="cuda")
        scores[:, 0] = 0.0
    return {"logits": x.to(DTYPES[c["dtype"]]), "scores": scores, "k": c["k"], "keep": c["keep"]}


def _run_beam(st):
    logits, scores, k, keep = st["logits"], st["scores"], st["k"], st["keep"]
    if own:
        from logkv_b200 import beam_select
        return beam_select(logits, scores, k, keep_places=keep)
    N, W, V = logits.shape
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    lse = top + (x - top).exp().sum(-1, keepdim=True).log()
    ok = lse.isfinite() & scores.double()[..., None].isfinite()
    total = (scores.double()[..., None] + (x - lse)).masked_fill(~ok, -math.inf)
    best, at = torch.sort(total.view(N, W * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    empty = best == -math.inf
    beam, token = at // V, (at % V).masked_fill(empty, 0)
    j = torch.arange(k, device=x.device)
    place = j.expand(N, k)
    if keep:
        # The best child of a beam takes the beam's own place, the others the free places in order.
        again = ((beam[:, :, None] == beam[:, None, :]) & (j[None, :] < j[:, None])).any(-1)
        first = ~again & ~empty
        used = torch.zeros(N, W + 1, dtype=torch.long, device=x.device)
        used.scatter_(1, torch.where(first, beam, torch.full_like(beam, W)), 1)
        free = torch.sort(used[:, :W], dim=-1, stable=True)[1]
        place = torch.where(first, beam, free.gather(1, ((~first).long().cumsum(-1) - 1).clamp_min(0)))
    beam = torch.where(empty, place.clamp(max=W - 1), beam)
    rows = beam + W * torch.arange(N, device=x.device)[:, None]
    put = lambda t: torch.empty_like(t).scatter_(1, place, t)  # noqa: E731
    return put(best.float()), put(rows), put(token)


def _exact_beam(c, seed):
    st = _plain_state(c, seed)
    N, W, k = c["N"], c["W"], c["k"]
    out = torch.full((N, k), -math.inf, dtype=torch.float64)
    rows, tokens = torch.zeros(N, k, dtype=torch.long), torch.zeros(N, k, dtype=torch.long)
    for n in range(N):
        cand = []
        for w in range(W):
            x = st["logits"][n, w].double()
            r = float(st["scores"][n, w])
            z = float(torch.logsumexp(x, 0))
            if not (math.isfinite(r) and math.isfinite(z)):
                continue
            x = x.cpu().numpy()
            near = np.nonzero(x >= np.partition(x, -min(k, x.size))[-min(k, x.size)])[0]
            cand += [(-(r + (float(x[v]) - z)), w, int(v)) for v in near if x[v] != -math.inf]
        cand.sort()
        cand = cand[:k]
        where = list(range(k))
        if c["keep"]:
            taken = {}
            for i, (_, w, _v) in enumerate(cand):
                taken.setdefault(w, i)
            free = [p for p in range(W) if p not in taken]
            where = [w if taken[w] == i else free.pop(0) for i, (_, w, _v) in enumerate(cand)] + free
        for p in range(k):
            rows[n, p] = n * W + min(p, W - 1)
        for i, (s, w, v) in enumerate(cand):
            out[n, where[i]], rows[n, where[i]], tokens[n, where[i]] = -s, n * W + w, v
    return out, rows, tokens


# ------------------------------------------------------------------ reorder
def _index(c):
    """[B] the old row that each row goes on from: within every request (`groups_of` rows), beams that
    go on keep their rows, and `moved` rows in all take over a beam that goes on."""
    rs = np.random.RandomState(c["shape"] + 2)
    B, n = c["B"], c["groups_of"]
    idx = np.arange(B)
    may = np.concatenate([i + 1 + rs.permutation(n - 1) for i in range(0, B, n)]) if n > 1 else np.zeros(0, int)
    gone = set(rs.permutation(may)[:c["moved"]].tolist())
    for r in sorted(gone):
        idx[r] = rs.choice([s for s in range(r - r % n, r - r % n + n) if s not in gone])
    return idx


def _prepare_reorder(c, gen):
    cos, sin = _rope_tables(c)
    b = _buffers(c, gen, True)
    st = {"index": torch.from_numpy(_index(c)).cuda(), "from": c["window_from"], "recent": c["recent"]}
    if own:
        from logkv_b200.attention import refresh_prefix
        cache = st["cache"] = _cache(c, b, cos, sin)
        names = list(b)
        del b
        read = refresh_prefix(cache)
        S = int(_prefix_rows(c).max())
        st["out"] = {name: getattr(cache, name) for name in names}
        st["out"].update(prefix_k=read.pk[:, :, :S], prefix_v=read.pv[:, :, :S], prefix_mass=read.mass[:, :, :S],
                         prefix_rows=read.length)
    else:
        k, v, mass = _packed(c, b, cos, sin)
        rows = torch.from_numpy(_prefix_rows(c)).to("cuda", torch.int32)
        dead = torch.arange(k.size(2), device="cuda") >= rows[..., None]
        b.update(prefix_k=k.masked_fill(dead[..., None], 0), prefix_v=v.masked_fill(dead[..., None], 0),
                 prefix_mass=mass.masked_fill(dead, 0), prefix_rows=rows)
        st["out"] = b
    return st


def _run_reorder(st):
    index, w0 = st["index"], st["from"]
    if own:
        st["cache"].reorder_batch(index, window_from=None if w0 < 0 else w0)
        return st["out"]
    for name, t in st["out"].items():
        if w0 < 0:
            t.copy_(t[index])
        elif name == "recent_pos":
            t[:, w0:st["recent"]] = t[:, w0:st["recent"]][index]
        elif name.startswith("recent_"):
            t[:, :, w0:st["recent"]] = t[:, :, w0:st["recent"]][index]
    return st["out"]


def _work_reorder(c):
    e, G, D, K, P, R = 2 if c["dtype"] == "bf16" else 4, c["G"], c["D"], c["K"], c["exact"], c["recent"]
    idx = _index(c)
    dst = np.nonzero(idx != np.arange(c["B"]))[0]
    src = np.unique(idx[dst])
    if c["window_from"] >= 0:
        row = (R - c["window_from"]) * (3 * G * D * e + 9)
        return {"bytes": int(row * (dst.size + src.size)) + c["B"] * 8, "flops": 0}
    slots, rows, L = _counts(c).sum((1, 2, 3)), _prefix_rows(c).sum(1), _geometry(c)[1]
    pool = P if c["levels"] else 0
    # Slots with their bookkeeping, the packed prefix, the pool, the window, the clusters' scalars.
    each = (slots * (2 * D * e + 37) + rows * (2 * D * e + 4) + pool * (2 * G * D * e + 14) + R * (3 * G * D * e + 9)
            + G * K * (2 * L + 4 * D + 29) + 8 * G)
    return {"bytes": int(each[src].sum() + each[idx[dst]].sum()) + c["B"] * 8, "flops": 0}


# ------------------------------------------------------------------ entry points
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1009 + case["shape"])
    st = {"tree": _prepare_tree, "beam": _prepare_beam, "reorder": _prepare_reorder}[case["op"]](case, gen)
    st["op"] = case["op"]
    return st


def _plain_state(case, seed):
    """prepare() of the plain form, whichever form is being measured."""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def run(state):
    return {"tree": _run_tree, "beam": _run_beam, "reorder": _run_reorder}[state["op"]](state)


def exact(case, seed):
    if case["op"] == "tree":
        return _exact_tree(case, seed)
    if case["op"] == "beam":
        return _exact_beam(case, seed)
    return None          # rows are moved, nothing is computed


def work(case):
    if case["op"] == "tree":
        return _work_tree(case)
    if case["op"] == "beam":
        e = 2 if case["dtype"] == "bf16" else 4
        n = case["N"] * case["W"]
        # Per logit: the maximum, the difference, the sum, the comparison with the best so far.
        return {"bytes": n * case["V"] * e + n * 4 + case["N"] * case["k"] * 20, "flops": 4 * n * case["V"]}
    return _work_reorder(case)
