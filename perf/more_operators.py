"""Workloads of a decoding step of several hypotheses, from the projections to the next tokens.

  rotate   queries and keys rotated at their positions (``logkv_b200.log_kv_rotate``);
  append   unrotated keys and values into the cache's window, rotated on the way
           (``LogStructuredKVCache.add_recent_rotated``);
  shared   attention of batch rows that share a long prefix, read once for all of them
           (``logkv_b200.log_kv_shared_attention``);
  logits   penalties of repeated tokens, biases and grammar masks (``logkv_b200.adjust_logits``).

``own`` chooses between the framework's kernels and the plain form: elementary torch operations in
float32.  Lengths and occupancies are fixed by a case's ``shape`` number, values by the seed.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def _rotate(name, **kw):
    """B rows of T tokens, G KV groups of rf query heads, head dim D of which `n` features rotate, tables of
    `rows` positions; `fused`: q, k and v are slices of one projection's output."""
    c = dict(op="rotate", name=name, dtype="bf16", B=1, T=1, G=8, rf=2, D=128, n=128, layout="half", rows=32768,
             fused=True, each=False)
    c.update(kw)
    return c


def _append(name, **kw):
    """T tokens of B rows behind `recent` window rows of `window`."""
    c = dict(op="append", name=name, dtype="bf16", B=1, T=2, G=8, D=128, n=128, layout="half", rows=32768,
             window=2048, recent=1000, each=True)
    c.update(kw)
    return c


def _shared(name, **kw):
    """R requests of W rows that agree in the packed prefix (K clusters of `slots` budgeted slots, `levels`
    occupied levels, `exact` pool rows) and in the window's first `w0` rows of `recent`; T query tokens over
    Tk new tokens."""
    c = dict(op="shared", name=name, dtype="bf16", R=1, W=4, G=8, rf=2, D=128, K=12, slots=128, exact=256,
             max_seq=32768, levels=4, window=2048, recent=1500, w0=1436, T=1, Tk=1, shape=1)
    c.update(kw)
    return c


def _logits(name, **kw):
    """rows x V logits, `L` tokens of history (`prompt` of them the prompt's), `bias` biased tokens a row,
    `mask`: part of the rows under a grammar; `each`: every row its own penalties and lengths."""
    c = dict(op="logits", name=name, dtype="fp32", N=1, W=4, V=32000, L=64, prompt=16, bias=0, mask=False, each=False,
             shape=1)
    c.update(kw)
    return c


def listed():
    return [
        # One decoding step of eight sequences: launch latency only.
        _rotate("rotate_decode_b8", B=8, each=True),
        # A prompt chunk of one window.
        _rotate("rotate_chunk_2048", T=2048),
        # Four sequences' chunks of a checkpoint with interleaved pairs, a quarter of the head rotated.
        _rotate("rotate_interleaved_part", B=4, T=1777, G=4, rf=5, D=64, n=16, layout="interleaved", dtype="fp32",
                each=True),
        # The pair of tokens that 64 sequences commit together.
        _append("append_pair_b64", B=64),
        # Window-sized chunks of eight sequences.
        _append("append_chunk_b8", B=8, T=2048, recent=2048),
        # One request with four beams over a 32K-token compressed cache, some steps after the fork.
        _shared("shared_r1_w4", shape=41),
        # The largest: eight requests of eight beams; a pending token beside the new one.
        _shared("shared_r8_w8", R=8, W=8, recent=2040, w0=1800, Tk=2, shape=42),
        # Three requests of sixteen beams, odd head grouping, short context, two drafted tokens each.
        _shared("shared_r3_w16_rf5", R=3, W=16, G=4, rf=5, D=64, K=8, slots=64, exact=64, max_seq=8192, levels=3,
                window=1024, recent=777, w0=700, T=2, Tk=2, shape=43),
        # A float32 cache, five samples of two prompts.
        _shared("shared_fp32_r2_w5", dtype="fp32", R=2, W=5, G=4, rf=3, D=64, K=8, slots=64, exact=64, max_seq=8192,
                window=512, recent=301, w0=256, shape=44),
        # Four beams of one request, a few tokens in: latency.
        _logits("logits_w4", shape=51),
        # A batch at an odd vocabulary, every row with its own penalties and biases, long histories.
        _logits("logits_n29_w5", N=29, W=5, V=50021, L=4097, prompt=3000, bias=37, each=True, shape=52),
        # The largest: wide beams over a 151936-token vocabulary, all of it.
        _logits("logits_n32_w16", dtype="bf16", N=32, W=16, V=151936, L=1024, prompt=512, bias=16, mask=True, each=True,
                shape=53),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "shared", "logits"])
    shape = rng.randrange(1, 1 << 20)
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op in ("rotate", "append"):
        D, G, rf = rng.choice([32, 64, 80, 128, 256]), rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 7, 8])
        n = rng.choice([D, D, D // 2, D // 4, 2 * rng.randrange(1, D // 2 + 1)])
        layout = rng.choice(["half", "half", "interleaved"])
        width = G * (rf + 2) * D
        if op == "rotate":
            most = (9_000_000 if dtype == "fp32" else 18_000_000) // width
            T = _log_int(rng, 1, min(4096, most))
            B = _log_int(rng, 1, max(1, min(64, most // T)))
            return _rotate("", dtype=dtype, B=B, T=T, G=G, rf=rf, D=D, n=n, layout=layout,
                           rows=rng.choice([8192, 32768, 131072]), fused=rng.random() < 0.7, each=rng.random() < 0.5)
        window = rng.choice([64, 512, 2048])
        T = _log_int(rng, 1, window)
        B = _log_int(rng, 1, max(1, min(64, 8 * 2048 * 8 * 128 // (G * D * T))))
        return _append("", dtype=dtype, B=B, T=T, G=G, D=D, n=n, layout=layout, window=window,
                       rows=rng.choice([8192, 32768]), recent=rng.randrange(0, window - T + 1),
                       each=rng.random() < 0.5)
    if op == "logits":
        W, V, L = _log_int(rng, 1, 16), _log_int(rng, 300, 151936), _log_int(rng, 1, 8192)
        N = _log_int(rng, 1, max(1, min(64, 70_000_000 // (W * (V + 8 * L)))))
        return _logits("", dtype=dtype, N=N, W=W, V=V, L=L, prompt=rng.randrange(0, L + 1),
                       bias=rng.choice([0, 0, 1, rng.randrange(1, 300)]), mask=rng.random() < 0.5,
                       each=rng.random() < 0.6, shape=shape)
    D, G, K = rng.choice([64, 128]), rng.choice([1, 2, 4, 8]), rng.choice([4, 8, 12])
    slots, levels, window = rng.choice([32, 64, 128]), rng.randrange(0, 5), rng.choice([256, 512, 2048])
    recent = rng.randrange(0, window + 1)
    tail = min(recent, _log_int(rng, 1, 600) - 1)
    W, T = _log_int(rng, 1, 32), rng.choice([1, 1, 1, 2, 3, 5])
    Tk = T if T > 1 else rng.choice([1, 2])
    rf = rng.choice([1, 2, 3, 4, 5, 7, 8])
    row = G * (K * levels * slots + 64 + recent + Tk) * D * (4 if dtype == "fp32" else 2)
    work = row * rf * T * (8 if dtype == "fp32" else 1)                # per row, against the largest listed case's
    R = _log_int(rng, 1, max(1, min(8, 64 // W, 64 * 8 * 8304 * 128 * 2 * 2 // (work * W))))
    return _shared("", dtype=dtype, R=R, W=W, G=G, rf=rf, D=D, K=K, slots=slots, exact=64, max_seq=8192, levels=levels,
                   window=window, recent=recent, w0=recent - tail, T=T, Tk=Tk, shape=shape)


# ------------------------------------------------------------------ rotation
def _tables(rows, n):
    """[rows, n] cosines and sines in both halves of the rotated features."""
    inv = 1.0 / (1e6 ** (np.arange(0, n, 2, dtype=np.float64) / n))
    ang = np.arange(rows, dtype=np.float64)[:, None] * inv[None]
    ang = np.concatenate([ang, ang], 1)
    return torch.from_numpy(np.cos(ang).astype(np.float32)).cuda(), torch.from_numpy(np.sin(ang).astype(np.float32)).cuda()


def _positions(c, gen):
    """Positions of the T tokens: [T], or each row's own [B, T]; consecutive from anywhere in the tables."""
    B, T = c["B"], c["T"]
    start = torch.randint(0, c["rows"] - T + 1, (B if c["each"] else 1, 1), generator=gen, device="cuda")
    pos = start + torch.arange(T, device="cuda")
    return pos if c["each"] else pos[0]


def _small_cache(c, cos, sin, window):
    """A cache with nothing flushed."""
    from logkv_b200 import LogStructuredKVCache
    shape = (c["B"], c["G"], c["rows"], c["D"])
    return LogStructuredKVCache(
        shape, shape, B=16, recent_size=window, device="cuda", dtype=DTYPES[c["dtype"]], semantic_clusters=True,
        semantic_anchor_mode="mid", allocate_second_order=False, cluster_k_max=4, semantic_flush_granularity=window,
        alpha_exact_tokens=16, alpha_span_max_tokens=8, beta_novelty=True, beta_adaptive_merge=True, cos_cache=cos,
        sin_cache=sin, rope_n_elem=c["n"])


def _halves(x, n):
    """Interleaved pairs of the first n features as halves."""
    return torch.cat([x[..., 0:n:2], x[..., 1:n:2], x[..., n:]], -1)


def _rotated(x, cos, sin, n):
    """x [B, heads, T, D] float32 in halves, tables [.., T, n]."""
    a = x[..., :n]
    turned = torch.cat([-a[..., n // 2:], a[..., :n // 2]], -1)
    return torch.cat([a * cos + turned * sin, x[..., n:]], -1)


def _rows_of(table, pos):
    """Table rows of positions [T] or [B, T] as [1 or B, 1, T, n]."""
    return table[pos if pos.dim() == 2 else pos[None]][:, None]


def _prepare_rotate(c, gen):
    dt, B, T, G, H, D = DTYPES[c["dtype"]], c["B"], c["T"], c["G"], c["G"] * c["rf"], c["D"]
    cos, sin = _tables(c["rows"], c["n"])
    pos = _positions(c, gen)
    if c["fused"]:
        # As one projection leaves them: [B, T, (H + 2 G) D], seen as [B, heads, T, D].
        x = torch.randn(B, T, H + 2 * G, D, generator=gen, device="cuda", dtype=dt).transpose(1, 2)
        q, k = x[:, :H], x[:, H:H + G]
    else:
        q = torch.randn(B, H, T, D, generator=gen, device="cuda", dtype=dt)
        k = torch.randn(B, G, T, D, generator=gen, device="cuda", dtype=dt)
    st = {"q": q, "k": k, "pos": pos, "layout": c["layout"], "n": c["n"], "cos": cos, "sin": sin}
    if own:
        st["cache"] = _small_cache(c, cos, sin, 8)
    return st


def _run_rotate(st):
    q, k, pos, layout, n = st["q"], st["k"], st["pos"], st["layout"], st["n"]
    if own:
        from logkv_b200 import log_kv_rotate
        out = log_kv_rotate(st["cache"], q, k, pos, layout=layout)
        return out if layout == "interleaved" else out[:2]          # in halves the raw keys are k itself
    cos, sin = _rows_of(st["cos"], pos), _rows_of(st["sin"], pos)
    if layout == "interleaved":
        raw = _halves(k, n)
        return (_rotated(_halves(q, n).float(), cos, sin, n).to(q.dtype),
                _rotated(raw.float(), cos, sin, n).to(q.dtype), raw)
    return _rotated(q.float(), cos, sin, n).to(q.dtype), _rotated(k.float(), cos, sin, n).to(q.dtype)


def _exact_rotated(x, pos, cos, sin, n, layout):
    """Feature pair by feature pair, in 64 bits."""
    B, _, T, _ = x.shape
    at = pos if pos.dim() == 2 else pos.expand(B, T)
    out = x.double().clone()
    for i in range(n // 2):
        lo, hi = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + n // 2)
        a, b = x[..., lo].double(), x[..., hi].double()
        c, s = cos[:, i].double()[at][:, None], sin[:, i].double()[at][:, None]
        out[..., i], out[..., i + n // 2] = a * c - b * s, a * s + b * c
    return out


def _exact_rotate(c, seed):
    st = _plain_state(c, seed)
    args = (st["pos"], st["cos"], st["sin"], st["n"], st["layout"])
    out = _exact_rotated(st["q"], *args), _exact_rotated(st["k"], *args)
    return out + (None,) if c["layout"] == "interleaved" else out


def _work_rotate(c):
    e = 2 if c["dtype"] == "bf16" else 4
    q, k = c["B"] * c["G"] * c["rf"] * c["T"] * c["D"], c["B"] * c["G"] * c["T"] * c["D"]
    at = c["T"] * (c["B"] if c["each"] else 1)
    raw = k if c["layout"] == "interleaved" else 0
    rotated = (q + k) // c["D"] * c["n"]
    return {"bytes": (2 * (q + k) + raw) * e + at * (8 * c["n"] // 2 + 8), "flops": 3 * rotated}


# ------------------------------------------------------------------ append
def _prepare_append(c, gen):
    dt, B, T, G, D = DTYPES[c["dtype"]], c["B"], c["T"], c["G"], c["D"]
    cos, sin = _tables(c["rows"], c["n"])
    pos = _positions(c, gen)
    x = torch.randn(B, T, 2 * G, D, generator=gen, device="cuda", dtype=dt).transpose(1, 2)
    st = {"k": x[:, :G], "v": x[:, G:], "pos": pos, "ends": torch.rand(B, T, generator=gen, device="cuda") < 0.05,
          "layout": c["layout"], "n": c["n"], "at": c["recent"], "cos": cos, "sin": sin}
    st["ends"] = st["ends"].to(torch.uint8)
    if own:
        st["cache"] = _small_cache(c, cos, sin, max(c["window"], c["recent"] + T))
    else:
        rows = (B, G, 2 * max(c["window"], c["recent"] + T), D)
        st["rows"] = [torch.zeros(rows, device="cuda", dtype=dt) for _ in range(3)]
        st["recent_pos"] = torch.zeros(B, rows[2], device="cuda", dtype=torch.int64)
        st["recent_ends"] = torch.zeros(B, rows[2], device="cuda", dtype=torch.uint8)
    return st


def _run_append(st):
    k, v, pos, layout, n, at = st["k"], st["v"], st["pos"], st["layout"], st["n"], st["at"]
    to = at + k.size(2)
    if own:
        cache = st["cache"]
        cache.recent_count = cache.token_count = at        # the rows of the pass before are given up again
        cache.add_recent_rotated(k, v, input_pos=pos, layout=layout, span_ends_device=st["ends"])
        return (cache.recent_k[:, :, at:to], cache.recent_k_raw[:, :, at:to], cache.recent_v[:, :, at:to],
                cache.recent_pos[:, at:to])
    raw = _halves(k, n) if layout == "interleaved" else k
    rk, rr, rv = st["rows"]
    rk[:, :, at:to] = _rotated(raw.float(), _rows_of(st["cos"], pos), _rows_of(st["sin"], pos), n).to(k.dtype)
    rr[:, :, at:to] = raw
    rv[:, :, at:to] = v
    st["recent_pos"][:, at:to] = pos
    st["recent_ends"][:, at:to] = st["ends"]
    return rk[:, :, at:to], rr[:, :, at:to], rv[:, :, at:to], st["recent_pos"][:, at:to]


def _exact_append(c, seed):
    st = _plain_state(c, seed)
    return (_exact_rotated(st["k"], st["pos"], st["cos"], st["sin"], st["n"], st["layout"]), None, None, None)


def _work_append(c):
    e, rows = 2 if c["dtype"] == "bf16" else 4, c["B"] * c["T"]
    at = c["T"] * (c["B"] if c["each"] else 1)
    return {"bytes": rows * (c["G"] * c["D"] * e * 5 + 10) + at * (8 * c["n"] // 2 + 8), "flops": 3 * rows * c["G"] * c["n"]}


# ------------------------------------------------------------------ shared prefix
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
    """[R, G, K, L] occupied slots per level, the same for all rows of a request."""
    Bs, L = _geometry(c)
    rs = np.random.RandomState(c["shape"])
    n = np.zeros((c["R"], c["G"], c["K"], L), np.int64)
    used = min(c["levels"], L)
    if used:
        n[..., :used] = rs.randint(Bs // 2, Bs + 1, n[..., :used].shape)
        if c["levels"] >= 4:      # a long context: three levels of four are full
            n[..., 1:used] = np.where(rs.rand(*n[..., 1:used].shape) < 0.9, Bs, n[..., 1:used])
    return n


def _prefix_rows(c):
    """[R, G] rows of the packed prefix: the occupied slots, then the exact pool."""
    return _counts(c).sum((2, 3)) + (c["exact"] if c["levels"] else 0)


def _buffers(c, gen):
    """Ladder and pool of every request by name; slots past a level's count hold an empty cache's values."""
    dt, R, G, D, K, P = DTYPES[c["dtype"]], c["R"], c["G"], c["D"], c["K"], c["exact"]
    Bs, L = _geometry(c)
    lc = torch.from_numpy(_counts(c)).cuda()
    occ = torch.arange(Bs, device="cuda") < lc[..., None]                        # [R, G, K, L, B']

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dt)

    def ints(hi, shape):
        return torch.randint(0, hi, shape, generator=gen, device="cuda")

    # Merged masses: most slots hold a few tokens, some hundreds; their positions anywhere before.
    u = torch.rand(occ.shape, generator=gen, device="cuda").clamp_min_(1e-6)
    w = torch.where(occ, (u.log() / math.log(0.9)).floor() + 1, torch.zeros_like(u))
    P_used = P if c["levels"] else 0
    return {"level_k": normal(R, G, K, L, Bs, D) * occ[..., None], "level_v": normal(R, G, K, L, Bs, D) * occ[..., None],
            "level_w": w, "level_sum_wp": w.long() * ints(c["max_seq"], occ.shape), "level_count": lc.to(torch.int16),
            "alpha_k_raw": normal(R, G, P, D), "alpha_v": normal(R, G, P, D), "alpha_pos": ints(c["max_seq"], (R, P)),
            "alpha_valid": torch.arange(P, device="cuda").expand(R, P) < P_used}


def _packed(c, b, cos, sin):
    """The packed prefix of every request ([R, G, S, D] keys and values, [R, G, S] log-mass terms): per lane the
    occupied slots (cluster by cluster, top level first) and the exact pool, keys rotated at their positions."""
    dt, R, G, D, K, P = DTYPES[c["dtype"]], c["R"], c["G"], c["D"], c["K"], c["exact"]
    Bs, L = _geometry(c)
    n, rows = _counts(c), _prefix_rows(c)
    S, cap = int(rows.max()), K * L * Bs
    slot = np.arange(cap).reshape(K, L, Bs)[:, ::-1]
    take = np.zeros((R, G, S), np.int64)
    for i in range(R):
        for g in range(G):
            at = slot[np.arange(Bs)[None, None] < n[i, g][:, ::-1, None]]
            take[i, g, :rows[i, g]] = np.concatenate([at, cap + np.arange(rows[i, g] - at.size)])
    take = torch.from_numpy(take).cuda()
    wide = take[..., None].expand(R, G, S, D)
    w, sw = b["level_w"].view(R, G, cap), b["level_sum_wp"].view(R, G, cap)
    ww = w.long().clamp_min(1)
    pos = torch.cat([torch.div(2 * sw + ww, 2 * ww, rounding_mode="floor"), b["alpha_pos"][:, None].expand(R, G, P)], 2)
    mass = torch.cat([w.clamp_min(1).log().to(dt).float(), torch.zeros(R, G, P, device="cuda")], 2).gather(2, take)
    x = torch.cat([b["level_k"].view(R, G, cap, D), b["alpha_k_raw"]], 2).gather(2, wide).float()
    v = torch.cat([b["level_v"].view(R, G, cap, D), b["alpha_v"]], 2).gather(2, wide)
    pos = pos.gather(2, take)
    return _rotated(x, cos[pos], sin[pos], D).to(dt), v, mass


def _prepare_shared(c, gen):
    dt, R, W, G, D = DTYPES[c["dtype"]], c["R"], c["W"], c["G"], c["D"]
    B, H, w0, n = R * W, G * c["rf"], c["w0"], c["recent"]
    cos, sin = _tables(c["max_seq"] + 64, D)
    b = _buffers(c, gen)
    # The window: rows [0, w0) of a request's first row for all of its rows, the tails their own.
    win = []
    for _ in range(2):
        first = torch.randn(R, 1, G, w0, D, generator=gen, device="cuda", dtype=dt).expand(R, W, G, w0, D)
        tail = torch.randn(R, W, G, n - w0, D, generator=gen, device="cuda", dtype=dt)
        win.append(torch.cat([first, tail], 3).view(B, G, n, D))
    st = {"scale": D ** -0.5, "W": W, "w0": w0}
    for name, heads, t in (("q", H, c["T"]), ("k", G, c["Tk"]), ("v", G, c["Tk"])):
        st[name] = torch.randn(B, t, heads, D, generator=gen, device="cuda", dtype=dt).transpose(1, 2)
    if own:
        from logkv_b200 import LogStructuredKVCache
        from logkv_b200.attention import refresh_prefix
        shape = (B, G, c["max_seq"], D)
        cache = LogStructuredKVCache(
            shape, shape, B=c["slots"], recent_size=c["window"], device="cuda", dtype=dt, semantic_clusters=True,
            semantic_anchor_mode="mid", allocate_second_order=False, cluster_k_max=c["K"],
            semantic_flush_granularity=c["window"], alpha_exact_tokens=c["exact"],
            alpha_span_max_tokens=min(64, c["exact"]), beta_novelty=True, beta_adaptive_merge=True, cos_cache=cos,
            sin_cache=sin, rope_n_elem=D)
        for name, t in b.items():
            getattr(cache, name).view(R, W, *t.shape[1:]).copy_(t[:, None].expand(R, W, *t.shape[1:]))
        cache.recent_k[:, :, :n], cache.recent_v[:, :, :n] = win
        cache._row_count.fill_(c["exact"] if c["levels"] else 0)
        cache._alpha_count_dev.fill_(c["exact"] if c["levels"] else 0)
        cache.recent_count = cache.token_count = n
        cache._ladder_epoch += 1
        refresh_prefix(cache)
        st["cache"] = cache
    else:
        st["pk"], st["pv"], st["mass"] = _packed(c, b, cos, sin)
        st["rows"] = torch.from_numpy(_prefix_rows(c)).cuda()
        st["rk"], st["rv"] = win
    return st


def _run_shared(st):
    q, k, v, scale, W, w0 = st["q"], st["k"], st["v"], st["scale"], st["W"], st["w0"]
    B, H, T, D = q.shape
    G, Tk = k.size(1), k.size(2)
    tail = T if T == Tk else 0                                         # causal, or one query that sees them all
    if own:
        from logkv_b200 import log_kv_shared_attention
        return log_kv_shared_attention(st["cache"], q, k, v, scale, beams=W, window_from=w0, causal_tail=tail)
    R, rf, S = B // W, H // G, st["pk"].size(2)
    x = q.float().reshape(R, W, G, rf * T, D)
    rk, rv = st["rk"].view(R, W, G, -1, D), st["rv"].view(R, W, G, -1, D)
    qx = float(torch.tensor(1.0 / scale, dtype=q.dtype))
    # The shared keys once per request, each row's own beside them.
    xs = x.transpose(1, 2).reshape(R, G, W * rf * T, D)
    za = xs @ torch.cat([st["pk"], rk[:, 0, :, :w0]], 2).float().transpose(2, 3)
    za[..., :S] += (qx * st["mass"])[:, :, None]
    za *= scale
    dead = torch.arange(S, device=q.device) >= st["rows"][..., None]
    za[..., :S].masked_fill_(dead[:, :, None], -math.inf)
    zb = scale * (x @ torch.cat([rk[:, :, :, w0:], k.view(R, W, G, Tk, D)], 3).float().transpose(3, 4))
    if tail:
        j = torch.arange(Tk, device=q.device)
        late = (j[None, :] > j[:, None]).repeat(rf, 1)                 # rows are heads x tokens
        zb[..., zb.size(-1) - Tk:].masked_fill_(late, -math.inf)
    ma = za.amax(-1, keepdim=True) if za.size(-1) else za.new_full((*za.shape[:-1], 1), -math.inf)
    ma = ma.view(R, G, W, rf * T, 1).transpose(1, 2)
    top = torch.maximum(ma, zb.amax(-1, keepdim=True))
    ea = (za - top.transpose(1, 2).reshape(R, G, W * rf * T, 1)).exp()
    eb = (zb - top).exp()
    back = lambda t: t.view(R, G, W, rf * T, -1).transpose(1, 2)  # noqa: E731
    total = back(ea.sum(-1, keepdim=True)) + eb.sum(-1, keepdim=True)
    out = back(ea @ torch.cat([st["pv"], rv[:, 0, :, :w0]], 2).float())
    out = (out + eb @ torch.cat([rv[:, :, :, w0:], v.view(R, W, G, Tk, D)], 3).float()) / total
    return out.reshape(B, H, T, D).to(q.dtype)


def _exact_shared(c, seed):
    st = _plain_state(c, seed)
    q, k, v, W = st["q"], st["k"], st["v"], c["W"]
    B, H, T, D = q.shape
    G, Tk = k.size(1), k.size(2)
    rows, rf = _prefix_rows(c), H // G
    out = torch.zeros(B, H, T, D, dtype=torch.float64, device="cuda")
    qx = float(torch.tensor(1.0 / st["scale"], dtype=q.dtype))
    for i in range(B):
        for g in range(G):
            n = int(rows[i // W, g])
            key = torch.cat([st["pk"][i // W, g, :n], st["rk"][i, g], k[i, g]]).double()
            val = torch.cat([st["pv"][i // W, g, :n], st["rv"][i, g], v[i, g]]).double()
            bias = torch.zeros(key.size(0), dtype=torch.float64, device="cuda")
            bias[:n] = qx * st["mass"][i // W, g, :n].double()
            for t in range(T):
                m = key.size(0) - (Tk - 1 - t if T == Tk else 0)
                z = st["scale"] * (q[i, g * rf:(g + 1) * rf, t].double() @ key[:m].T + bias[:m])
                out[i, g * rf:(g + 1) * rf, t] = torch.softmax(z, -1) @ val[:m]
    return out


def _work_shared(c):
    e, B, G, D, T = 2 if c["dtype"] == "bf16" else 4, c["R"] * c["W"], c["G"], c["D"], c["T"]
    rows = int(_prefix_rows(c).sum())
    keys = rows + c["R"] * G * c["w0"] + B * G * (c["recent"] - c["w0"] + c["Tk"])
    new = T * (T + 1) // 2 if T == c["Tk"] else T * c["Tk"]
    pairs = c["W"] * c["rf"] * T * rows + B * G * c["rf"] * (T * c["recent"] + new)
    return {"bytes": keys * 2 * D * e + rows * 4 + 2 * B * G * c["rf"] * T * D * e, "flops": 4 * D * pairs}


# ------------------------------------------------------------------ logits
def _prepare_logits(c, gen):
    N, W, V, L, K = c["N"], c["W"], c["V"], c["L"], c["bias"]

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    x = torch.randn(N, W, V, generator=gen, device="cuda") * 2.5
    st = {"logits": x.to(DTYPES[c["dtype"]])}
    # Tokens of a text: a few often, most once or twice.
    st["history"] = (V * rand(N, W, L) ** 6).long().clamp_(max=V - 1).to(torch.int32)
    if c["each"]:
        st["lengths"] = (rand(N, W) * (L - c["prompt"] + 1)).to(torch.int32) + c["prompt"]
        st["prompt"] = (rand(N, W) * (c["prompt"] + 1)).to(torch.int32)
        st["repetition"], st["presence"], st["frequency"] = 1 + 0.5 * rand(N, W), rand(N, W), 0.5 * rand(N, W) - 0.1
    else:
        st["lengths"], st["prompt"] = L, c["prompt"]
        st["repetition"], st["presence"], st["frequency"] = 1.2, 0.4, 0.1
    st["bias"] = None
    if K:
        # A token may be biased twice: the biases add up.
        st["bias"] = ((V * rand(N, W, K)).long().clamp_(max=V - 1), 8 * rand(N, W, K) - 4)
    st["mask"] = None
    if c["mask"]:
        # A third of the rows under a grammar that allows a few tokens, a third under one that bans a few.
        kind = (3 * rand(N, W)).long()
        p = torch.tensor([1.0, 20.0 / V, 0.95], device="cuda")[kind]
        words = (V + 31) // 32
        st["mask"] = torch.zeros(N, W, words, dtype=torch.int32, device="cuda")
        for j in range(32):
            st["mask"] |= (rand(N, W, words) < p[..., None]).int() << j
    return st


def _run_logits(st):
    x = st["logits"]
    if own:
        from logkv_b200 import adjust_logits
        return adjust_logits(x, history=st["history"], lengths=st["lengths"], prompt=st["prompt"],
                             repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"],
                             bias=st["bias"], mask=st["mask"])
    N, W, V = x.shape
    each = lambda t: t[..., None] if isinstance(t, torch.Tensor) else t  # noqa: E731
    hist = st["history"].long()
    at = torch.arange(hist.size(-1), device=x.device)
    live, new = (at < each(st["lengths"])).expand(hist.shape), (at >= each(st["prompt"])).expand(hist.shape)
    count = torch.zeros(N, W, V, device=x.device).scatter_add_(2, hist, (live & new).float())
    seen = torch.zeros(N, W, V, device=x.device).scatter_add_(2, hist, live.float()) > 0
    y = x.float()
    y = torch.where(seen, torch.where(y > 0, y / each(st["repetition"]), y * each(st["repetition"])), y)
    y = y - (each(st["frequency"]) * count + each(st["presence"]) * (count > 0))
    if st["bias"] is not None:
        y = y + torch.zeros(N, W, V, device=x.device, dtype=torch.float64).scatter_add_(
            2, st["bias"][0], st["bias"][1].double()).float()
    if st["mask"] is not None:
        v = torch.arange(V, device=x.device)
        y = y.masked_fill((st["mask"][..., v >> 5] >> (v & 31).int() & 1) == 0, -math.inf)
    return y.to(x.dtype)


def _exact_logits(c, seed):
    st = _plain_state(c, seed)
    N, W, V = st["logits"].shape
    out = torch.empty(N, W, V, dtype=torch.float64)
    get = lambda t, n, w: t[n, w].item() if isinstance(t, torch.Tensor) else t  # noqa: E731
    for n in range(N):
        for w in range(W):
            y = st["logits"][n, w].double().cpu().numpy()
            hist = st["history"][n, w].cpu().numpy()[:get(st["lengths"], n, w)]
            rep, pres, freq = (get(st[name], n, w) for name in ("repetition", "presence", "frequency"))
            for v in np.unique(hist):
                y[v] = y[v] / rep if y[v] > 0 else y[v] * rep
            v, times = np.unique(hist[get(st["prompt"], n, w):], return_counts=True)
            y[v] -= freq * times + pres
            if st["bias"] is not None:
                np.add.at(y, st["bias"][0][n, w].cpu().numpy(), st["bias"][1][n, w].double().cpu().numpy())
            if st["mask"] is not None:
                bits = np.unpackbits(st["mask"][n, w].cpu().numpy().view(np.uint8), bitorder="little")[:V]
                y[bits == 0] = -math.inf
            out[n, w] = torch.from_numpy(y)
    return out


def _work_logits(c):
    e, rows = 2 if c["dtype"] == "bf16" else 4, c["N"] * c["W"]
    mask = (c["V"] + 31) // 32 * 4 if c["mask"] else 0
    return {"bytes": rows * (2 * c["V"] * e + c["L"] * 4 + c["bias"] * 12 + mask + (20 if c["each"] else 0)),
            "flops": rows * (4 * c["L"] + c["bias"])}


# ------------------------------------------------------------------ entry points
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1009 + case.get("shape", case.get("T", 0)))
    st = {"rotate": _prepare_rotate, "append": _prepare_append, "shared": _prepare_shared,
          "logits": _prepare_logits}[case["op"]](case, gen)
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
    return {"rotate": _run_rotate, "append": _run_append, "shared": _run_shared, "logits": _run_logits}[state["op"]](state)


def exact(case, seed):
    return {"rotate": _exact_rotate, "append": _exact_append, "shared": _exact_shared, "logits": _exact_logits}[case["op"]](
        case, seed)


def work(case):
    return {"rotate": _work_rotate, "append": _work_append, "shared": _work_shared, "logits": _work_logits}[case["op"]](case)
