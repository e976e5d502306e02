"""Beam selection against its 64-bit form, and beam search over decoders against one cache per beam."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from hypotheses import make_cache

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")


def reference(logits, scores, k, keep):
    """(scores float64, rows, tokens) in numpy float64; beams and places as documented."""
    x = logits.double().cpu().numpy()
    r = scores.double().cpu().numpy()
    N, W, V = x.shape
    out_s = np.full((N, k), -np.inf)
    out_r = np.arange(N)[:, None] * W + np.minimum(np.arange(k), W - 1)
    out_t = np.zeros((N, k), np.int64)
    for n in range(N):
        total = np.full((W, V), -np.inf)
        for w in range(W):
            top = x[n, w].max()
            if np.isfinite(r[n, w]) and np.isfinite(top):
                total[w] = r[n, w] + (x[n, w] - (top + math.log(np.exp(x[n, w] - top).sum())))
        flat = total.reshape(-1)
        order = np.argsort(-flat, kind="stable")[:k]
        order = order[flat[order] > -np.inf]
        where = list(range(k))
        if keep:
            first = {}
            for i, f in enumerate(order):
                first.setdefault(f // V, i)
            free = [p for p in range(W) if p not in first]
            where = [f // V if first[f // V] == i else free.pop(0) for i, f in enumerate(order)]
        for i, f in enumerate(order):
            out_s[n, where[i]], out_r[n, where[i]], out_t[n, where[i]] = flat[f], n * W + f // V, f % V
    return out_s, out_r, out_t


def check(logits, scores, k, keep=False):
    """Rows and tokens equal; scores off by their own rounding (2^-24 relative) and the sums' error: every
    term of the sum of exponentials is off by less than 2^-20 relative (the rounded difference and product,
    each half a unit of a number below 2^5 where the term matters, and the exponential), a thread's 32
    terms add 2^-19."""
    from logkv_b200 import beam_select
    got = beam_select(logits, scores, k, keep_places=keep)
    torch.cuda.synchronize()
    want = reference(logits, scores, k, keep)
    assert torch.equal(got[1].cpu(), torch.from_numpy(want[1]))
    assert torch.equal(got[2].cpu(), torch.from_numpy(want[2]))
    s = got[0].double().cpu().numpy()
    none = want[0] == -np.inf
    assert (s[none] == -np.inf).all()
    err = np.abs(s[~none] - want[0][~none])
    assert (err <= 2.0 ** -24 * np.abs(want[0][~none]) + 2.0 ** -18).all(), err.max()


def draw(N, W, V, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(N, W, V, generator=gen, device="cuda") * 3).to(dtype)
    return x, -5 * torch.rand(N, W, generator=gen, device="cuda")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,W,V,k,keep", [
    (1, 1, 1, 1, False), (1, 1, 1, 1, True), (3, 2, 1, 2, True), (2, 1, 7, 7, False), (1, 3, 5, 15, False),
    (2, 4, 33, 8, False), (5, 3, 500, 3, True), (1, 1, 4095, 1, False), (1, 1, 4096, 32, False), (2, 1, 4097, 33, False),
    (1, 2, 16384, 64, False), (1, 2, 16385, 65, False), (2, 5, 50021, 5, True), (1, 4, 32000, 8, False),
    (1, 16, 40001, 128, False), (60, 5, 16391, 10, False), (1, 128, 300, 128, True), (2, 256, 77, 100, False),
    (300, 2, 1000, 4, False), (1, 1, 300000, 17, False)])
def test_selection(dtype, N, W, V, k, keep):
    x, r = draw(N, W, V, dtype, seed=V + k)
    check(x, r, k, keep)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties_go_to_the_lowest_index(dtype):
    """Equal logits everywhere, equal beams, and many equal logits at the border (more than are gathered)."""
    x = torch.zeros(2, 3, 20001, device="cuda", dtype=dtype)
    r = torch.zeros(2, 3, device="cuda")
    r[1] = torch.tensor([-1.0, 0.0, 0.0])
    for k in (1, 3, 40, 128):
        check(x, r, k)
    check(x, r, 3, True)
    gen = torch.Generator(device="cuda").manual_seed(1)
    y = torch.randint(0, 3, (2, 3, 40000), generator=gen, device="cuda").to(dtype)
    y[:, :, :100] = -7.0
    check(y, r, 64)
    z = torch.full((1, 256, 500), -1.0, device="cuda", dtype=dtype)     # ties over many lists
    check(z, torch.zeros(1, 256, device="cuda"), 128)
    z[0, 200, 499] = 0.0
    check(z, torch.zeros(1, 256, device="cuda"), 128)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_flat_distributions(dtype):
    """Uniform logits over many slices (every one ties), and two levels split in the middle of a slice."""
    x = torch.full((2, 3, 151936), 1.5, device="cuda", dtype=dtype)
    r = torch.tensor([[0.0, 0.0, 0.0], [-2.0, -1.0, -3.0]], device="cuda")
    check(x, r, 32)
    x[:, :, 70000:] = 1.75
    check(x, r, 32)
    x[0, 2, 151935] = 2.0
    check(x, r, 3, True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_and_broken_logits(dtype):
    low = torch.finfo(dtype).min
    x, r = draw(8, 4, 9001, dtype, seed=2)
    x[0, 0] = -INF                       # a beam without a finite logit
    x[0, 1, 1:] = -INF                   # one finite logit
    x[1, 2, 77] = float("nan")
    x[1, 0, 9000] = INF
    x[2] = -INF                          # nothing at all
    x[3, :, 10:] = -INF                  # fewer continuations than places
    x[4, :, 20:] = low                   # masked with the type's lowest value
    x[5, 1] = low                        # ... in every place: a flat distribution
    r[5, 0] = -INF
    r[5, 2] = float("nan")
    r[6] = torch.tensor([0.0, -INF, -INF, -INF])
    r[7, 1] = INF
    for k, keep in ((4, True), (4, False), (60, False)):
        check(x, r, k, keep)


def test_uneven_places():
    """The best of a slice all in one thread's registers, and increasing and decreasing logits."""
    base = torch.linspace(-20, 20, 60000, device="cuda")
    x = torch.stack([base, base.flip(0), torch.zeros_like(base)])[None].contiguous()
    x[0, 2, 40:48] = torch.arange(8, device="cuda") * 0.5 + 3
    r = torch.tensor([[0.0, -0.25, 5.0]], device="cuda")
    for k in (1, 7, 8, 64, 128):
        check(x, r, k)
    check(x.bfloat16(), r, 128)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(dtype):
    """Rows at every offset from a 16-byte boundary, padded vocabularies, sliced and transposed beams."""
    from logkv_b200 import beam_select
    x, r = draw(3, 4, 5003, dtype, seed=3)
    wide, _ = draw(3, 4, 5040, dtype, seed=4)
    for off in range(9):
        v = wide[:, :, off:off + 5003]
        v.copy_(x)
        want = reference(x, r, 6, False)
        got = beam_select(v, r, 6)
        assert torch.equal(got[1].cpu(), torch.from_numpy(want[1])) and torch.equal(got[2].cpu(), torch.from_numpy(want[2]))
        wide.normal_()                   # values around the view are not read as logits
    check(x.transpose(0, 1), r.t(), 5)
    check(x[:, ::2], r[:, ::2], 2, True)
    check(x[:, :1].expand(3, 4, 5003), r, 9)
    check(x.transpose(1, 2).contiguous().transpose(1, 2), r, 3)


def test_streams_graphs_and_repeats():
    from logkv_b200 import beam_select
    sets = [draw(4, 5, 30000, d, seed=s) for s, d in ((5, F32), (6, BF16))]
    first = [beam_select(x, r, 7) for x, r in sets]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for s, (x, r) in zip(streams, sets):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(beam_select(x, r, 7))
        graphs.append(g)
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(first, outs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    x, r = sets[0]
    x.copy_(draw(4, 5, 30000, F32, seed=9)[0])
    torch.cuda.synchronize()
    graphs[0].replay()
    torch.cuda.synchronize()
    want = reference(x, r, 7, False)
    assert torch.equal(outs[0][1].cpu(), torch.from_numpy(want[1])) and torch.equal(outs[0][2].cpu(), torch.from_numpy(want[2]))


def test_no_requests_and_refusals():
    from logkv_b200 import beam_select
    x, r = draw(2, 3, 100, F32)
    assert [t.shape for t in beam_select(x[:0], r[:0], 4)] == [(0, 4)] * 3
    beam_select(x, r, 3)                 # from here on the host binding takes the calls it covers
    for args, kw, match in [((x, r.cpu(), 3), {}, "one device"), ((x.half(), r, 3), {}, "not supported"),
                            ((x, r[:1], 3), {}, "scores must be"), ((x, r, 0), {}, "k must be"),
                            ((x, r, 301), {}, "k must be"), ((x, r, 2), {"keep_places": True}, "keep_places"),
                            ((x[0], r, 2), {}, "logits must be")]:
        with pytest.raises(ValueError, match=match):
            beam_select(*args, **kw)
    assert [t.shape for t in beam_select(x[:0], r[:0], 4)] == [(0, 4)] * 3


# ---------------------------------------------------------------- beam search over decoders
class Toy:
    """A model of `layers` attention layers over LogKV decoders: embeddings to q, k, v per layer, logits
    from the last layer's output."""

    def __init__(self, layers, H, G, D, V, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        mk = lambda *s: torch.randn(*s, generator=gen, device="cuda") * 0.7  # noqa: E731
        self.q, self.k, self.v = mk(layers, V, H, D), mk(layers, V, G, D), mk(layers, V, G, D)
        self.head = mk(H * D, V)

    def __call__(self, decoders, tokens, position):
        y = 0
        for i, d in enumerate(decoders):
            pick = lambda t: t[i][tokens][:, :, None].bfloat16()  # noqa: E731
            n = tokens.numel()
            ends = (tokens % 5 == 0).to(torch.uint8).view(n, 1)
            out = d.step(pick(self.q), pick(self.k), pick(self.v), k_raw=pick(self.k),
                         input_pos=torch.full((n, 1), position, device="cuda"), span_ends_device=ends)
            y = y + out.float()
        return y.reshape(tokens.numel(), -1) @ self.head


@pytest.mark.parametrize("steps,granularity", [(9, 32), (60, 16)])
def test_beam_search_equals_one_cache_per_row(steps, granularity):
    """LogKVBeams against the same search in which every step copies whole caches row by row with torch
    indexing; long enough in the second case that the window overflows and flushes in between."""
    from logkv_b200.decode import LogKVBeams, LogKVDecoder
    from test_reorder_gpu import ROWS
    N, W, V, D = 2, 3, 101, 64
    mk = lambda s: make_cache(BF16, B=N * W, G=2, D=D, K=4, levels=2, R=20, recent=32, granularity=granularity, seed=s)  # noqa: E731
    model = Toy(2, 4, 2, D, V, seed=21)
    ours = [LogKVDecoder(mk(s), D ** -0.5) for s in (22, 23)]
    theirs = [LogKVDecoder(mk(s), D ** -0.5) for s in (22, 23)]

    def take(decoders, index):
        for d in decoders:
            for n in ROWS:
                t = getattr(d.cache, n)
                t.copy_(t[index].clone())
            for t in (d._k, d._v, d._kr, d._pos, d._ends):
                t.copy_(t[index].clone())
            d.cache._ladder_epoch += 1

    beams = LogKVBeams(ours, N, W)
    beams.fork()
    take(theirs, torch.tensor([0, 0, 0, 3, 3, 3], device="cuda"))
    scores = torch.full((N, W), -INF, device="cuda")
    scores[:, 0] = 0
    tokens = torch.tensor([7, 7, 7, 9, 9, 9], device="cuda")
    for step in range(steps):
        a = model(ours, tokens, 500 + step)
        b = model(theirs, tokens, 500 + step)
        assert torch.equal(a, b), step
        tokens, rows = beams.advance(a)
        want = reference(b.view(N, W, V), scores, W, True)
        index = torch.from_numpy(want[1]).cuda().view(-1)
        assert torch.equal(rows, index) and torch.equal(tokens.cpu(), torch.from_numpy(want[2]).view(-1)), step
        scores = beams.scores.clone()
        take(theirs, index)
        for x, y in zip(ours, theirs):
            for n in ROWS:
                assert torch.equal(getattr(x.cache, n), getattr(y.cache, n)), (step, n)
    flushed = ours[0].cache._flush_cursor > 0
    assert flushed == (steps == 60)


def test_pending_host_flags_cannot_be_reordered():
    from logkv_b200.decode import LogKVBeams, LogKVDecoder
    d = LogKVDecoder(make_cache(BF16, B=2, G=1, D=64, R=4, seed=24), 0.125)
    q = torch.randn(2, 1, 1, 64, device="cuda").bfloat16()
    d.step(q, q, q, k_raw=q, span_ends=[[False], [True]])
    with pytest.raises(RuntimeError, match="span_ends_device"):
        d.reorder([1, 0])
    with pytest.raises(ValueError, match="rows"):
        LogKVBeams([d], 2, 2)


# ---------------------------------------------------------------- large finite logits
def masked_requests(dtype, V, low, seed):
    """Four requests of three beams: few live tokens, beams masked throughout or but for one token, every
    beam masked, and the first half masked."""
    x, r = draw(4, 3, V, dtype, seed=seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x[0, :, torch.randperm(V, generator=gen, device="cuda")[30:]] = low
    x[1, 1] = low
    x[1, 2, 1:] = low
    x[2] = low
    x[3, :, :V // 2] = low
    return x, r


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [-1e4, -1e9, -1e10, -1e20, -1e30, None])
def test_logits_masked_with_large_numbers(dtype, low):
    """Masks of every magnitude, over one slice and over many.  Scores near a mask's magnitude are rounded
    in float64 (1e10: 2e-6), which the tolerance's 2^-18 covers."""
    low = torch.finfo(dtype).min if low is None else low
    for V in (520, 40000):
        x, r = masked_requests(dtype, V, low, seed=31)
        for k, keep in ((3, True), (8, False), (64, False)):
            check(x, r, k, keep)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("high", [2e6, 5e9, 1e30, None])
def test_large_maxima(dtype, high):
    """A few logits far above the others, and beams of nothing else: the others count for nothing."""
    high = torch.finfo(dtype).max if high is None else high
    x, r = draw(3, 4, 40000, dtype, seed=32)
    x[0, :, 7::5000] = high              # eight places
    x[1, 1] = high
    x[1, 3, 39999] = high
    x[2, 0, :4] = high
    x[2, 0, 30000:30002] = high / 2
    for k, keep in ((4, True), (8, False)):
        check(x, r, k, keep)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [1500, 5003, 20007])
def test_ties_at_every_alignment(dtype, V):
    """More equal logits than are gathered, in views at every offset from a 16-byte boundary: larger values
    in front of a row and behind it are not its own."""
    r = torch.tensor([[0.0, -0.5, -0.25], [-1.0, 0.0, -2.0]], device="cuda")
    for off in (*range(9), 24):          # 24: the last row ends where the buffer does
        wide = torch.full((2, 3, V + 24), 7.0, device="cuda", dtype=dtype)
        x = wide[:, :, off:off + V]
        x.fill_(1.5)
        x[1, 1, V - 1] = x[1, 2, 0] = 1.75
        check(x, r, 7)
        x.fill_(-1e30)
        x[0, 0, ::400] = 1.0
        check(x, r, 3, True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [37, 500, 5003, 16384, 50021, 151936])
def test_equal_beams_tie(dtype, V):
    """Beams with the same logits and score tie token by token, whatever their rows' alignment and slices:
    the lower beam comes first."""
    x, r = draw(5, 6, V, dtype, seed=33 + V)
    x[:, 1] = x[:, 0]
    x[:, 4] = x[:, 0]
    x[:, 5] = x[:, 2]
    r[:, 1] = r[:, 4] = r[:, 0]
    r[:, 5] = r[:, 2]
    for k, keep in ((6, True), (6, False), (24, False)):
        check(x, r, k, keep)
    same, _ = draw(7, 1, V, dtype, seed=34 + V)
    check(same.expand(7, 16, V).contiguous(), torch.zeros(7, 16, device="cuda"), 33)


def test_gradients_are_refused_not_dropped():
    from logkv_b200 import beam_select
    x, r = draw(2, 3, 100, F32)
    want = beam_select(x, r, 3)          # from here on the host binding takes the calls it covers
    for a, b in ((x.clone().requires_grad_(), r), (x, r.clone().requires_grad_())):
        with pytest.raises(NotImplementedError, match="forward-only"):
            beam_select(a, b, 3)
        with torch.no_grad():
            got = beam_select(a, b, 3)
        assert not got[0].requires_grad and all(torch.equal(s, t) for s, t in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [40, 501, 30001])
def test_scores_closer_than_float32_sums(dtype, V):
    """Beams whose best scores differ by 1e-9 or so (all but certain tokens, equal beam scores), chosen and at
    the border of the choice: float64's order.  The scores of two beams are at least 1e-12 apart, where
    float64 sums in another order are off by 1e-15."""
    x = torch.empty(3, 12, V, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(35)
    for n in range(3):
        for w, c in enumerate(torch.randperm(12, generator=g, device="cuda").tolist()):
            x[n, w] = -(20.0 + c / 2) - torch.rand(V, generator=g, device="cuda")
            x[n, w, (7 * w) % V] = 0.0
    x = x.to(dtype)
    r = torch.tensor([-0.5, -3.0, 0.0], device="cuda")[:, None].expand(3, 12).contiguous()
    for k, keep in ((12, True), (12, False), (5, False), (1, False), (60, False)):
        check(x, r, k, keep)
    x[1, 3] = x[1, 9]                    # and two that are equal
    check(x, r, 12, True)
