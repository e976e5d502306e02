"""Penalties, biases and masks on logits (adjust_logits) against their 64-bit form."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")


def each(value, r, rows):
    return value.reshape(rows)[r].item() if isinstance(value, torch.Tensor) and value.dim() else value


def reference(x, history=None, lengths=None, prompt=0, repetition=1.0, presence=0.0, frequency=0.0, bias=None, mask=None):
    """(result float64, bound, touched) per row.

    Bound: the quotient or product, the penalty's product and sum (one fused), the difference and every biased sum are
    float32 operations, each off by at most 2^-24 of its value, which the sum of the magnitudes bounds; the result is
    rounded once to the storage type."""
    V = x.size(-1)
    rows = x.numel() // V
    z = x.double().cpu().numpy().reshape(rows, V).copy()
    size = np.abs(z)
    touched = np.zeros((rows, V), bool)
    hist = None if history is None else history.cpu().numpy().reshape(rows, -1)
    for r in range(rows):
        if hist is not None:
            L = hist.shape[1]
            n = min(max(each(lengths, r, rows) if lengths is not None else L, 0), L)
            p = min(max(each(prompt, r, rows), 0), n)
            rep, pres, freq = (each(t, r, rows) for t in (repetition, presence, frequency))
            seen = hist[r, :n]
            seen = np.unique(seen[(seen >= 0) & (seen < V)])
            z[r, seen] = np.where(z[r, seen] > 0, z[r, seen] / rep, z[r, seen] * rep)
            size[r, seen] = np.abs(z[r, seen])
            touched[r, seen] = True
            new = hist[r, p:n]
            v, c = np.unique(new[(new >= 0) & (new < V)], return_counts=True)
            z[r, v] -= freq * c + pres
            size[r, v] += 2 * (np.abs(freq) * c + abs(pres)) + np.abs(z[r, v])
        if bias is not None:
            t, b = (y.cpu().numpy() for y in bias)
            t, b = (y.reshape(rows, -1)[r] if y.ndim > 1 else y for y in (t, b))
            for tok in np.unique(t[(t >= 0) & (t < V)]):
                mine = b[t == tok].astype(np.float64)
                z[r, tok] += mine.sum()
                size[r, tok] += len(mine) * np.abs(mine).sum() + np.abs(z[r, tok])
                touched[r, tok] = True
        if mask is not None:
            w = mask.cpu().numpy().reshape(-1, mask.size(-1))
            bits = np.unpackbits(w[r if len(w) > 1 or mask.dim() > 1 else 0].view(np.uint8), bitorder="little")[:V]
            z[r, bits == 0] = -np.inf
    u = torch.finfo(x.dtype).eps / 2 if x.dtype == BF16 else 0.0
    size = np.where(np.isfinite(size), size, 0)
    bound = 2.0 ** -24 * 2 * size + u * np.abs(np.where(np.isfinite(z), z, 0)) * 1.001 + 1e-44
    return z, bound, touched


def check(x, inplace=False, out=None, **kw):
    from logkv_b200 import adjust_logits
    want, bound, touched = reference(x, **kw)
    before = x.clone()
    got = adjust_logits(x, out=x if inplace else out, **kw)
    assert got.shape == x.shape and got.dtype == x.dtype
    if not inplace:
        assert torch.equal(x.view(torch.int16 if x.dtype == BF16 else torch.int32),
                           before.view(torch.int16 if x.dtype == BF16 else torch.int32))
    V = x.size(-1)
    y = got.double().cpu().numpy().reshape(-1, V)
    same = (y == want) | (np.isnan(y) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        near = np.abs(y - want) <= bound
    assert (same | near).all(), np.argwhere(~(same | near))[:5]
    old = before.double().cpu().numpy().reshape(-1, V)
    free = ~touched & (want != -np.inf)
    assert ((y == old) | np.isnan(old))[free].all()
    return got


def inputs(N, W, V, L, K, dtype, seed, wide=False, masked=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
    it = torch.int64 if wide else torch.int32
    x = (torch.randn(N, W, V, generator=gen, device="cuda") * 3).to(dtype)
    kw = dict(history=(V * rand(N, W, L) ** 3).to(it) - (rand(N, W, L) < 0.05).to(it) * V)
    kw["lengths"], kw["prompt"] = (rand(N, W) * (L + 1)).to(it), (rand(N, W) * (L + 1)).to(it)
    kw["repetition"], kw["presence"], kw["frequency"] = 0.7 + rand(N, W), rand(N, W) - 0.5, rand(N, W) - 0.5
    if K:
        kw["bias"] = ((V * rand(N, W, K)).to(it) - 1, 4 * rand(N, W, K) - 2)
    if masked:
        kw["mask"] = (rand(N, W, (V + 31) // 32) * 2 ** 32 - 2 ** 31).to(torch.int32)
    return x, kw


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,W,V,L,K", [(1, 1, 1, 1, 1), (2, 3, 5, 9, 7), (1, 2, 31, 40, 3), (3, 1, 32, 7, 0), (2, 2, 33, 0, 4),
                                       (1, 4, 1000, 300, 20), (2, 5, 4099, 1031, 0), (1, 3, 50021, 5000, 300),
                                       (40, 16, 2051, 65, 5), (40, 16, 9001, 33, 0)])
def test_against_64_bits(dtype, N, W, V, L, K):
    """Slices of every size; rows that start anywhere; without history, biases or mask, and with all of them."""
    for wide in (False, True):
        x, kw = inputs(N, W, V, L, K, dtype, V + wide, wide)
        check(x, **kw)
        check(x.flatten(0, 1), **{name: (tuple(t.flatten(0, 1) for t in v) if name == "bias" else v.flatten(0, 1))
                                  for name, v in kw.items()})
    hist = kw["history"]
    check(x, history=hist, repetition=1.5)
    check(x, history=hist, lengths=L // 2, prompt=L // 4, frequency=0.25, presence=-1.5)
    check(x, mask=kw["mask"][0, 0])
    check(x, mask=kw["mask"])
    if K:
        check(x, bias=(kw["bias"][0][0, 0], kw["bias"][1][0, 0]))
    assert torch.equal(check(x), x)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_and_places(dtype):
    """A vocabulary padded to another length, rows off every alignment, outputs given, and in place."""
    for V, pad, off in ((1000, 8, 0), (1003, 5, 0), (999, 4, 1), (2051, 1, 3), (515, 13, 7)):
        x, kw = inputs(3, 2, V, 50, 6, dtype, V)
        base = torch.full((3, 2, V + pad), 7.0, dtype=dtype, device="cuda")
        view = base[:, :, off:off + V] if off + V <= V + pad else base[:, :, :V]
        view.copy_(x)
        a = check(view, **kw)
        room = torch.zeros(3 * 2 * V + 3, dtype=dtype, device="cuda")
        b = check(view, out=room[1:1 + 6 * V].view(3, 2, V), **kw)
        assert torch.equal(a.nan_to_num(), b.nan_to_num()) and room[0] == 0 and not room[1 + 6 * V:].any()
        c = check(view, inplace=True, **kw)
        assert c is view and torch.equal(a.nan_to_num(), c.nan_to_num())
        left = torch.ones(V + pad, dtype=torch.bool, device="cuda")
        left[view.storage_offset():view.storage_offset() + V] = False
        assert (base[:, :, left] == 7).all()
        swapped = x.transpose(0, 1).contiguous().transpose(0, 1)     # requests inside beams
        assert torch.equal(check(swapped, **kw).nan_to_num(), a.nan_to_num())
    x, kw = inputs(2, 2, 640, 30, 4, dtype, 9)
    a = check(x.transpose(1, 2).contiguous().transpose(1, 2), **kw)  # vocabulary not contiguous
    assert torch.equal(a.nan_to_num(), check(x, **kw).nan_to_num())
    from logkv_b200 import adjust_logits
    room = torch.zeros(2, 2, 1280, dtype=dtype, device="cuda")
    with pytest.raises(ValueError, match="memory of its own"):
        adjust_logits(room[..., 640:], out=room.view(-1)[:2560].view(2, 2, 640))
    with pytest.raises(ValueError, match="share memory"):
        adjust_logits(one := room[:1, :1, :640].expand(2, 2, 640), out=one)
    grown = torch.full((2, 2, 90), 3, dtype=torch.int32, device="cuda")   # a history buffer with room
    grown[..., :30] = kw["history"]
    assert torch.equal(check(x, **{**kw, "history": grown[..., :30]}).nan_to_num(), a.nan_to_num())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_that_are_not_finite(dtype):
    V = 700
    x, kw = inputs(1, 3, V, 400, 30, dtype, 4)
    at = torch.arange(V, device="cuda")
    x[:, :, at % 7 == 0], x[:, :, at % 11 == 0], x[:, :, at % 13 == 0] = -INF, INF, float("nan")
    x[:, :, 100:110] = torch.finfo(dtype).min
    got = check(x, **kw)
    banned = check(x, mask=torch.zeros((V + 31) // 32, dtype=torch.int32, device="cuda"))
    assert (banned == -INF).all()
    # The last word's bits past the vocabulary do not matter.
    full = torch.full(((V + 31) // 32,), -1, dtype=torch.int32, device="cuda")
    full[-1] = (1 << V % 32) - 1
    assert torch.equal(check(x, mask=full).nan_to_num(), x.nan_to_num())
    assert not torch.equal(got.nan_to_num(), x.nan_to_num())


def test_repeated_entries():
    """Every token of the history and every bias the same one: one counter takes them all; the sums keep their order."""
    x = torch.zeros(1, 1, 3000, device="cuda")
    hist = torch.full((1, 1, 4000), 2047, device="cuda")
    y = check(x, history=hist, frequency=0.5, presence=3.0)
    assert y[0, 0, 2047] == -2003 and y.count_nonzero() == 1
    tok = torch.full((1024,), 5, device="cuda")
    val = torch.randn(1024, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda") * 1e3
    a = check(x, bias=(tok, val))
    for _ in range(3):
        assert torch.equal(check(x, bias=(tok, val)), a)
    # Any length and prompt a device tensor holds is clamped.
    odd = torch.tensor([[-5], [9000]], device="cuda")
    check(x.expand(2, 1, 3000).contiguous(), history=hist.expand(2, 1, 4000), lengths=odd, prompt=odd.flip(0),
          frequency=0.5, repetition=2.0)


def test_capture_replay_and_streams():
    from logkv_b200 import adjust_logits
    x, kw = inputs(4, 3, 5000, 100, 8, F32, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        adjust_logits(x, **kw)
        with torch.cuda.graph(graph, stream=side):
            out = adjust_logits(x, **kw)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (5, 6):
        new, more = inputs(4, 3, 5000, 100, 8, F32, seed)
        x.copy_(new)
        for name in kw:
            for old, t in zip(kw[name] if name == "bias" else (kw[name],), more[name] if name == "bias" else (more[name],)):
                old.copy_(t)
        graph.replay()
        assert torch.equal(out, adjust_logits(new, **more))


def test_in_front_of_beam_selection():
    """Banned tokens are not chosen and the scores are those of the adjusted distribution; a row with every token
    banned offers nothing."""
    from logkv_b200 import adjust_logits, beam_select
    x, kw = inputs(2, 3, 800, 60, 5, F32, 8)
    kw["mask"][1, 2] = 0
    y = adjust_logits(x, **kw)
    scores = torch.zeros(2, 3, device="cuda")
    s, rows, tokens = beam_select(y, scores, 4)
    want, _, _ = reference(x, **kw)
    flat = torch.log_softmax(torch.from_numpy(want), -1).view(2, -1).nan_to_num(nan=-INF).cuda()
    top = flat.topk(4, -1)[0]
    assert (s.double() - top).abs().max() < 1e-4
    assert (rows[1] != 5).all()
    bits = kw["mask"].view(6, -1)[rows.view(-1), tokens.view(-1) >> 5] >> (tokens.view(-1) & 31) & 1
    assert bits.all()


def test_repeated_calls_are_checked_like_the_first():
    """The host binding takes calls that fit; everything else is refused or done as the first call is."""
    from logkv_b200 import adjust_logits as f
    x, kw = inputs(2, 3, 70, 5, 4, F32, 3)
    want = f(x, **kw)
    assert torch.equal(f(x, **kw), want)
    h, n = kw["history"], kw["lengths"]
    t, b = kw["bias"]
    for args, more, match in [
            (x[0, 0], {}, "logits must be"), (x.half(), {}, "dtype"), (x, {"repetition": 0.0}, "positive"),
            (x, {"repetition": float("inf")}, "finite"), (x, {"presence": float("nan")}, "finite"),
            (x, {"repetition": b}, "repetition must be"), (x, {"presence": n}, "presence must be"),
            (x, {"history": h[0]}, "history must be"), (x, {"history": h.float()}, "history must be"),
            (x, {"history": h.cpu()}, "history must be"), (x, {"lengths": 6}, "at most"), (x, {"lengths": -1}, "negative"),
            (x, {"lengths": n[0]}, "lengths must be"), (x, {"history": None}, "without a history"), (x, {"prompt": -2}, "negative"),
            (x, {"bias": (t, b[..., :3])}, "one shape"), (x, {"bias": (t[0, 0], b)}, "one shape"), (x, {"bias": (b, b)}, "bias tokens"),
            (x, {"mask": kw["mask"][..., :2]}, "3 words"), (x, {"mask": kw["mask"].long()}, "mask must be")]:
        with pytest.raises(ValueError, match=match):
            f(args, **{**kw, **more})
    with pytest.raises(NotImplementedError):
        f(x.clone().requires_grad_(), **kw)
    with pytest.raises(NotImplementedError):
        f(x, **{**kw, "presence": kw["presence"].clone().requires_grad_()})
    for name in ("lengths", "prompt", "repetition", "presence"):      # strided numbers
        t2 = kw[name].t().contiguous().t()
        assert torch.equal(f(x, **{**kw, name: t2}), want)
    wide = torch.zeros(2, 3, 9, dtype=h.dtype, device="cuda")         # rows of unlike distances
    wide[..., :5] = h
    assert torch.equal(f(x, **{**kw, "history": wide[..., :5]}), want)
    across = h.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(f(x, **{**kw, "history": across}), want)
    assert f(x[:0], history=h[:0]).shape == (0, 3, 70)
    assert torch.equal(f(x, **{**kw, "repetition": torch.full((2, 3), 1.5, device="cuda")}), f(x, **{**kw, "repetition": 1.5}))
    assert torch.equal(f(x, **{**kw, "repetition": 2}), f(x, **{**kw, "repetition": 2.0}))
    for bad in (x.to_sparse(), x.to(torch.float32).to_sparse()):      # no strides to look at
        with pytest.raises((RuntimeError, ValueError)):
            f(bad, **kw)
    with pytest.raises((RuntimeError, ValueError)):
        f(x, **{**kw, "mask": kw["mask"].to_sparse()})
