"""Refusals of the hypothesis-decoding operators, checked on the host before anything is launched."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from hypotheses import make_cache, random_tree, visible


@pytest.fixture(scope="module")
def lib():
    from logkv_b200 import build
    build.build()
    from logkv_b200 import _lib
    return _lib.lib()


@pytest.fixture()
def cache(lib):
    return make_cache(torch.float32, B=2, G=2, D=64, levels=0, R=5, device="cpu")


def test_visible_follows_the_parents():
    p = np.array([[-1, 0, 0, 2, -2, 4, -1, 9]])
    see = visible(p)[0]
    assert [np.nonzero(r)[0].tolist() for r in see] == [[0], [0, 1], [0, 2], [0, 2, 3], [], [], [6], []]
    assert visible(random_tree(np.random.RandomState(0), 3, 9))[:, np.arange(9), np.arange(9)].all()


def test_tree_refusals(cache):
    from logkv_b200 import log_kv_tree_attention as f
    q, k = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 3, 64)
    for args, match in [
            ((q[:1], k, k, [-1, 0, 1]), "q must be"), ((q[..., :32], k, k, [-1, 0, 1]), "q must be"),
            ((q[0], k, k, [-1, 0, 1]), "q must be"), ((q.bfloat16(), k, k, [-1, 0, 1]), "q must be"),
            ((q, k[:, :1], k, [-1, 0, 1]), "k must be"), ((q, k, k[:, :, :2], [-1, 0, 1]), "v shape"),
            ((q, k.bfloat16(), k, [-1, 0, 1]), "dtype"), ((q[:, :, :2], k, k, [-1, 0]), "same drafted tokens"),
            ((q[:, :3], k, k, [-1, 0, 1]), "multiple"), ((q, k, k, [-1, 0]), "parents must be"),
            ((q, k, k, [[-1, 0, 1]]), "parents must be"), ((q, k, k, [-1.0, 0, 1]), "integers"),
            ((q, k, k, [0, 0, 1]), "earlier token"), ((q, k, k, [-1, 2, 1]), "earlier token"),
            ((q, k, k, [-1, -3, 1]), "earlier token"),
            ((torch.zeros(2, 4, 257, 64), torch.zeros(2, 2, 257, 64), torch.zeros(2, 2, 257, 64), [-1] * 257), "at most")]:
        with pytest.raises(ValueError, match=match):
            f(cache, *args[:3], 0.125, args[3])
    with pytest.raises(NotImplementedError):
        f(cache, q.requires_grad_(), k, k, 0.125, [-1, 0, 1])
    with pytest.raises(ValueError, match="out must be"):
        f(cache, q.detach(), k, k, 0.125, [-1, 0, 1], out=torch.zeros(2, 4, 3, 32))


def test_tree_c_abi_checks(lib):
    from logkv_b200 import _lib
    layout = _lib.Layout(1, 8, 128, 12, 7, 125, 4096, 256, 64, 1, 1, 1.0, 2048.0, 1.0)
    size = lambda lay, *a: lib.logkv_tree_attention_workspace_bytes(ctypes.byref(lay), *a)  # noqa: E731
    assert size(layout, 16, 7, 10756) > 0 and size(layout, 8, 256, 10756) > 0 and size(layout, 8, 1, 0) > 0
    assert size(layout, 12, 7, 10756) == 0 and size(layout, 16, 0, 10756) == 0 and size(layout, 16, 257, 10756) == 0
    odd = _lib.Layout(1, 8, 96, 12, 7, 125, 4096, 256, 64, 1, 1, 1.0, 2048.0, 1.0)
    f32 = _lib.Layout(1, 8, 256, 12, 7, 125, 4096, 256, 64, 1, 0, 1.0, 2048.0, 1.0)
    assert size(odd, 16, 7, 10756) == 0 and size(f32, 16, 7, 10756) == 0
    state, pre, args = _lib.State(), _lib.Prefix(), _lib.TreeArgs()
    call = lambda a, n: lib.logkv_tree_attention(ctypes.byref(layout), ctypes.byref(state), ctypes.byref(pre),  # noqa: E731
                                                 ctypes.byref(a), 1 << 20, n, None)
    args.heads, args.tokens = 16, 7
    assert call(args, 1 << 30) == -4                      # null pointers
    assert lib.logkv_tree_attention(None, None, None, None, None, 0, None) == -4
    for name in ("recent_k", "recent_v"):
        setattr(state, name, 1 << 20)
    pre.k = pre.v = pre.mass = pre.length = 1 << 20
    pre.capacity = 10756
    args.q = args.k_new = args.v_new = args.out = args.parents = 1 << 20
    assert call(args, 16) == -3                           # workspace too small
    args.q_strides[2] = 4
    assert call(args, 1 << 30) == -4                      # rows not 16-byte aligned
    args.q_strides[2] = 8
    args.recent_count = 4097
    assert call(args, 1 << 30) == -1
    args.recent_count, args.heads = 0, 15
    assert call(args, 1 << 30) == -1


def test_reorder_refusals(cache):
    for index, match in [([0], "row indices must be"), ([[0, 1]], "row indices must be"), ([0.0, 1.0], "integers"),
                         ([0, 2], "in \\[0, 2\\)"), ([-1, 0], "in \\[0, 2\\)"),
                         (torch.tensor([0, 1], dtype=torch.uint8), "integers")]:
        with pytest.raises(ValueError, match=match):
            cache.reorder_batch(index)
    for w in (-1, 6):
        with pytest.raises(ValueError, match="window_from"):
            cache.reorder_batch([0, 1], window_from=w)
    from logkv_b200 import _SemanticReplayUpdates
    with cache._semantic_update_context(_SemanticReplayUpdates()):
        with pytest.raises(RuntimeError, match="update tapes"):
            cache.reorder_batch([0, 1])
    cache._deferred_take = 4
    with pytest.raises(RuntimeError, match="commit_deferred"):
        cache.reorder_batch([0, 1])
    k = torch.zeros(2, 2, 3, 64)
    with pytest.raises(RuntimeError, match="commit_deferred"):
        cache.add_recent_path(k, k, [0], k_raw=k, span_ends=[[0, 0, 0]] * 2)


def test_path_refusals(cache):
    k = torch.zeros(2, 2, 3, 64)
    ends = [[False] * 3] * 2
    f = lambda *a, **kw: cache.add_recent_path(*a, **{"k_raw": k, "span_ends": ends, **kw})  # noqa: E731
    for args, kw, match in [((k[:1], k, [0]), {}, "k must be"), ((k, k[:, :, :2], [0]), {}, "v must be"),
                            ((k, k, [0]), {"k_raw": k[..., :32]}, "k_raw must be"), ((k, k, [0.5]), {}, "integers"),
                            ((k, k, [[0]]), {}, "path must be"), ((k, k, torch.zeros(1, 2, 1).long()), {}, "path must be"),
                            ((k, k, [3]), {}, "path entries"), ((k, k, [-1]), {}, "path entries"),
                            ((k, k, [0]), {"span_ends": None}, "boundaries"), ((k, k, [0]), {"span_ends": ends[:1]}, "boundaries"),
                            ((k, k, [0]), {"span_ends_device": torch.zeros(2, 1)}, "boundaries"),
                            ((k, k, [0]), {"input_pos": torch.zeros(2)}, "input_pos length"),
                            ((k, k, [0] * 257), {}, "exceeds recent_size")]:
        with pytest.raises(ValueError, match=match):
            f(*args, **kw)
    before = cache.recent_count
    f(k, k, [])
    assert cache.recent_count == before
    cache.token_count = cache.max_seq_length
    with pytest.raises(RuntimeError, match="token overflow"):
        f(k, k, [0])


def test_reorder_c_abi_checks(lib):
    from logkv_b200 import _lib
    layout = _lib.Layout(4, 8, 128, 12, 7, 125, 4096, 256, 64, 1, 1, 1.0, 2048.0, 1.0)
    state = _lib.State(**{n: 1 << 20 for n in _lib.STATE_FIELDS})
    call = lambda lay, st, rc, w, idx: lib.logkv_reorder_batch(  # noqa: E731
        ctypes.byref(lay), ctypes.byref(st), None, rc, w, idx, 1, None, None)
    assert call(layout, state, 10, -1, None) == -4
    assert call(layout, _lib.State(), 10, -1, 1 << 20) == -4
    assert call(layout, state, 4097, -1, 1 << 20) == -1 and call(layout, state, 10, 11, 1 << 20) == -1
    assert call(layout, state, 10, -2, 1 << 20) == -1
    big = _lib.Layout(4096, 8, 128, 12, 7, 125, 4096, 256, 64, 1, 1, 1.0, 2048.0, 1.0)
    assert call(big, state, 10, -1, 1 << 20) == -1
    rows = (_lib.Rows * 2)(_lib.Rows(None, 8), _lib.Rows(1 << 20, 8))
    assert lib.logkv_reorder_rows(rows, 2, 4, 1 << 20, 1, None, None) == -4
    assert lib.logkv_reorder_rows(rows, 41, 4, 1 << 20, 1, None, None) == -1
    assert lib.logkv_reorder_rows(None, 1, 4, 1 << 20, 1, None, None) == -4
    chunk = _lib.Chunk()
    assert lib.logkv_window_append_path(ctypes.byref(layout), ctypes.byref(state), ctypes.byref(chunk), 4, None, 0, 1,
                                        0, None, None) == -4
    assert lib.logkv_window_append_path(ctypes.byref(layout), ctypes.byref(state), ctypes.byref(chunk), 0, 1 << 20, 0,
                                        1, 0, None, None) == -1


def test_beam_refusals(lib):
    from logkv_b200 import beam_select
    x, r = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    for args, kw, match in [((x[0], r, 1), {}, "logits must be"), ((x.double(), r, 1), {}, "not supported"),
                            ((x, r[:1], 1), {}, "scores must be"), ((x, r.double(), 1), {}, "scores must be"),
                            ((x, r, 0), {}, "k must be"), ((x, r, 31), {}, "k must be"),
                            ((torch.zeros(1, 1, 500), torch.zeros(1, 1), 129), {}, "k must be"),
                            ((x, r, 2), {"keep_places": True}, "keep_places"),
                            ((torch.zeros(1, 257, 2), torch.zeros(1, 257), 2), {}, "supported range"),
                            ((x[:, :, :0], r, 1), {}, "k must be"), ((x, r, 3), {}, "CUDA")]:
        with pytest.raises(ValueError, match=match):
            beam_select(*args, **kw)


def test_beam_c_abi_checks(lib):
    from logkv_b200 import _lib
    size = lib.logkv_beam_workspace_bytes
    assert size(2, 4, 32000, 8) > 0 and size(1, 1, 1, 1) > 0
    for bad in [(0, 4, 10, 1), (1, 0, 10, 1), (1, 257, 10, 1), (1, 1, 0, 1), (1, 1, 4, 5), (1, 4, 1000, 129),
                (1, 4, 1000, 0), (16384, 4, 10, 1), (1, 4, 1 << 29, 1)]:
        assert size(*bad) == 0, bad
    a = _lib.BeamArgs()
    call = lambda n: lib.logkv_beam_select(ctypes.byref(a), 1 << 20, n, None)  # noqa: E731
    assert lib.logkv_beam_select(None, None, 0, None) == -4
    assert call(1 << 30) == -1
    a.requests, a.width, a.vocab, a.k = 2, 4, 100, 8
    assert call(1 << 30) == -4
    a.logits = a.scores = a.out_scores = a.out_rows = a.out_tokens = 1 << 20
    assert call(16) == -3
    a.keep_places = 1
    assert call(1 << 30) == -1
    a.keep_places, a.dtype = 0, 7
    assert call(1 << 30) == -2


@pytest.fixture()
def two_layers(lib, monkeypatch):
    """Two decoders over host caches whose row moves are recorded in ``moves`` instead of launched, and a
    selection that keeps every beam."""
    from logkv_b200 import decode
    moves = []
    layers = [decode.LogKVDecoder(make_cache(torch.float32, B=4, G=2, D=64, levels=0, R=5, device="cpu", recent=32),
                                  0.125) for _ in range(2)]
    for i, d in enumerate(layers):
        def move(index, *, window_from=None, i=i, c=d.cache):
            c._check_reorder(window_from)
            moves.append((i, window_from))
        monkeypatch.setattr(d.cache, "reorder_batch", move)
    monkeypatch.setattr(decode, "beam_select", lambda logits, scores, k, keep_places: (
        scores - 1, torch.arange(4).view(2, 2), torch.zeros(2, 2, dtype=torch.int64)))
    return decode.LogKVBeams(layers, 2, 2), moves


@pytest.mark.parametrize("why,match", [("flags", "span_ends_device"), ("op_log", "op-log"), ("deferred", "commit_deferred")])
def test_beams_refuse_before_anything_moves(two_layers, why, match):
    """A layer that cannot be reordered leaves the scores and the other layers as they were."""
    beams, moves = two_layers
    last = beams.decoders[1]
    if why == "flags":
        last.pending, last._ends_host = True, [[False]] * 4
    elif why == "op_log":
        last.cache.op_log = torch.zeros(1)
    else:
        last.cache._deferred_take = 4
    beams.scores[:] = torch.tensor([[0.0, -2.0], [-1.0, -3.0]])
    before = beams.scores.clone()
    for call in (beams.fork, lambda: beams.advance(torch.zeros(4, 10))):
        with pytest.raises(RuntimeError, match=match):
            call()
        assert moves == [] and torch.equal(beams.scores, before) and beams._forked is None


def test_beams_keep_the_scores_of_a_failed_step(two_layers):
    beams, moves = two_layers
    beams.fork()
    assert moves == [(0, None), (1, None)]
    beams.advance(torch.zeros(4, 10))
    assert moves[2:] == [(0, 5), (1, 5)]
    before = beams.scores.clone()
    beams.decoders[1].cache.recent_count = 3         # fewer window rows than at the fork
    with pytest.raises(ValueError, match="window_from"):
        beams.advance(torch.zeros(4, 10))
    assert torch.equal(beams.scores, before) and len(moves) == 4


def test_a_reset_cache_moves_whole_rows(two_layers):
    """What a fork said about the window holds until the cache is filled anew, whose rows may differ
    anywhere."""
    beams, moves = two_layers
    beams.fork()
    for d in beams.decoders:
        d.cache.reset_parameters()
        d.cache.recent_count = d.cache.token_count = 9
    beams.advance(torch.zeros(4, 10))
    assert moves[2:] == [(0, None), (1, None)]
    beams.fork()
    beams.advance(torch.zeros(4, 10))
    assert moves[6:] == [(0, 9), (1, 9)]


def test_beam_gradients_are_refused(lib):
    from logkv_b200 import beam_select
    x, r = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    for a, b in ((x.clone().requires_grad_(), r), (x, r.clone().requires_grad_())):
        with pytest.raises(NotImplementedError, match="forward-only"):
            beam_select(a, b, 3)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            beam_select(a, b, 3)


def test_reorder_of_too_many_rows(lib):
    """More batch rows than one call takes are refused with the number, by the cache and before a beam step."""
    from logkv_b200 import _lib, decode
    cache = make_cache(torch.float32, B=514, G=1, D=16, K=2, levels=0, R=1, P=8, recent=8, max_seq=64, device="cpu")
    for call in (lambda: cache.reorder_batch(list(range(514))),
                 decode.LogKVBeams([decode.LogKVDecoder(cache, 0.25)], 257, 2).fork):
        with pytest.raises(ValueError, match=f"514 batch rows.*{_lib.REORDER_MAX_BATCH}"):
            call()


@pytest.mark.parametrize("what", ["torch", "python"])
def test_host_binding_of_another_torch_or_python(lib, monkeypatch, what):
    """A binding built for another torch or interpreter is not loaded, the error asks for a build, and the
    build does one."""
    import sysconfig
    from logkv_b200 import _lib, build
    assert _lib.host().__file__ == build.host_file()
    built = []
    monkeypatch.setattr(build, "build_host", lambda: built.append(build.host_file()))
    build.build()
    assert built == []
    monkeypatch.setattr(_lib, "_host", None)
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "0.0.0+none")
    else:
        monkeypatch.setattr(sysconfig, "get_config_var", lambda name: ".cpython-000-none.so")
    with pytest.raises(RuntimeError, match="logkv_b200.build"):
        _lib.host()
    build.build()
    assert built == [build.host_file()]
