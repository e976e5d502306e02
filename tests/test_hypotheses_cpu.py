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
