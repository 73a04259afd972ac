"""Refusals of the C entries for trees of drafted tokens, and their workspace sizes, on the CPU: every call here returns from
host-side validation (pointers are never dereferenced)."""

from __future__ import annotations

import ctypes
import math

import pytest

from torch2vk_amd import _lib

OK, NULL, SHAPE, DTYPE, UNSUPPORTED, ARG, WORKSPACE, ALIGN = 0, 1, 2, 3, 4, 5, 6, 7
P, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1002)


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libt2h.so not built")
    return _lib.lib()


def attn(lib, **kw):
    a = dict(q=P, q_row=2048, k_new=P, k_row=1024, v_new=P, v_row=1024, q_norm_w=None, k_norm_w=None, eps=1e-6, theta=1e6, lengths=P,
             parents=None, counts=None, k_cache=P, k_seq=64 * 1024, v_cache=P, v_seq=64 * 1024, s_cap=64, out=P, n=4, n_seq=2, nh=16,
             nk=8, d=128, workspace=P, workspace_bytes=0, stream=None)
    return lib.t2h_attn_tree(*(a | kw).values())


def test_attention_refuses(lib):
    for name in ("q", "k_new", "v_new", "lengths", "k_cache", "v_cache", "out", "workspace"):
        assert attn(lib, **{name: None}) == NULL, name
    assert attn(lib, q_norm_w=P) == NULL
    assert attn(lib, d=64) == UNSUPPORTED
    assert attn(lib, nh=17 * 8, q_row=17 * 1024) == UNSUPPORTED
    for kw in (dict(nh=15), dict(nh=0), dict(nk=0), dict(n_seq=0), dict(n=65), dict(s_cap=0), dict(s_cap=0x80000000),
               dict(s_cap=2 ** 29, k_seq=2 ** 42, v_seq=2 ** 42), dict(q_row=2047), dict(k_row=1023), dict(v_row=1000), dict(k_seq=64 * 1024 - 8), dict(v_seq=8)):
        assert attn(lib, **kw) == SHAPE, kw
    for kw in (dict(k_cache=ODD), dict(v_cache=ODD), dict(out=ODD), dict(workspace=ODD), dict(k_seq=64 * 1024 + 4)):
        assert attn(lib, **kw) == ALIGN, kw
    assert attn(lib) == WORKSPACE
    assert attn(lib, n=0) == OK  # no rows: nothing is launched


def test_attention_workspace(lib):
    size = lib.t2h_attn_tree_workspace_bytes
    assert size(1, 8, 16, 8, 128, 2048) > 0
    for shape in ((0, 8, 16, 8, 128, 64), (1, 0, 16, 8, 128, 64), (1, 65, 16, 8, 128, 64), (1, 8, 15, 8, 128, 64), (1, 8, 16, 0, 128, 64),
                  (1, 8, 16, 8, 64, 64), (1, 8, 16, 8, 128, 0), (1, 8, 34, 2, 128, 64)):
        assert size(*shape) == 0, shape


def verify(lib, **kw):
    a = dict(logits=P, row_stride=100, draft=None, draft_stride=0, dtype=0, tokens=P, parents=None, counts=None, uniforms=P,
             temperature=1.0, temperatures=None, path=P, kept=P, next_token=P, n=4, n_seq=2, vocab=100, workspace=P,
             workspace_bytes=0, stream=None)
    return lib.t2h_tree_verify(*(a | kw).values())


def test_verification_refuses(lib):
    for name in ("logits", "tokens", "path", "kept", "next_token", "workspace", "uniforms"):
        assert verify(lib, **{name: None}) == NULL, name
    assert verify(lib, uniforms=None, temperature=0.0, temperatures=P) == NULL
    assert verify(lib, dtype=2) == DTYPE
    for kw in (dict(n=0), dict(n=65), dict(n_seq=0), dict(vocab=0), dict(vocab=0x80000000, row_stride=1 << 40), dict(row_stride=99),
               dict(draft=P, draft_stride=99)):
        assert verify(lib, **kw) == SHAPE, kw
    for kw in (dict(temperature=math.inf), dict(temperature=math.nan), dict(draft=P, draft_stride=100, parents=P)):
        assert verify(lib, **kw) == ARG, kw
    for kw in (dict(logits=ODD), dict(logits=ctypes.c_void_p(0x1001), dtype=1), dict(draft=ODD, draft_stride=100),
               dict(workspace=ODD)):
        assert verify(lib, **kw) == ALIGN, kw
    assert verify(lib) == WORKSPACE
    assert verify(lib, uniforms=None, temperature=0.0) == WORKSPACE  # greedy needs no numbers


def test_verification_workspace(lib):
    size = lib.t2h_tree_verify_workspace_bytes
    assert 0 < size(2, 4, 100, 0) <= size(2, 4, 100, 1)
    for shape in ((0, 4, 100, 0), (1, 0, 100, 0), (1, 65, 100, 0), (1, 4, 0, 0)):
        assert size(*shape) == 0, shape


def keep(lib, **kw):
    a = dict(k_cache=P, k_layer=2 * 64 * 1024, k_seq=64 * 1024, v_cache=P, v_layer=2 * 64 * 1024, v_seq=64 * 1024, layers=3, s_cap=64,
             path=P, kept=P, lengths=P, n=4, n_seq=2, nk=8, d=128, stream=None)
    return lib.t2h_tree_keep(*(a | kw).values())


def test_keeping_refuses(lib):
    for name in ("k_cache", "v_cache", "path", "kept", "lengths"):
        assert keep(lib, **{name: None}) == NULL, name
    assert keep(lib, d=64) == UNSUPPORTED
    for kw in (dict(n=0), dict(n=65), dict(n_seq=0), dict(layers=0), dict(nk=0), dict(s_cap=0), dict(k_seq=8), dict(v_layer=8)):
        assert keep(lib, **kw) == SHAPE, kw
    for kw in (dict(k_cache=ODD), dict(v_cache=ODD), dict(k_seq=64 * 1024 + 4), dict(v_layer=4 * 64 * 1024 + 4)):
        assert keep(lib, **kw) == ALIGN, kw
