"""What the trained block's operators refuse, checked before any launch (no GPU needed)."""

import ctypes

import pytest
import torch

from tao_memory_b200 import _lib, embed, expert_linear, gather_tokens, linear, return_tokens, sort_tokens

ARG = _lib.TAO_ERR_ARG


def test_no_cpu_fallback():
    x, w = torch.randn(4, 64).bfloat16(), torch.randn(32, 64).bfloat16()
    ids = torch.zeros(4, 2, dtype=torch.int64)
    for bad in (lambda: linear(x, w), lambda: expert_linear(x, w[None], torch.zeros(2, dtype=torch.int32)),
                lambda: sort_tokens(ids, 4), lambda: gather_tokens(x, None), lambda: return_tokens(x, None),
                lambda: embed(ids, w), lambda: linear(x, w[None]), lambda: expert_linear(x, w, None)):
        with pytest.raises(ValueError):
            bad()


def _linear(**kw):
    a = dict(x=16, xs=64, w=16, ws=64, we=0, up=None, us=0, ue=0, bias=None, res=None, rs=0, off=None, e=1, rows=4, n=32,
             k=64, type=0, act=0, y=16, z=None, u=None, zs=0)
    a.update(kw)
    return _lib.lib().tao_linear(*a.values(), None)


def test_linear_refusals():
    for bad in (dict(type=2), dict(act=5), dict(act=-1), dict(rows=-1), dict(n=0), dict(k=0), dict(x=None), dict(w=None),
                dict(y=None), dict(x=18), dict(w=24), dict(xs=63), dict(xs=56), dict(ws=60), dict(y=17), dict(bias=17),
                dict(res=17, rs=32), dict(e=2), dict(e=0), dict(off=16, e=513), dict(off=18, e=2, we=2048),
                dict(off=16, e=2, we=2047), dict(off=16, e=2, we=0), dict(up=16, us=64),
                dict(off=16, e=2, we=2048, bias=16), dict(off=16, e=2, we=2048, up=16, us=64, ue=2048, z=16, zs=32),
                dict(rows=(1 << 30) + 1), dict(n=(1 << 24) + 1)):
        assert _linear(**bad) == ARG, bad
    assert _linear(rows=0) == _lib.TAO_OK


def test_gradient_refusals():
    lib = _lib.lib()

    def dinput(**kw):
        a = dict(dz=16, du=None, ds=32, w=16, ws=64, we=0, up=None, us=0, ue=0, off=None, e=1, rows=4, n=32, k=64, type=0,
                 dx=16)
        a.update(kw)
        return lib.tao_linear_input_gradient(*a.values(), None)

    def dweight(**kw):
        a = dict(dz=16, du=None, ds=32, x=16, xs=64, off=None, e=1, rows=4, n=32, k=64, type=0, dw=16, dup=None)
        a.update(kw)
        return lib.tao_linear_weight_gradient(*a.values(), None)

    def slope(**kw):
        a = dict(dy=16, dys=32, z=16, u=None, zs=32, rows=4, n=32, type=0, act=2, dz=16, du=None, ds=32, db=None, ws=None,
                 size=0)
        a.update(kw)
        return lib.tao_linear_slope(*a.values(), None)

    for bad in (dict(dz=None), dict(dx=None), dict(du=16), dict(up=16), dict(ds=30), dict(dz=20), dict(w=20), dict(type=3),
                dict(dx=17)):
        assert dinput(**bad) == ARG, bad
    for bad in (dict(dz=None), dict(dw=None), dict(du=16), dict(dup=16), dict(xs=62), dict(x=24), dict(dw=17), dict(e=0)):
        assert dweight(**bad) == ARG, bad
    for bad in (dict(dy=None), dict(dz=None), dict(u=16), dict(dy=17), dict(db=16), dict(db=16, ws=16, size=64),
                dict(act=9), dict(z=None, dz=None)):
        assert slope(**bad) == ARG, bad
    assert dinput(rows=0) == _lib.TAO_OK and slope(rows=0) == _lib.TAO_OK
    assert lib.tao_linear_slope_workspace_bytes(0, 8) == 0 and lib.tao_linear_slope_workspace_bytes(1, 8) == 32


def test_token_refusals():
    lib = _lib.lib()
    assert lib.tao_sort_tokens(16, 2, 8, 4, 16, 16, 16, None, 0, None) == ARG
    assert lib.tao_sort_tokens(16, 8, 8, 0, 16, 16, 16, None, 0, None) == ARG
    assert lib.tao_sort_tokens(16, 8, 8, 513, 16, 16, 16, None, 0, None) == ARG
    assert lib.tao_sort_tokens(16, 8, -1, 4, 16, 16, 16, None, 0, None) == ARG
    assert lib.tao_sort_tokens(20, 8, 8, 4, 16, 16, 16, None, 0, None) == ARG
    assert lib.tao_sort_tokens(16, 8, 8, 4, 16, 16, None, None, 0, None) == ARG
    assert lib.tao_sort_tokens(None, 8, 8, 4, 16, 16, 16, None, 0, None) == ARG
    assert lib.tao_sort_tokens(16, 8, 100000, 4, 16, 16, 16, None, 0, None) == ARG  # no workspace
    assert lib.tao_sort_tokens_workspace_bytes(8192, 4) == 0 and lib.tao_sort_tokens_workspace_bytes(100000, 4) > 0
    assert lib.tao_gather_tokens(16, 64, 16, 4, 2, 64, 3, 16, None) == ARG
    assert lib.tao_gather_tokens(17, 64, 16, 4, 2, 64, 0, 16, None) == ARG
    assert lib.tao_gather_tokens(16, 64, 16, 4, 0, 64, 0, 16, None) == ARG
    assert lib.tao_gather_tokens(16, 64, 16, 1 << 30, 2, 64, 0, 16, None) == ARG
    assert lib.tao_gather_tokens(16, 64, 16, 0, 2, 64, 0, 16, None) == _lib.TAO_OK
    assert lib.tao_return_tokens(16, 64, 16, None, 16, 1, 4, 2, 64, 0, 16, None) == ARG  # weights of another 16-bit type
    assert lib.tao_return_tokens(16, 64, None, None, None, 0, 4, 2, 64, 0, 16, None) == ARG
    assert lib.tao_return_tokens_gradient(16, 64, None, 64, 16, None, 16, 2, 4, 2, 64, 0, 16, 16, None) == ARG
    assert lib.tao_return_tokens_gradient(16, 64, 16, 64, 16, None, None, 2, 4, 2, 64, 0, None, None, None) == ARG


def test_embedding_refusals():
    lib = _lib.lib()
    assert lib.tao_embed(16, 3, 4, 16, 64, 10, 64, 0, 1.0, 16, None) == ARG
    assert lib.tao_embed(16, 8, 4, 16, 64, 0, 64, 0, 1.0, 16, None) == ARG
    assert lib.tao_embed(16, 8, 4, 16, 64, (1 << 26) + 1, 64, 0, 1.0, 16, None) == ARG
    assert lib.tao_embed(16, 8, 4, 16, 64, 10, 64, 3, 1.0, 16, None) == ARG
    assert lib.tao_embed(20, 8, 4, 16, 64, 10, 64, 0, 1.0, 16, None) == ARG
    assert lib.tao_embed(16, 8, 4, None, 64, 10, 64, 0, 1.0, 16, None) == ARG
    assert lib.tao_embed(16, 8, 0, 16, 64, 10, 64, 0, 1.0, 16, None) == _lib.TAO_OK
    size = lib.tao_embed_gradient_workspace_bytes(100, 10, 64)
    assert size > 0
    assert lib.tao_embed_gradient(16, 8, 100, 16, 64, 10, 64, 0, 1.0, 16, 16, size - 1, None) == ARG
    assert lib.tao_embed_gradient(16, 8, 100, 16, 64, 10, 64, 0, 1.0, 16, 24, size, None) == ARG
    assert lib.tao_embed_gradient(16, 8, 100, None, 64, 10, 64, 0, 1.0, 16, 16, size, None) == ARG
    assert lib.tao_embed_gradient(16, 8, 100, 16, 64, 10, 64, 0, 1.0, None, 16, size, None) == ARG
