"""What the trained block's operators refuse, checked before any launch (no GPU needed)."""

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


def _described(**kw):
    a = dict(x=256, w=256, x_row=64, x_col=1, w_row=64, w_col=1, rows=4, n=32, k=64, experts=1, y=256)
    a.update(kw)
    return _lib.TaoLinear(**a)


EXPERTS = dict(offsets=16, experts=2, w_expert=2048)


def test_linear_refusals():
    lib = _lib.lib()
    for bad in (dict(type=2), dict(activation=5), dict(activation=-1), dict(rows=-1), dict(n=0), dict(k=0), dict(x=None),
                dict(w=None), dict(y=None), dict(x=17), dict(w=19), dict(y=17), dict(bias=17), dict(residual=17, r_row=32),
                dict(experts=2), dict(experts=0), dict(offsets=16, experts=513), dict(EXPERTS, offsets=18),
                dict(up=256, up_row=64, up_col=1), dict(EXPERTS, bias=16), dict(EXPERTS, residual=16, r_row=32),
                dict(EXPERTS, up=256, up_row=64, up_col=1, up_expert=2048, z=16, z_row=32), dict(rows=(1 << 30) + 1),
                dict(n=(1 << 24) + 1), dict(k=(1 << 24) + 1),
                # what has to be copied first has no room, too little, or one off its alignment
                dict(x_row=63), dict(x_col=2), dict(w=24), dict(x_row=0), dict(x_row=63, workspace=256, workspace_bytes=256),
                dict(x_row=63, workspace=128, workspace_bytes=1 << 20), dict(EXPERTS, w_expert=2047),
                dict(EXPERTS, w_expert=0)):
        assert lib.tao_linear(_described(**bad), None) == ARG, bad
    assert lib.tao_linear(_described(rows=0), None) == _lib.TAO_OK
    assert lib.tao_linear(None, None) == ARG


def test_linear_workspace():
    size = lambda gradient, **kw: _lib.lib().tao_linear_workspace_bytes(_described(**kw), gradient)
    assert size(0) == 0 and size(0, rows=0, x_row=63) == 0 and size(0, type=7) == 0
    assert size(0, x_row=63) == 512 and size(0, x=258, rows=1) == 256 and size(0, rows=1, x_row=63) == 0
    assert size(0, w_row=1, w_col=64) == 4096 and size(0, **dict(EXPERTS, w_expert=0)) == 8192
    grad = dict(dy=256, dy_row=32, dx=256, dw=256)
    assert size(1, **grad) == 0 and size(1, **dict(grad, dy_row=33)) == 256
    assert size(1, activation=2, z=256, z_row=32, **grad) == 256 and size(1, db=256, **grad) == 256
    assert size(1, db=256, activation=2, z=256, z_row=32, **dict(grad, dx=None, dw=None)) == 256
    gated = dict(EXPERTS, up=256, up_row=64, up_col=1, up_expert=2048, u=256, z=256, z_row=32, dup=256)
    assert size(1, **grad, **gated) == 512


def test_gradient_refusals():
    lib = _lib.lib()
    grad = dict(dy=256, dy_row=32, dx=256, dw=256)
    for bad in (dict(dy=None), dict(dy=17), dict(dx=17), dict(dw=17), dict(db=17), dict(x=None), dict(w=None), dict(dup=256),
                dict(activation=2), dict(activation=2, z=256, z_row=32), dict(db=256), dict(dy_row=33),
                dict(EXPERTS, up=256, up_row=64, up_col=1, up_expert=2048, z=256, u=256, z_row=32),
                dict(EXPERTS, up=256, up_row=64, up_col=1, up_expert=2048, z=256, z_row=32, dup=256)):
        assert lib.tao_linear_gradient(_described(**dict(grad, **bad)), None) == ARG, bad
    assert lib.tao_linear_gradient(_described(rows=0), None) == _lib.TAO_OK


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
