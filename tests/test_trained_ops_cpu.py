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


# addresses a megabyte apart, none of which is read before a refusal
X, W, UP, Y, Z, U, LOW, DY, DX, DW, DUP, DB, ROOM = (i << 20 for i in range(1, 14))


def _described(**kw):
    a = dict(x=X, w=W, x_row=64, x_col=1, w_row=64, w_col=1, rows=4, n=32, k=64, experts=1, y=Y)
    a.update(kw)
    return _lib.TaoLinear(**a)


EXPERTS = dict(offsets=16, experts=2, w_expert=2048)
GATED = dict(EXPERTS, up=UP, up_row=64, up_col=1, up_expert=2048)


def test_linear_refusals():
    lib = _lib.lib()
    for bad in (dict(type=2), dict(activation=5), dict(activation=-1), dict(rows=-1), dict(n=0), dict(k=0), dict(x=None),
                dict(w=None), dict(y=None), dict(x=X + 1), dict(w=W + 3), dict(y=Y + 1), dict(bias=17),
                dict(residual=17, r_row=32), dict(experts=2), dict(experts=0), dict(offsets=16, experts=513),
                dict(EXPERTS, offsets=18), dict(up=UP, up_row=64, up_col=1), dict(EXPERTS, bias=16),
                dict(EXPERTS, residual=16, r_row=32), dict(GATED, z=Z, z_row=32), dict(GATED, z=Z, u=U, z_row=32),
                dict(GATED, z=Z, u=U, low=LOW, z_row=40), dict(GATED, z=Z + 8, u=U, low=LOW, z_row=32),
                dict(GATED, z=Z, u=U, low=LOW + 8, z_row=32), dict(GATED, z=Z, u=U, low=U + 128, z_row=32),
                dict(rows=(1 << 30) + 1),
                dict(n=(1 << 24) + 1), dict(k=(1 << 24) + 1),
                # what has to be copied first has no room, too little, or one off its alignment
                dict(x_row=63), dict(x_col=2), dict(w=W + 8), dict(x_row=0), dict(x_row=63, workspace=ROOM, workspace_bytes=256),
                dict(x_row=63, workspace=ROOM + 128, workspace_bytes=1 << 20), dict(EXPERTS, w_expert=2047),
                dict(EXPERTS, w_expert=0),
                # outputs over operands: the last row of x, the bias, a residual one row on, z over y
                dict(y=X + 3 * 128), dict(y=W - 2), dict(bias=Y + 4), dict(residual=Y + 64, r_row=32),
                dict(residual=Y, r_row=40), dict(z=Y, z_row=32), dict(z=X, z_row=32), dict(GATED, z=Z, u=Z, low=LOW, z_row=32),
                dict(GATED, y=UP + 8000)):
        assert lib.tao_linear(_described(**bad), None) == ARG, bad
    assert lib.tao_linear(_described(rows=0), None) == _lib.TAO_OK
    assert lib.tao_linear(None, None) == ARG


def test_linear_workspace():
    size = lambda gradient, **kw: _lib.lib().tao_linear_workspace_bytes(_described(**kw), gradient)
    assert size(0) == 0 and size(0, rows=0, x_row=63) == 0 and size(0, type=7) == 0
    assert size(0, x_row=63) == 512 and size(0, x=X + 2, rows=1) == 256 and size(0, rows=1, x_row=63) == 0
    assert size(0, w_row=1, w_col=64) == 4096 and size(0, **dict(EXPERTS, w_expert=0)) == 8192
    grad = dict(dy=DY, dy_row=32, dx=DX, dw=DW)
    assert size(1, **grad) == 0 and size(1, **dict(grad, dy_row=33)) == 256
    assert size(1, activation=2, z=Z, z_row=32, **grad) == 256 and size(1, db=DB, **grad) == 256
    assert size(1, db=DB, activation=2, z=Z, z_row=32, **dict(grad, dx=None, dw=None)) == 256
    assert size(1, **grad, **GATED, u=U, z=Z, low=LOW, z_row=32, dup=DUP) == 512


def test_gradient_refusals():
    lib = _lib.lib()
    grad = dict(dy=DY, dy_row=32, dx=DX, dw=DW)
    for bad in (dict(dy=None), dict(dy=DY + 1), dict(dx=DX + 1), dict(dw=DW + 1), dict(db=DB + 1), dict(x=None), dict(w=None),
                dict(dup=DUP), dict(activation=2), dict(activation=2, z=Z, z_row=32), dict(db=DB), dict(dy_row=33),
                dict(GATED, z=Z, u=U, low=LOW, z_row=32), dict(GATED, z=Z, z_row=32, dup=DUP),
                dict(GATED, z=Z, u=U, z_row=32, dup=DUP, workspace=ROOM, workspace_bytes=1 << 20), dict(dx=X), dict(dx=DY), dict(dw=W + 64),
                dict(dw=DX), dict(db=DY, workspace=ROOM, workspace_bytes=1 << 20),
                dict(GATED, z=Z, u=U, low=LOW, z_row=32, dup=DW, workspace=ROOM, workspace_bytes=1 << 20)):
        assert lib.tao_linear_gradient(_described(**dict(grad, **bad)), None) == ARG, bad
    assert lib.tao_linear_gradient(_described(rows=0), None) == _lib.TAO_OK


def test_token_refusals():
    lib = _lib.lib()
    sort = lambda **kw: lib.tao_sort_tokens(*dict(dict(ids=X, id_bytes=8, pairs=8, experts=4, sorted=Y, places=Z, offsets=U,
                                                       ws=None, size=0, stream=None), **kw).values())
    for bad in (dict(id_bytes=2), dict(experts=0), dict(experts=513), dict(pairs=-1), dict(pairs=(1 << 30) + 1), dict(ids=X + 4),
                dict(offsets=None), dict(ids=None), dict(sorted=None), dict(places=None), dict(places=Z + 2),
                dict(pairs=100000), dict(pairs=100000, ws=ROOM, size=8), dict(sorted=X + 32), dict(places=Y + 28),
                dict(offsets=Z), dict(offsets=X - 16)):
        assert sort(**bad) == ARG, bad
    assert lib.tao_sort_tokens_workspace_bytes(4096, 4) == 0 and lib.tao_sort_tokens_workspace_bytes(100000, 4) > 0
    gather = lambda **kw: lib.tao_gather_tokens(*dict(dict(x=X, stride=64, places=Z, tokens=4, k=2, width=64, type=0, xs=Y,
                                                           stream=None), **kw).values())
    for bad in (dict(type=3), dict(x=X + 1), dict(k=0), dict(width=0), dict(width=(1 << 20) + 1), dict(tokens=1 << 30),
                dict(x=None), dict(places=None), dict(xs=None), dict(xs=X), dict(xs=X + 511), dict(xs=Z)):
        assert gather(**bad) == ARG, bad
    assert gather(tokens=0) == _lib.TAO_OK
    back = lambda **kw: lib.tao_return_tokens(*dict(dict(ys=X, stride=64, places=Z, kept=None, w=U, wtype=2, tokens=4, k=2, width=64,
                                                         type=0, y=Y, stream=None), **kw).values())
    for bad in (dict(wtype=1), dict(places=None), dict(ys=None), dict(y=X + 1000), dict(y=U), dict(kept=Y), dict(w=U + 2)):
        assert back(**bad) == ARG, bad
    grad = lambda **kw: lib.tao_return_tokens_gradient(
        *dict(dict(dy=DY, stride=64, ys=X, ystride=64, places=Z, kept=None, w=U, wtype=2, tokens=4, k=2, width=64, type=0, dys=Y,
                   dw=DW, stream=None), **kw).values())
    for bad in (dict(ys=None), dict(w=None), dict(dys=None, dw=None), dict(dys=X), dict(dys=DY + 100), dict(dw=U), dict(dw=Y),
                dict(wtype=1), dict(dw=DW + 2)):
        assert grad(**bad) == ARG, bad


def test_embedding_refusals():
    lib = _lib.lib()
    embed_ = lambda **kw: lib.tao_embed(*dict(dict(ids=X, id_bytes=8, n=4, table=W, stride=64, vocab=10, width=64, type=0, scale=1.0,
                                                   y=Y, stream=None), **kw).values())
    for bad in (dict(id_bytes=3), dict(vocab=0), dict(vocab=(1 << 26) + 1), dict(type=3), dict(ids=X + 4), dict(table=None),
                dict(y=None), dict(width=(1 << 20) + 1), dict(n=-1), dict(y=W + 100), dict(y=X)):
        assert embed_(**bad) == ARG, bad
    assert embed_(n=0) == _lib.TAO_OK
    size = lib.tao_embed_gradient_workspace_bytes(100, 10, 64)
    assert size > 0 and lib.tao_embed_gradient_workspace_bytes(0, 10, 64) == 0
    grad = lambda **kw: lib.tao_embed_gradient(*dict(dict(ids=X, id_bytes=8, n=100, dy=DY, stride=64, vocab=10, width=64, type=0,
                                                          scale=1.0, out=Y, ws=ROOM, size=size, stream=None), **kw).values())
    for bad in (dict(size=size - 1), dict(ws=ROOM + 8), dict(ws=None), dict(dy=None), dict(out=None), dict(out=DY), dict(out=X),
                dict(type=3)):
        assert grad(**bad) == ARG, bad
