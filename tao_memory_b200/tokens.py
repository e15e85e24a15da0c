"""Tokens sorted by expert and back: ``sort_tokens`` makes the order from a router's choices, ``gather_tokens``
brings the tokens' rows into it, ``return_tokens`` adds the experts' rows into their tokens by weight.  Between
them stands ``expert_linear``.  All on the device, without a copy to the host; the last two are differentiable.
"""

import torch

from . import _lib
from .norm import TYPES, _rows, refuse_tangents, wants_gradient

MOST_EXPERTS, MOST_CHANNELS = 512, 1 << 20


class TokenOrder:
    """Pairs (token, choice) sorted by expert, stably; pair t * top_k + j is token t's choice j, and pairs without
    an expert come last.  ``pairs`` [tokens * top_k]: the pair at each place; ``places`` [tokens, top_k]: its
    inverse; ``offsets`` [experts + 1]: the first place of each expert, and the end of the last one's (int32)."""

    __slots__ = ("pairs", "places", "offsets")

    def __init__(self, pairs, places, offsets):
        for t in (pairs, places, offsets):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != places.device:
                raise ValueError("an order's parts are contiguous int32 tensors on one device")
        if places.dim() != 2 or places.shape[1] == 0 or pairs.shape != (places.numel(),) or offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError("an order has pairs [tokens * top_k], places [tokens, top_k] and offsets [experts + 1]")
        self.pairs, self.places, self.offsets = pairs, places, offsets

    experts = property(lambda self: self.offsets.shape[0] - 1)
    tokens = property(lambda self: self.places.shape[0])
    top_k = property(lambda self: self.places.shape[1])


def sort_tokens(ids, experts):
    """``TokenOrder`` of a router's choices ids [tokens, top_k] (int32 or int64, up to 512 experts); an id outside
    of 0 .. experts - 1 is no expert (a padded token's)."""
    if ids.dtype not in (torch.int32, torch.int64) or not ids.is_cuda or ids.dim() != 2 or ids.shape[1] == 0:
        raise ValueError("ids are an int32 or int64 CUDA tensor [tokens, top_k] (no CPU fallback)")
    if not 1 <= experts <= MOST_EXPERTS:
        raise ValueError(f"there are 1 to {MOST_EXPERTS} experts")
    ids = ids.contiguous()
    count, lib = ids.numel(), _lib.lib()
    pairs, places, offsets = (ids.new_empty(shape, dtype=torch.int32) for shape in (count, ids.shape, experts + 1))
    size = lib.tao_sort_tokens_workspace_bytes(count, experts)
    room = ids.new_empty(size, dtype=torch.uint8) if size else None
    _lib.on_device(ids.device.index, lib.tao_sort_tokens, ids.data_ptr(), ids.element_size(), count, experts,
                   pairs.data_ptr(), places.data_ptr(), offsets.data_ptr(), None if room is None else room.data_ptr(), size)
    order = TokenOrder.__new__(TokenOrder)  # what was just made need not be looked at
    order.pairs, order.places, order.offsets = pairs, places, offsets
    return order


def _check(name, rows, order, count):
    if rows.dtype not in TYPES or not rows.is_cuda or rows.dim() != 2 or rows.shape[1] == 0:
        raise ValueError(f"{name} takes bf16, fp16 or fp32 CUDA rows [rows, width] (no CPU fallback)")
    if not isinstance(order, TokenOrder) or order.places.device != rows.device:
        raise ValueError(f"{name} takes a TokenOrder on the rows' device")
    if rows.shape[1] > MOST_CHANNELS:
        raise ValueError("a row has up to 2^20 channels")
    if rows.shape[0] != count:
        raise ValueError(f"{name}: {rows.shape[0]} rows, and {count} in the order")


def _kept(offsets):
    """The address of the number of pairs that have an expert."""
    return offsets.data_ptr() + 4 * (offsets.shape[0] - 1)


def _return(ys, places, offsets, weights):
    """The sum of each token's rows; offsets None: of pairs without an expert too."""
    (tokens, top_k), width = places.shape, ys.shape[1]
    y = ys.new_empty((tokens, width))
    ys = _rows(ys, width)
    _lib.on_device(ys.device.index, _lib.lib().tao_return_tokens, ys.data_ptr(), ys.stride(0), places.data_ptr(),
                   None if offsets is None else _kept(offsets), None if weights is None else weights.data_ptr(),
                   0 if weights is None else TYPES[weights.dtype], tokens, top_k, width, TYPES[ys.dtype], y.data_ptr())
    return y


def _gather(x, places):
    (tokens, top_k), width = places.shape, x.shape[1]
    xs = x.new_empty((tokens * top_k, width))
    x = _rows(x, width)
    _lib.on_device(x.device.index, _lib.lib().tao_gather_tokens, x.data_ptr(), x.stride(0), places.data_ptr(), tokens, top_k,
                   width, TYPES[x.dtype], xs.data_ptr())
    return xs


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, places):
        ctx.save_for_backward(places)
        return _gather(x, places)

    @staticmethod
    def backward(ctx, dxs):
        if torch.is_grad_enabled():
            raise RuntimeError("gather_tokens is differentiable once (its gradient has none)")
        places, = ctx.saved_tensors
        return _return(dxs, places, None, None), None


class _Return(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, weights, places, offsets):
        ctx.save_for_backward(ys if weights is not None and ctx.needs_input_grad[1] else None, weights, places, offsets)
        return _return(ys, places, offsets, weights)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("return_tokens is differentiable once (its gradient has none)")
        ys, weights, places, offsets = ctx.saved_tensors
        (tokens, top_k), width = places.shape, dy.shape[1]
        want_ys, want_w = ctx.needs_input_grad[:2]
        dys = dy.new_empty((tokens * top_k, width)) if want_ys else None
        dw = torch.empty_like(weights) if want_w else None
        dy = _rows(dy, width)
        ys = None if ys is None else _rows(ys, width)
        _lib.on_device(dy.device.index, _lib.lib().tao_return_tokens_gradient, dy.data_ptr(), dy.stride(0),
                       None if ys is None else ys.data_ptr(), 0 if ys is None else ys.stride(0), places.data_ptr(),
                       _kept(offsets), None if weights is None else weights.data_ptr(),
                       0 if weights is None else TYPES[weights.dtype], tokens, top_k, width, TYPES[dy.dtype],
                       None if dys is None else dys.data_ptr(), None if dw is None else dw.data_ptr())
        return dys, dw, None, None


def gather_tokens(x, order):
    """The rows of x [tokens, width] (bf16, fp16 or fp32) in the order's places [tokens * top_k, width].
    Differentiable (in reverse mode, once): a token's gradient is the sum of its rows'."""
    _check("gather_tokens", x, order, order.tokens if isinstance(order, TokenOrder) else 0)
    refuse_tangents("gather_tokens", x)
    return _Gather.apply(x, order.places) if wants_gradient(x) else _gather(x, order.places)


def return_tokens(ys, order, weights=None):
    """y[t] = sum over token t's choices j that have an expert of weights[t, j] ys[places[t, j]], in fp32 in the
    order of the choices, rounded once: ys [tokens * top_k, width] bf16, fp16 or fp32, weights [tokens, top_k] fp32
    or of ys' type (None: ones).  Differentiable (in reverse mode, once) in ys and weights; the gradients of
    pairs without an expert are zeros."""
    _check("return_tokens", ys, order, order.tokens * order.top_k if isinstance(order, TokenOrder) else 0)
    if weights is not None:
        if weights.shape != order.places.shape or weights.dtype not in (torch.float32, ys.dtype) \
                or weights.device != ys.device:
            raise ValueError("weights are one value a choice, fp32 or of the rows' type, on their device")
    refuse_tangents("return_tokens", ys, weights)
    if weights is not None:
        weights = weights.contiguous()
    if wants_gradient(ys, weights):
        return _Return.apply(ys, weights, order.places, order.offsets)
    return _return(ys, order.places, order.offsets, weights)


__all__ = ["TokenOrder", "sort_tokens", "gather_tokens", "return_tokens"]
