"""Rows of a table by tokens' ids, scaled (``embed``), and the table's gradient, whose sums have a fixed order."""

import torch

from . import _lib
from .norm import TYPES, _rows, refuse_tangents, wants_gradient

MOST_ROWS, MOST_CHANNELS = 1 << 26, 1 << 20


def _forward(ids, table, scale):
    vocab, width = table.shape
    y = table.new_empty((*ids.shape, width))
    ids, table = ids.contiguous(), _rows(table, width)
    _lib.on_device(table.device.index, _lib.lib().tao_embed, ids.data_ptr(), ids.element_size(), ids.numel(),
                   table.data_ptr(), table.stride(0), vocab, width, TYPES[table.dtype], scale, y.data_ptr())
    return y


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.fixed = table.shape, scale
        return _forward(ids, table, scale)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("embed is differentiable once (its gradient has none)")
        ids, = ctx.saved_tensors
        (vocab, width), scale = ctx.fixed
        lib, ids = _lib.lib(), ids.contiguous()
        rows = _rows(dy, width)
        out = dy.new_empty((vocab, width))
        size = lib.tao_embed_gradient_workspace_bytes(ids.numel(), vocab, width)
        room = dy.new_empty(size, dtype=torch.uint8)
        _lib.on_device(dy.device.index, lib.tao_embed_gradient, ids.data_ptr(), ids.element_size(), ids.numel(),
                       rows.data_ptr(), rows.stride(0), vocab, width, TYPES[dy.dtype], scale, out.data_ptr(),
                       room.data_ptr(), size)
        return out, None, None


def embed(ids, table, scale=1.0):
    """scale * table[ids]: table [vocab, width] bf16, fp16 or fp32, ids int32 or int64 of any shape on its device;
    returns [*ids.shape, width], scaled in fp32 and rounded once.  An id outside of the table (padding) gives
    zeros and adds to no gradient.  Differentiable (in reverse mode, once) in the table: a dense gradient, each
    row's sum in fp32 in the order of the tokens, in runs of 16 of the sorted tokens, rounded once."""
    if table.dtype not in TYPES or not table.is_cuda or table.dim() != 2 or 0 in table.shape:
        raise ValueError("embed takes a bf16, fp16 or fp32 CUDA table [vocab, width] (no CPU fallback)")
    if table.shape[0] > MOST_ROWS or table.shape[1] > MOST_CHANNELS:
        raise ValueError("a table has up to 2^26 rows of up to 2^20 channels")
    if ids.dtype not in (torch.int32, torch.int64) or ids.device != table.device:
        raise ValueError("ids are an int32 or int64 tensor on the table's device")
    scale = float(scale)
    refuse_tangents("embed", table)
    return _Embed.apply(table, ids, scale) if wants_gradient(table) else _forward(ids, table, scale)


__all__ = ["embed"]
