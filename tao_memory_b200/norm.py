"""Root-mean-square norm with the residual's addition: what stands between two halves of
a decoder block.  ``add_rms_norm`` (16 or 32 bits, differentiable) and
``add_rms_norm_fp8`` (e4m3 with scales, for the products that take 8-bit activations).

One library kernel forward; the gradient is one kernel and, for the weight, a second one
that adds the blocks' parts in a fixed order.
"""

import torch
from torch.autograd import forward_ad

from . import _lib

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
# F.rms_norm's default eps: the epsilon of its fp32 compute type (also for 16-bit inputs)
RMS_EPS = float(torch.finfo(torch.float32).eps)


def _rows(t, width):
    """``t`` as rows [n, width] with a contiguous last axis; copied only where its strides ask for it."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    return t if t.stride(1) == 1 or width == 1 else t.contiguous()


def wants_gradient(*operands):
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                return True
    return False


def refuse_tangents(operator, *operands):
    """Forward-mode derivatives would be dropped with the operands' addresses."""
    if forward_ad._current_level < 0:  # none is being taken
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in operands):
        raise ValueError(f"{operator} has no forward-mode derivative")


def refuse_derivatives(operator, *operands):
    """For an operator without a gradient."""
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                raise ValueError(f"{operator} has no gradient, for activations or weights: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        refuse_tangents(operator, *operands)


def _check(x, weight, residual):
    if x.dtype not in TYPES or not x.is_cuda:
        raise ValueError("the norm takes a bf16, fp16 or fp32 CUDA tensor (no CPU fallback)")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("the norm needs a last axis to sum over")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.device != x.device):
        raise ValueError("the residual must have x's shape, type and device")
    if weight is not None and (weight.shape != x.shape[-1:] or weight.dtype != x.dtype or weight.device != x.device):
        raise ValueError("the weight must be one value per channel, of x's type and device")


def _new(x, dtype=None):
    if dtype is None and x.is_contiguous():
        return torch.empty_like(x)
    return torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)


def _forward(x, weight, residual, eps):
    width = x.shape[-1]
    rows = _rows(x, width)
    y = _new(x)
    res, stride, s = None, 0, x
    if residual is not None:
        residual = _rows(residual, width)
        res, stride, s = residual.data_ptr(), residual.stride(0), _new(x)
    if weight is not None:
        weight = weight.contiguous()
    _lib.on_device(x.device.index, _lib.lib().tao_add_rms_norm, rows.data_ptr(), rows.stride(0), res, stride,
                   None if weight is None else weight.data_ptr(), rows.shape[0], width, TYPES[x.dtype], eps,
                   None if res is None else s.data_ptr(), y.data_ptr())
    return y, s


class _Room:
    """The weight gradient's scratch: one buffer for a device and stream, whose calls run in
    order; a captured call gets one of its own."""

    cache = {}

    @classmethod
    def get(cls, device, size):
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(size, dtype=torch.uint8, device=device)
        key = (device.index, torch._C._cuda_getCurrentRawStream(device.index))
        buf = cls.cache.get(key)
        if buf is None or buf.numel() < size:
            buf = cls.cache[key] = torch.empty(max(size, 1 << 20), dtype=torch.uint8, device=device)
        return buf


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, s = _forward(x, weight, residual, eps)
        ctx.save_for_backward(s, weight)
        ctx.added = residual is not None
        ctx.fixed = x.shape[-1], TYPES[x.dtype], eps, x.device
        ctx.set_materialize_grads(False)
        return (y, s) if ctx.added else y

    @staticmethod
    def backward(ctx, dy, ds=None):
        if torch.is_grad_enabled():
            raise RuntimeError("add_rms_norm is differentiable once (its gradient has none)")
        s, weight = ctx.saved_tensors
        if dy is None:  # only the stream was used
            return ds, None, ds if ctx.added else None, None
        width, code, eps, device = ctx.fixed
        lib = _lib.lib()
        rows, dy = _rows(s, width), _rows(dy, width)
        count = rows.shape[0]
        dx = _new(s)
        ds_at = w_at = dw = dw_at = ws_at = None
        ds_stride = size = 0
        if ds is not None:
            ds = _rows(ds, width)
            ds_at, ds_stride = ds.data_ptr(), ds.stride(0)
        if weight is not None:
            weight = weight.contiguous()
            w_at = weight.data_ptr()
            if ctx.needs_input_grad[1]:
                dw = torch.empty_like(weight)
                size = lib.tao_add_rms_norm_workspace_bytes(count, width, code)
                room = _Room.get(device, size)  # held until the launch
                dw_at, ws_at = dw.data_ptr(), room.data_ptr()
        _lib.on_device(device.index, lib.tao_add_rms_norm_backward, dy.data_ptr(), dy.stride(0), ds_at, ds_stride,
                       rows.data_ptr(), rows.stride(0), w_at, count, width, code, eps, dx.data_ptr(), dw_at, ws_at,
                       size)
        return dx, dw, dx if ctx.added else None, None


def add_rms_norm(x, weight=None, residual=None, eps=RMS_EPS):
    """(y, s): s = x + residual rounded to x's type (the stream the next block adds to; x
    itself without a residual) and y = s * rsqrt(mean(s^2) + eps) * weight over the last axis,
    in fp32, rounded once.  x, residual [..., width] bf16, fp16 or fp32; weight [width] of the
    same type or None (ones).  Differentiable (in reverse mode) in x, residual and weight."""
    _check(x, weight, residual)
    refuse_tangents("add_rms_norm", x, weight, residual)
    if wants_gradient(x, weight, residual):
        if residual is None:
            return _AddNorm.apply(x, weight, None, eps), x
        return _AddNorm.apply(x, weight, residual, eps)
    return _forward(x, weight, residual, eps)


def add_rms_norm_fp8(x, weight=None, residual=None, eps=RMS_EPS, group=None):
    """(q, scale, s): ``add_rms_norm`` with y in e4m3, y = q * scale: one fp32 scale a row
    (``group=None``: scale [..., 1], as ``linear4`` and row-scaled products take it) or one for
    128 channels (``group=128``: [..., ceil(width / 128)]).  Not differentiable."""
    _check(x, weight, residual)
    refuse_derivatives("add_rms_norm_fp8", x, weight, residual)
    if group not in (None, 128):
        raise ValueError("8-bit scales are by row (None) or by 128 channels")
    width = x.shape[-1]
    rows = _rows(x, width)
    q = _new(x, torch.float8_e4m3fn)
    scale = x.new_empty((*x.shape[:-1], 1 if group is None else -(-width // 128)), dtype=torch.float32)
    res, stride, s = None, 0, x
    if residual is not None:
        residual = _rows(residual, width)
        res, stride, s = residual.data_ptr(), residual.stride(0), _new(x)
    if weight is not None:
        weight = weight.contiguous()
    _lib.on_device(x.device.index, _lib.lib().tao_add_rms_norm_fp8, rows.data_ptr(), rows.stride(0), res, stride,
                   None if weight is None else weight.data_ptr(), rows.shape[0], width, TYPES[x.dtype], eps,
                   group or 0, None if res is None else s.data_ptr(), q.data_ptr(), scale.data_ptr())
    return q, scale, s


__all__ = ["add_rms_norm", "add_rms_norm_fp8", "RMS_EPS"]
