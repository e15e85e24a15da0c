"""16-bit products with what stands around them in one kernel, differentiable: ``linear`` (bias, activation,
residual) and ``expert_linear`` (rows sorted by expert, each through its expert's weights, gated).

Forward one library kernel; the gradient is one for the activation's slope (where there is an activation or a
bias), one for the input and one for the weights.  Operands whose rows do not start on 16 bytes are copied to
rows that do first.
"""

import torch

from . import _lib
from .norm import TYPES, _rows, refuse_tangents, wants_gradient

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
MOST_EXPERTS = 512


def _room(like, *shape):
    """An uninitialised [..., width] whose rows start on 16 bytes."""
    width = shape[-1]
    return like.new_empty((*shape[:-1], -(-width // 8) * 8))[..., :width]


def _laid(t):
    """``t`` [..., rows, width] as the products fetch it: neighbours next to each other, everything else on 16 bytes."""
    width = t.shape[-1]
    if (t.stride(-1) == 1 or width == 1) and t.data_ptr() % 16 == 0:
        least = width  # rows do not overlap, nor do matrices
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size > 1 and (stride % 8 or stride < least):
                break
            least = max(least, stride * size)
        else:
            return t
    return _room(t, *t.shape).copy_(t)


def _check(name, x, weight, activation):
    if x.dtype not in (torch.bfloat16, torch.float16) or not x.is_cuda:
        raise ValueError(f"{name} takes bf16 or fp16 CUDA activations (no CPU fallback)")
    if weight.dtype != x.dtype or weight.device != x.device:
        raise ValueError("the weight has the activations' type and device")
    if 0 in weight.shape[-2:]:
        raise ValueError("the weight has at least one output and one input channel")
    if x.dim() == 0 or x.shape[-1] != weight.shape[-1]:
        raise ValueError(f"activations have {weight.shape[-1]} channels, as the weight")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation is one of {tuple(ACTIVATIONS)}")


def _forward(rows, weight, up, bias, residual, offsets, act, keep):
    """(y, z, u) of laid-out operands: z, u are None unless ``keep``."""
    count, n, k = rows.shape[0], weight.shape[-2], weight.shape[-1]
    y = rows.new_empty((count, n))
    z = u = None
    if keep:
        z = _room(rows, count, n)
        u = None if up is None else _room(rows, count, n)
    grouped = offsets is not None
    _lib.on_device(
        rows.device.index, _lib.lib().tao_linear, rows.data_ptr(), rows.stride(0), weight.data_ptr(), weight.stride(-2),
        weight.stride(0) if grouped else 0, None if up is None else up.data_ptr(), 0 if up is None else up.stride(-2),
        0 if up is None else up.stride(0), None if bias is None else bias.data_ptr(),
        None if residual is None else residual.data_ptr(), 0 if residual is None else residual.stride(0),
        offsets.data_ptr() if grouped else None, weight.shape[0] if grouped else 1, count, n, k, TYPES[rows.dtype], act,
        y.data_ptr(), None if z is None else z.data_ptr(), None if u is None else u.data_ptr(),
        0 if z is None else z.stride(0))
    return y, z, u


def _slope(dy, z, u, act, db):
    """(dz, du) of dy [rows, n], and the rows' sum into ``db``."""
    count, n = dy.shape
    lib = _lib.lib()
    dz = None if z is None else _room(dy, count, n)
    du = None if u is None else _room(dy, count, n)
    room = None
    if db is not None:
        room = dy.new_empty(lib.tao_linear_slope_workspace_bytes(count, n), dtype=torch.uint8)
    _lib.on_device(
        dy.device.index, lib.tao_linear_slope, dy.data_ptr(), dy.stride(0), None if z is None else z.data_ptr(),
        None if u is None else u.data_ptr(), 0 if z is None else z.stride(0), count, n, TYPES[dy.dtype], act,
        None if dz is None else dz.data_ptr(), None if du is None else du.data_ptr(), 0 if dz is None else dz.stride(0),
        None if db is None else db.data_ptr(), None if room is None else room.data_ptr(), 0 if room is None else room.numel())
    return dy if dz is None else dz, du


class _Product(torch.autograd.Function):
    """x [rows, k], residual [rows, n]; offsets None: one weight."""

    @staticmethod
    def forward(ctx, x, weight, up, bias, residual, offsets, act):
        rows, w = _laid(x), _laid(weight)
        u_w = None if up is None else _laid(up)
        sloped = any(ctx.needs_input_grad[:4]) and (act != 0 or up is not None)
        y, z, u = _forward(rows, w, u_w, bias, residual, offsets, act, sloped)
        ctx.save_for_backward(rows, w, u_w, z, u, offsets)
        ctx.act = act
        ctx.has_bias = bias is not None
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("linear and expert_linear are differentiable once (their gradients have none)")
        if dy is None:
            return (None,) * 7
        rows, weight, up, z, u, offsets = ctx.saved_tensors
        want_x, want_w, want_up, want_b, want_res = ctx.needs_input_grad[:5]
        dx = dw = dup = db = None
        if want_x or want_w or want_up or want_b:
            (count, k), n = rows.shape, weight.shape[-2]
            lib, device, code = _lib.lib(), rows.device.index, TYPES[rows.dtype]
            grad = _rows(dy, n)
            du = None
            if want_b:
                db = dy.new_empty(n)
            if z is not None or want_b:
                dz, du = _slope(grad, z, u, ctx.act, db)
            else:
                dz = grad
            grouped = offsets is not None
            at, experts = (offsets.data_ptr(), weight.shape[0]) if grouped else (None, 1)
            if want_x or want_w or want_up:
                dz = _laid(dz)
                du_at = None if du is None else du.data_ptr()
            if want_x:
                dx = rows.new_empty((count, k))
                _lib.on_device(
                    device, lib.tao_linear_input_gradient, dz.data_ptr(), du_at, dz.stride(0), weight.data_ptr(),
                    weight.stride(-2), weight.stride(0) if grouped else 0, None if up is None else up.data_ptr(),
                    0 if up is None else up.stride(-2), 0 if up is None else up.stride(0), at, experts, count, n, k, code,
                    dx.data_ptr())
            if want_w or want_up:
                dw = weight.new_empty(weight.shape)
                dup = None if up is None else weight.new_empty(weight.shape)
                _lib.on_device(
                    device, lib.tao_linear_weight_gradient, dz.data_ptr(), du_at, dz.stride(0), rows.data_ptr(),
                    rows.stride(0), at, experts, count, n, k, code, dw.data_ptr(), None if dup is None else dup.data_ptr())
        return (dx, dw if want_w else None, dup if want_up else None, db, dy if want_res else None, None, None)


def linear(x, weight, bias=None, residual=None, activation=None):
    """act(x W^T + bias) + residual: x [..., k] and weight [n, k] bf16 or fp16, bias [n] and residual [..., n] of
    the same type; sums, activation and addition in fp32, rounded once.  ``activation``: None, "relu", "silu",
    "gelu" (by the error function) or "gelu_tanh".

    For one row to many; up to 64 rows take time for the weight's bytes.  Differentiable (in reverse mode, once)
    in all four; the activation's argument is kept, rounded to the type, for the gradient, and dz = dy act'(z) is
    rounded to it before the products that it goes into."""
    if weight.dim() != 2:
        raise ValueError("linear takes one weight matrix [n, k]")
    _check("linear", x, weight, activation)
    n, k = weight.shape
    shape = (*x.shape[:-1], n)
    if bias is not None and (bias.shape != (n,) or bias.dtype != x.dtype or bias.device != x.device):
        raise ValueError("the bias is one value per output, of the activations' type and device")
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("the residual has the output's shape and the activations' type and device")
    refuse_tangents("linear", x, weight, bias, residual)
    rows = _rows(x, k)
    if bias is not None:
        bias = bias.contiguous()
    if residual is not None:
        residual = _rows(residual, n)
    act = ACTIVATIONS[activation]
    if wants_gradient(x, weight, bias, residual):
        y = _Product.apply(rows, weight, None, bias, residual, None, act)
    else:
        y, _, _ = _forward(_laid(rows), _laid(weight), None, bias, residual, None, act, False)
    return y if x.dim() == 2 else y.view(shape)


def expert_linear(x, weight, offsets, up=None, activation=None):
    """Rows through their experts' weights: x [rows, k] sorted by expert, offsets [experts + 1] int32 on the
    device (``sort_tokens`` makes them; the first is 0), weight [experts, n, k]: y = act(x W_e^T), or with ``up``
    (like weight) the gated act(x W_e^T) * (x U_e^T), for the rows offsets[e] to offsets[e + 1] of each expert e.
    Rows behind the last expert's give zeros.  bf16 or fp16, sums and activation in fp32, rounded once.

    The offsets are read on the device only.  Differentiable (in reverse mode, once) in x, weight and up, as
    ``linear`` is; an expert without rows has a gradient of zeros, rows of no expert too."""
    if weight.dim() != 3:
        raise ValueError("expert_linear takes weights [experts, n, k]")
    _check("expert_linear", x, weight, activation)
    if x.dim() != 2:
        raise ValueError("expert_linear takes rows [rows, k] sorted by expert")
    experts = weight.shape[0]
    if not 1 <= experts <= MOST_EXPERTS:
        raise ValueError(f"there are 1 to {MOST_EXPERTS} experts")
    if up is not None and (up.shape != weight.shape or up.dtype != weight.dtype or up.device != weight.device):
        raise ValueError("up has the weight's shape, type and device")
    if offsets.shape != (experts + 1,) or offsets.dtype != torch.int32 or offsets.device != x.device:
        raise ValueError("offsets are experts + 1 int32 values on the activations' device")
    refuse_tangents("expert_linear", x, weight, up)
    offsets = offsets.contiguous()
    act = ACTIVATIONS[activation]
    rows = _rows(x, x.shape[1])
    if wants_gradient(x, weight, up):
        return _Product.apply(rows, weight, up, None, None, offsets, act)
    return _forward(_laid(rows), _laid(weight), None if up is None else _laid(up), None, None, offsets, act, False)[0]


__all__ = ["linear", "expert_linear", "ACTIVATIONS"]
