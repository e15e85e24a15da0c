"""16-bit products with what stands around them in one kernel, differentiable: ``linear`` (bias, activation,
residual) and ``expert_linear`` (rows sorted by expert, each through its expert's weights, gated).

Forward one library kernel; the gradient is one for the activation's slope (where there is an activation or a
bias), one for the input and one for the weights.  Operands whose rows do not start on 16 bytes are copied to
rows that do first, by the library.
"""

from ctypes import byref

import torch

from . import _lib
from .norm import TYPES, _rows, refuse_tangents, wants_gradient

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
MOST_EXPERTS = 512


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


def _address(t):
    return None if t is None else t.data_ptr()


def _describe(rows, weight, up, bias, residual, offsets, act):
    """The library's description of a product, without its outputs."""
    n, k = weight.shape[-2:]
    grouped = offsets is not None
    w = weight.stride() if grouped else (0, *weight.stride())
    u = (0, 0, 0) if up is None else up.stride()
    x = rows.stride()
    return _lib.TaoLinear(
        rows.data_ptr(), weight.data_ptr(), _address(up), _address(bias), _address(residual), _address(offsets), x[0], x[1],
        w[0], w[1], w[2], u[0], u[1], u[2], 0 if residual is None else residual.stride(0), 0, rows.shape[0], n, k,
        weight.shape[0] if grouped else 1, TYPES[rows.dtype], act)


def _room(p, rows, gradient):
    """The workspace that ``p`` needs, held by the caller until the launch; the allocator orders its next use."""
    size = _lib.lib().tao_linear_workspace_bytes(byref(p), gradient)
    if size == 0:
        return None
    room = torch.empty(size + 256, dtype=torch.uint8, device=rows.device)
    at = room.data_ptr()
    p.workspace, p.workspace_bytes = at + -at % 256, size
    return room


def _point(p, kept, up):
    at = kept.data_ptr()
    p.z, p.z_row = at, kept.shape[-1]
    if up is not None:
        plane = 2 * kept.shape[1] * kept.shape[2]
        p.u, p.low = at + plane, at + 2 * plane


def _forward(p, rows, up, keep):
    """(y, kept) of a described product: kept is None unless ``keep``."""
    count, n = rows.shape[0], p.n
    y = rows.new_empty((count, n))
    p.y = y.data_ptr()
    kept = None
    if keep:
        row = -(-n // 16) * 16
        # act's argument, or 24 bits each of a gate's two factors: their upper 16 and behind them their lower 8
        kept = rows.new_empty((count, row) if up is None else (3, count, row))
        _point(p, kept, up)
    room = _room(p, rows, 0)
    _lib.on_device(rows.device.index, _lib.lib().tao_linear, byref(p))
    del room
    return y, kept


class _Product(torch.autograd.Function):
    """x [rows, k], residual [rows, n]; offsets None: one weight."""

    @staticmethod
    def forward(ctx, x, weight, up, bias, residual, offsets, act):
        p = _describe(x, weight, up, bias, residual, offsets, act)
        sloped = any(ctx.needs_input_grad[:4]) and (act != 0 or up is not None)
        y, kept = _forward(p, x, up, sloped)
        ctx.save_for_backward(x, weight, up, kept, offsets)
        ctx.act = act
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("linear and expert_linear are differentiable once (their gradients have none)")
        if dy is None:
            return (None,) * 7
        want_x, want_w, want_up, want_b, want_res = ctx.needs_input_grad[:5]
        dx = dw = dup = db = None
        if want_x or want_w or want_up or want_b:
            x, weight, up, kept, offsets = ctx.saved_tensors
            p = _describe(x, weight, up, None, None, offsets, ctx.act)
            grad = _rows(dy, p.n)
            p.dy, p.dy_row = grad.data_ptr(), grad.stride(0)
            if kept is not None:
                _point(p, kept, up)
            if want_x:
                dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
                p.dx = dx.data_ptr()
            if want_w or want_up:
                dw = torch.empty(weight.shape, dtype=x.dtype, device=x.device)
                p.dw = dw.data_ptr()
                if up is not None:
                    dup = torch.empty(weight.shape, dtype=x.dtype, device=x.device)
                    p.dup = dup.data_ptr()
            if want_b:
                db = torch.empty(p.n, dtype=x.dtype, device=x.device)
                p.db = db.data_ptr()
            room = _room(p, x, 1)
            _lib.on_device(x.device.index, _lib.lib().tao_linear_gradient, byref(p))
            del room
        return (dx, dw if want_w else None, dup if want_up else None, db, dy if want_res else None, None, None)


def linear(x, weight, bias=None, residual=None, activation=None):
    """act(x W^T + bias) + residual: x [..., k] and weight [n, k] bf16 or fp16, bias [n] and residual [..., n] of
    the same type; sums, activation and addition in fp32, rounded once.  ``activation``: None, "relu", "silu",
    "gelu" (by the error function) or "gelu_tanh".

    For one row to many; one row takes 1.2 to 1.5 times what the weight's bytes do, up to 64 rows 1.2 to 3 times.
    Differentiable (in reverse mode, once) in all four; the activation's argument is kept, rounded to the type, for the
    gradient (sums beyond fp16 have the slopes of very large ones), and dz = dy act'(z) is rounded to the type before the
    products that it goes into: in fp16 one beyond 65504 is infinite, as a loss scaler expects."""
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
    rows = x if x.dim() == 2 else x.reshape(-1, k)
    if bias is not None:
        bias = bias.contiguous()
    if residual is not None:
        residual = _rows(residual, n)
    act = ACTIVATIONS[activation]
    if wants_gradient(x, weight, bias, residual):
        y = _Product.apply(rows, weight, None, bias, residual, None, act)
    else:
        y, _ = _forward(_describe(rows, weight, None, bias, residual, None, act), rows, None, False)
    return y if x.dim() == 2 else y.view(shape)


def expert_linear(x, weight, offsets, up=None, activation=None):
    """Rows through their experts' weights: x [rows, k] sorted by expert, offsets [experts + 1] int32 on the
    device (``sort_tokens`` makes them; the first is 0), weight [experts, n, k]: y = act(x W_e^T), or with ``up``
    (like weight) the gated act(x W_e^T) * (x U_e^T), for the rows offsets[e] to offsets[e + 1] of each expert e.
    Rows behind the last expert's give zeros.  bf16 or fp16, sums and activation in fp32, rounded once.

    The offsets are read on the device only.  Differentiable (in reverse mode, once) in x, weight and up, as
    ``linear`` is, but that a gate's two factors are kept in 24 bits (dz = dy u act'(z) and du = dy act(z) are rounded to
    the type); an expert without rows has a gradient of zeros, rows of no expert too."""
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
    if wants_gradient(x, weight, up):
        return _Product.apply(x, weight, up, None, None, offsets, act)
    return _forward(_describe(x, weight, up, None, None, offsets, act), x, up, False)[0]


__all__ = ["linear", "expert_linear", "ACTIVATIONS"]
