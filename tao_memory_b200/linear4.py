"""Products of a few rows with 4-bit weights: the projections of a decode step, whose time
is the time to read their weights.

``quantize4`` makes a ``Weight4`` from a weight matrix, ``Weight4.from_codes`` from codes,
scales and zero points quantised elsewhere; ``linear4`` is the product.  A ``Weight4`` holds
the codes in the order in which the kernel's warps read them (laid out once, here).
"""

import torch

from . import _lib
from .norm import TYPES, _rows, refuse_derivatives

GROUPS = (32, 64, 128)
E4M3 = 3  # the library's code of the type, beside TYPES
_TILE, _BLOCK = 16, 128


def _padded(t, n, k, value=0):
    """``t`` [.., a, b] with its last axes filled up to n and k."""
    if t.shape[-2:] == (n, k):
        return t
    return torch.nn.functional.pad(t, (0, k - t.shape[-1], 0, n - t.shape[-2]), value=value)


class Weight4:
    """4-bit weights [..., n, k]: W = (code - zero) * scale with one scale, and optionally one
    zero point, for ``group`` consecutive k of a row.  Leading axes are matrices of a stack
    (one for each expert).  May be copied, saved and loaded; its tensors cannot be exchanged."""

    def __init__(self, shape, group, codes, scales, zeros):
        self.shape, self.group = tuple(shape), group
        self._tensors = codes, scales, zeros

    codes = property(lambda self: self._tensors[0])
    scales = property(lambda self: self._tensors[1])
    zeros = property(lambda self: self._tensors[2])
    dtype = property(lambda self: self._tensors[1].dtype)
    device = property(lambda self: self._tensors[0].device)

    @property
    def args(self):
        """What tao_linear4 takes of it: of the tensors as they are now, not as they were before a copy or a file."""
        codes, scales, zeros = self._tensors
        return (codes.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), self.group,
                TYPES[scales.dtype])

    def bytes(self):
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.zeros) if t is not None)

    @classmethod
    def from_codes(cls, codes, scales, zeros=None, group=128):
        """codes uint8 [..., n, k] of 0..15, scales [..., n, ceil(k / group)] bf16 or fp16, zeros
        uint8 like scales of 0..15 (None: 8 everywhere)."""
        if group not in GROUPS:
            raise ValueError("a group is 32, 64 or 128 weights")
        if codes.dtype != torch.uint8 or codes.dim() < 2 or 0 in codes.shape:
            raise ValueError("codes are a uint8 tensor [..., n, k]")
        *lead, n, k = codes.shape
        parts = -(-k // group)
        if scales.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("4-bit scales are bf16 or fp16")
        if zeros is not None and zeros.dtype != torch.uint8:
            raise ValueError("zero points are uint8")
        for t in (scales,) if zeros is None else (scales, zeros):
            if tuple(t.shape) != (*lead, n, parts) or t.device != codes.device:
                raise ValueError("scales and zeros have one value for each group of a row, on the codes' device")
        if int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 15):
            raise ValueError("codes and zero points are 0..15")
        tiles, blocks, per = -(-n // _TILE), -(-k // _BLOCK), _BLOCK // group
        count = codes[..., 0, 0].numel()
        laid = torch.empty(count, tiles, blocks, 1024, dtype=torch.uint8, device=codes.device)
        flat = codes.reshape(count, n, k)
        most = max(1, (1 << 25) // (tiles * blocks * _TILE * _BLOCK))
        for i in range(0, count, most):  # a few matrices at a time: the intermediate orders stay small
            c = _padded(flat[i:i + most], tiles * _TILE, blocks * _BLOCK)
            # n = (tile, row half, g), k = (block, half, i, t, f, e high, e low)
            c = c.view(-1, tiles, 2, 8, blocks, 2, 2, 4, 2, 2, 2)
            # -> tile, block, half, g, t, i, f, e low, e high, then the byte's nibbles: rows g, g + 8
            c = c.permute(0, 1, 4, 5, 3, 7, 6, 8, 10, 9, 2).reshape(-1, tiles, blocks, 1024, 2)
            torch.bitwise_or(c[..., 0], c[..., 1] << 4, out=laid[i:i + most])

        def by_tile(t):
            t = _padded(t.reshape(count, n, parts), tiles * _TILE, blocks * per)
            # a lane's rows g and g + 8 next to each other, the groups of a block within them
            return t.view(count, tiles, 2, 8, blocks, per).permute(0, 1, 4, 3, 5, 2).contiguous()

        return cls(codes.shape, group, laid, by_tile(scales), None if zeros is None else by_tile(zeros))

    def to_codes(self):
        """(codes, scales, zeros) as ``from_codes`` takes them."""
        *lead, n, k = self.shape
        count, tiles, blocks, _ = self.codes.shape
        c = torch.stack((self.codes & 15, self.codes >> 4), -1).view(count, tiles, blocks, 2, 8, 4, 2, 2, 2, 2, 2)
        c = c.permute(0, 1, 10, 4, 2, 3, 6, 5, 7, 9, 8).reshape(count, tiles * _TILE, blocks * _BLOCK)

        def rows(t):
            t = t.permute(0, 1, 5, 3, 2, 4).reshape(count, tiles * _TILE, -1)
            return t[:, :n, :-(-k // self.group)].reshape(*lead, n, -1)

        return (c[:, :n, :k].reshape(*lead, n, k), rows(self.scales),
                None if self.zeros is None else rows(self.zeros))

    def dequantize(self):
        """The weights in fp32 [..., n, k]."""
        codes, scales, zeros = self.to_codes()
        wide = lambda t: t.float().repeat_interleave(self.group, -1)[..., :codes.shape[-1]]
        return (codes.float() - (8 if zeros is None else wide(zeros))) * wide(scales)


def quantize4(weight, group=128, zeros=False):
    """``Weight4`` of ``weight`` [..., n, k] (bf16 or fp16, or fp32 with bf16 scales), each group
    rounded to the nearest of 16 evenly spaced values: from -8 to 7 scales around zero, or
    (``zeros=True``) over the group's range, which zero is always part of."""
    if group not in GROUPS:
        raise ValueError("a group is 32, 64 or 128 weights")
    if weight.dtype not in TYPES or weight.dim() < 2:
        raise ValueError("quantize4 takes a bf16, fp16 or fp32 weight [..., n, k]")
    dtype = torch.bfloat16 if weight.dtype == torch.float32 else weight.dtype
    *lead, n, k = weight.shape
    parts = -(-k // group)
    w = _padded(weight.detach().float(), n, parts * group).view(*lead, n, parts, group)
    if zeros:
        low, high = w.amin(-1).clamp_max(0), w.amax(-1).clamp_min(0)
        scales = ((high - low) / 15).to(dtype)
    else:
        scales = torch.maximum(w.amax(-1) / 7, -w.amin(-1) / 8).to(dtype)
    step = scales.float()
    # steps whose reciprocal would be infinite are taken 2^64 times as large, the weights with them
    grow = torch.where(step < 2.0 ** -100, 2.0 ** 64, 1.0)
    step, w = step * grow, w * grow.unsqueeze(-1)
    up = torch.where(step > 0, 1 / step, torch.zeros_like(step)).unsqueeze(-1)
    if zeros:
        zero = (-low * grow * up.squeeze(-1)).round().clamp(0, 15)
        codes = ((w * up).round() + zero.unsqueeze(-1)).clamp(0, 15)
    else:
        zero, codes = None, ((w * up).round() + 8).clamp(0, 15)
    return Weight4.from_codes(codes.to(torch.uint8).view(*lead, n, parts * group)[..., :k], scales,
                              None if zero is None else zero.to(torch.uint8), group)


def linear4(x, weight, bias=None, x_scale=None, out=None):
    """x W^T + bias: x [..., k] in the weight's type, or in e4m3 with one fp32 scale a row
    (``x_scale`` [..., 1], as ``add_rms_norm_fp8`` gives them); returns [..., n] in the weight's type.

    Made for few rows (a decode step's): the weight is read once for up to 64 rows, and from L2
    for each 64 more.  One or two rows are taken as fixed-point numbers, to 2^-27 of the largest
    magnitude of their 128 channels; more rows as they are.  ``out`` must not overlap an operand.
    No gradient."""
    if not isinstance(weight, Weight4) or len(weight.shape) != 2:
        raise ValueError("linear4 takes one Weight4 matrix")
    n, k = weight.shape
    scales = weight.scales
    device, dtype = scales.device, scales.dtype
    if x.device != device or device.type != "cuda":
        raise ValueError("linear4 takes CUDA activations on the weight's device (no CPU fallback)")
    if x.dim() == 0 or x.shape[-1] != k:
        raise ValueError(f"activations have {k} channels, as the weight")
    code = TYPES.get(x.dtype)
    if x.dtype == torch.float8_e4m3fn:
        code = E4M3
    elif x.dtype != dtype:
        raise ValueError("activations have the type of the weight's scales, or are e4m3")
    refuse_derivatives("linear4", x, x_scale, bias, scales)
    rows = _rows(x, k)
    count = rows.shape[0]
    scale_at = bias_at = None
    if x_scale is not None:
        if code != E4M3 or x_scale.dtype != torch.float32 or x_scale.numel() != count or x_scale.device != device:
            raise ValueError("x_scale is one fp32 value a row of e4m3 activations, on their device")
        x_scale = x_scale.contiguous()
        scale_at = x_scale.data_ptr()
    if bias is not None:
        if bias.shape != (n,) or bias.dtype != dtype or bias.device != device:
            raise ValueError("the bias is one value per output, of the weight's type and device")
        bias = bias.contiguous()
        bias_at = bias.data_ptr()
    shape = (count, n) if x.dim() == 2 else (*x.shape[:-1], n)
    if out is None:
        out = x.new_empty(shape, dtype=dtype) if code == E4M3 else x.new_empty(shape)
    elif out.shape != shape or out.dtype != dtype or out.device != device or not out.is_contiguous():
        raise ValueError("out is a contiguous tensor of the result's shape, type and device")
    _lib.on_device(device.index, _lib.lib().tao_linear4, rows.data_ptr(), rows.stride(0), code, scale_at,
                   *weight.args, bias_at, count, n, k, out.data_ptr())
    return out


__all__ = ["Weight4", "quantize4", "linear4"]
