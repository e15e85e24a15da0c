"""The 16-bit products in 64 bits, and how far a kernel's outputs may be from them.

u = eps / 2 is a rounding to the operands' type.  A sum of K terms in fp32 by matrix instructions of 16 terms is off
by at most (K / 16 + 16) 2^-22 of the sum of the terms' magnitudes (each of its additions by 2^-23 of a partial sum
or, where the instruction cuts off instead of rounding, 2^-22).  Activations are computed to 2^-19 of their value; act
has a slope of at most 1.13, act' one of at most 1.13 (silu 0.5, both gelus below 1.13), but relu's, which jumps at 0.
"""

import math

import torch

ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]
SLOPE = 1.13


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def act(z, name):
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return z * (1 + t) / 2, (1 + t) / 2 + z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z) / 2
    return z, torch.ones_like(z)


def lost(terms):
    return (terms / 16 + 16) * 2.0 ** -22


def close(got, want, off, what=""):
    bad = (got.double() - want).abs() - off
    assert got.shape == want.shape and not got.isnan().any(), what
    assert bad.numel() == 0 or bad.max() <= 0, (what, bad.max().item(), want.abs().max().item())


class Product:
    """y = act(x W^T + b) (* (x U^T)) + residual of 64-bit operands, its gradient, and both's bounds."""

    def __init__(self, x, w, dtype, b=None, residual=None, up=None, name=None):
        self.u, self.tiny, self.name = half_step(dtype), tiny(dtype), name
        x, w, b, residual, up = (None if t is None else t.detach().double() for t in (x, w, b, residual, up))
        self.x, self.w, self.up = x, w, up
        k = x.shape[1]
        self.z = x @ w.T + (0 if b is None else b)
        self.z_off = lost(k) * (x.abs() @ w.abs().T + (0 if b is None else b.abs())) + 1e-37
        self.a, self.slope = act(self.z, name)
        self.g = torch.ones_like(self.z) if up is None else x @ up.T
        self.g_off = torch.zeros_like(self.z) if up is None else lost(k) * (x.abs() @ up.abs().T) + 1e-37
        self.y = self.a * self.g + (0 if residual is None else residual)
        a_off = SLOPE * self.z_off + 2.0 ** -19 * self.a.abs() + 1e-37
        self.y_off = a_off * (self.g.abs() + self.g_off) + self.a.abs() * self.g_off + 2.0 ** -22 * self.y.abs()
        self.y_off += self.u * (self.y.abs() + self.y_off) + self.tiny

    def backward(self, dy):
        """{dx, dw, dup, db}: (value, bound)."""
        dy = dy.detach().double()
        u, tiny_ = self.u, self.tiny
        z_off = self.z_off + u * (self.z.abs() + self.z_off) + tiny_  # z is kept rounded, and so is the gate's factor
        if self.name is None:
            z_off = self.z_off if self.up is None else z_off
        g_off = self.g_off if self.up is None else self.g_off + u * (self.g.abs() + self.g_off) + tiny_
        a_off = SLOPE * z_off + 2.0 ** -18 * (1 + self.z.abs())
        s_off = SLOPE * z_off + 2.0 ** -18 * (1 + self.z.abs()) if self.name else torch.zeros_like(self.z)
        if self.name == "relu":
            s_off = (self.z.abs() <= z_off).double()
        dz = dy * self.g * self.slope
        dz_off = dy.abs() * (s_off * (self.g.abs() + g_off) + g_off * self.slope.abs())
        dz_off = dz_off + u * (dz.abs() + dz_off) + tiny_
        k, (rows, n) = self.x.shape[1], dz.shape
        pairs = 1 if self.up is None else 2
        dx, dx_off = dz @ self.w, dz_off @ self.w.abs()
        size = (dz.abs() + dz_off) @ self.w.abs()
        out = {}

        def weight(d, d_off):
            value, off = d.T @ self.x, d_off.T @ self.x.abs()
            off = off + lost(rows) * ((d.abs() + d_off).T @ self.x.abs())
            return value, off + u * (value.abs() + off) + tiny_

        out["dw"] = weight(dz, dz_off)
        if self.up is not None:
            du = dy * self.a
            du_off = dy.abs() * a_off
            du_off = du_off + u * (du.abs() + du_off) + tiny_
            dx, dx_off = dx + du @ self.up, dx_off + du_off @ self.up.abs()
            size = size + (du.abs() + du_off) @ self.up.abs()
            out["dup"] = weight(du, du_off)
        dx_off = dx_off + lost(n * pairs) * size
        out["dx"] = dx, dx_off + u * (dx.abs() + dx_off) + tiny_
        db, db_off = dz.sum(0), dz_off.sum(0) + lost(16 * rows) * dz.abs().sum(0)
        out["db"] = db, db_off + u * (db.abs() + db_off) + tiny_
        return out
