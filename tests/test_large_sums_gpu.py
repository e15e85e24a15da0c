"""Gradients where the activation's argument is beyond what fp16 holds: the forward pass is finite (or is brought back
by the residual), and silu, gelu and relu have slopes of 0 and 1 there."""

import pytest
import torch

from _products import ACTS, SLOPE, Product, close, lost

pytestmark = pytest.mark.gpu


def _inputs(rows, k, n, dtype, seed=0):
    """Every other row has sums of about +-70400 in two thirds of the outputs, +- in turn; the rest are moderate."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, device="cuda", generator=g)
    w = torch.randn(n, k, device="cuda", generator=g) * k ** -0.5
    x[::2, 0], x[1::2, 0] = 1100.0, 2.0 ** -7
    w[::3, 0], w[1::3, 0], w[2::3, 0] = 64.0, -64.0, 0.0
    return x.to(dtype), w.to(dtype), torch.randn(rows, n, device="cuda", generator=g).to(dtype)


def _near(got, value, off, what):
    """``close``, but that what is beyond fp16 for certain (its greatest value and half a step: 65520) is infinite, and
    what the bound leaves open may be."""
    low, high = value.abs() - off, value.abs() + off
    beyond, within = low >= 65520, high < 65520
    assert torch.equal(got[beyond].double(), value[beyond].sign() * float("inf")), what
    close(got[within], value[within], off[within], what)
    rest = ~(beyond | within)
    assert (got[rest].double() * value[rest].sign() >= low[rest]).all(), what


def _gradient(p, dy):
    """{dx, dw, db}: (value, bound) of a product without a gate, as Product.backward, but that a slope from |z| = 64 on
    is 0 or 1 whatever z is kept as (silu's is 64 e^-64 off there, the gelus' less)."""
    dy, u = dy.double(), p.u
    z_off = p.z_off + u * (p.z.abs() + p.z_off) + p.tiny
    s_off = torch.where(p.z.abs() >= 64, 1e-25, SLOPE * z_off + 2.0 ** -18 * (1 + p.z.abs()))
    if p.name is None:
        s_off = torch.zeros_like(s_off)
    if p.name == "relu":
        s_off = (p.z.abs() <= z_off).double()
    dz, dz_off = dy * p.slope, dy.abs() * s_off
    dz_off = dz_off + u * (dz.abs() + dz_off) + p.tiny
    rows, n = dz.shape
    size = dz.abs() + dz_off
    out = {"dx": (dz @ p.w, dz_off @ p.w.abs() + lost(n) * (size @ p.w.abs())),
           "dw": (dz.T @ p.x, dz_off.T @ p.x.abs() + lost(rows) * (size.T @ p.x.abs())),
           "db": (dz.sum(0), dz_off.sum(0) + lost(16 * rows) * dz.abs().sum(0))}
    return {key: (v, off + u * (v.abs() + off) + p.tiny) for key, (v, off) in out.items()}


# few rows without shared memory; columns of 64 rows, split or not; 128 and 256 outputs; a pair of blocks
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("rows,k,n", [(3, 72, 48), (50, 72, 264), (50, 4096, 250), (200, 72, 264), (200, 4096, 130), (2500, 72, 2304),
                                      (2500, 71, 515), (5120, 2048, 2560)])
def test_linear(rows, k, n, name):
    from tao_memory_b200 import linear
    x, w, dy = _inputs(rows, k, n, torch.float16)
    b = (torch.arange(n, device="cuda") % 5 - 2).half()
    res = torch.zeros(rows, n, device="cuda", dtype=torch.float16)
    want = Product(x, w, torch.float16, b, name=name)
    high = want.y > 60000
    assert (want.z.abs() > 65520).any() and (want.z.abs() < 64).any()
    res[high] = -65504.0
    want = Product(x, w, torch.float16, b, res, name=name)
    if name is None:
        res[want.y < -60000] = 65504.0
        want = Product(x, w, torch.float16, b, res, name=name)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]
    y = linear(*leaves, activation=name)
    close(y.detach(), want.y, want.y_off, "y")
    ref = _gradient(want, dy)
    *grads, dres = torch.autograd.grad(y, leaves, dy)
    for key, got in zip(("dx", "dw", "db"), grads):
        _near(got, *ref[key], key)
    assert torch.equal(dres, dy)


@pytest.mark.parametrize("name", ACTS[1:])
@pytest.mark.parametrize("counts", [[9, 0, 14], [50, 61], [300, 129]])
def test_experts_without_a_gate(counts, name):
    from tao_memory_b200 import expert_linear
    offsets = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    x, w, dy = _inputs(sum(counts), 136, 264, torch.float16)
    w = torch.stack([w] * len(counts))
    w[:, 2::3] *= torch.linspace(0.5, 1, len(counts), device="cuda").view(-1, 1, 1)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    y = expert_linear(*leaves, offsets, activation=name)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    limits = offsets.tolist()
    for e in range(len(counts)):
        at = slice(limits[e], limits[e + 1])
        if limits[e] == limits[e + 1]:
            assert (dw[e] == 0).all()
            continue
        want = Product(x[at], w[e], torch.float16, name=name)
        fits = want.y < 60000
        assert (y[at][want.y > 65520] == float("inf")).all()  # as fp16 has it
        close(y[at][fits].detach(), want.y[fits], want.y_off[fits], "y")
        ref = _gradient(want, dy[at])
        _near(dx[at], *ref["dx"], "dx")
        _near(dw[e], *ref["dw"], "dw")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", ACTS[1:])
@pytest.mark.parametrize("rows", [3, 50, 200, 2500])
def test_nan_stays(rows, name, dtype):
    """An undefined argument does not become a slope of 0 or 1."""
    from tao_memory_b200 import linear
    x, w, dy = _inputs(rows, 72, 264, dtype)
    x[::2, 0] = 1.0
    clean = [t.clone().requires_grad_(True) for t in (x, w)]
    dx0, = torch.autograd.grad(linear(*clean, activation=name), clean[:1], dy)
    x[1, 5] = float("nan")
    leaves = [t.requires_grad_(True) for t in (x, w)]
    y = linear(*leaves, activation=name)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    assert y[1].isnan().all() and dw[:, 5].isnan().all()
    if name != "relu":  # its slope at NaN is 0, as comparisons have it
        assert dx[1].isnan().all()
    keep = torch.arange(rows, device="cuda") != 1
    assert torch.equal(dx[keep], dx0[keep])
