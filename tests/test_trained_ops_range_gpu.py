"""The trained block's operators at the ends of their sizes: elements beyond 2^31, sums over a million rows and over
very long rows, one row and one channel, and first calls inside a capture."""

import os
import subprocess
import sys

import pytest
import torch

from _products import Product, close, half_step, lost

pytestmark = pytest.mark.gpu


def _normal(*shape, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", dtype=torch.bfloat16, generator=g) * scale


@pytest.mark.parametrize("act", [None, "gelu"])
def test_outputs_beyond_31_bits(act):
    from tao_memory_b200 import linear
    rows, k, n = 270001, 64, 8192  # 2.2e9 outputs
    x, w = _normal(rows, k).requires_grad_(True), _normal(n, k, scale=0.125, seed=1)
    y = linear(x, w, activation=act)
    for at in (slice(0, 5), slice(262140, 262150), slice(rows - 5, rows)):  # where the outputs pass 2^31, too
        want = Product(x[at], w, torch.bfloat16, name=act)
        close(y[at].detach(), want.y, want.y_off)
    dy = torch.zeros_like(y)
    dy[-3:] = _normal(3, n, seed=2)
    dx, = torch.autograd.grad(y, x, dy)
    ref = Product(x[-3:], w, torch.bfloat16, name=act).backward(dy[-3:])["dx"]
    close(dx[-3:], *ref)
    assert (dx[:-3] == 0).all()


def test_rows_beyond_31_bits():
    from tao_memory_b200 import embed, gather_tokens, return_tokens, sort_tokens
    tokens, k, width = 33001, 8, 8200  # 2.16e9 elements of sorted rows
    ids = torch.randint(0, 5, (tokens, k), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    order = sort_tokens(ids, 5)
    x = _normal(tokens, width)
    xs = gather_tokens(x, order)
    for at in (0, 1, 2 ** 31 // width, tokens * k - 1):
        assert torch.equal(xs[at], x[order.pairs[at].long() // k])
    xs.requires_grad_(True)
    w = torch.ones(tokens, k, device="cuda", requires_grad=True)
    y = return_tokens(xs, order, w)
    assert torch.equal(y, (x.float() * k).bfloat16())
    dxs, dw = torch.autograd.grad(y, (xs, w), x)
    assert torch.equal(dxs[-1], x[order.pairs[-1].long() // k]) and torch.equal(dxs[2 ** 31 // width], xs[2 ** 31 // width])
    size = x.double().square().sum(-1, keepdim=True)
    assert ((dw - size).abs() <= (width + 1) * 2.0 ** -24 * size).all()
    del xs, dxs, y
    table = _normal(262200, 8200, scale=0.5).requires_grad_(True)
    ids = torch.tensor([262199, 262199, 0, 262143], device="cuda")
    y = embed(ids, table)
    assert torch.equal(y, table.detach()[ids])
    dt, = torch.autograd.grad(y, table, torch.ones_like(y))
    assert (dt[262199] == 2).all() and (dt[0] == 1).all() and (dt[262143] == 1).all() and (dt[1:262143] == 0).all()


def test_sums_over_a_million_rows():
    from tao_memory_b200 import linear
    rows, k, n = 1 << 20, 72, 40
    x, dy = _normal(rows, k), _normal(rows, n, seed=1)
    w, b = _normal(n, k).requires_grad_(True), _normal(n).requires_grad_(True)
    dw, db = torch.autograd.grad(linear(x, w, b), (w, b), dy)
    want, size = dy.double().T @ x.double(), dy.double().abs().T @ x.double().abs()
    off = lost(rows) * size
    close(dw, want, off + half_step(torch.bfloat16) * (want.abs() + off))
    want, off = dy.double().sum(0), rows * 2.0 ** -24 * dy.double().abs().sum(0)
    close(db, want, off + half_step(torch.bfloat16) * (want.abs() + off))


@pytest.mark.parametrize("rows", [1, 20, 40, 300])
def test_long_sums(rows):
    from tao_memory_b200 import linear
    x, w = _normal(rows, 70001), _normal(24, 70001, scale=2.0 ** -8, seed=1)
    want = Product(x, w, torch.bfloat16)
    close(linear(x, w), want.y, want.y_off)


def test_one_of_everything():
    from tao_memory_b200 import embed, expert_linear, gather_tokens, linear, return_tokens, sort_tokens
    one = torch.full((1, 1), 3.0, device="cuda", dtype=torch.bfloat16)
    order = sort_tokens(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), 1)
    assert linear(one, one).item() == 9 and gather_tokens(one, order).item() == 3 and return_tokens(one, order).item() == 3
    assert expert_linear(one, one[None], order.offsets).item() == 9
    assert embed(torch.zeros(1, dtype=torch.int64, device="cuda"), one, 2.0).item() == 6


def test_first_calls_inside_a_capture():
    """What a process sets up once (shared memory, clusters that fit) may be set up while it captures."""
    code = """
import torch, tao_memory_b200 as tb
from tao_memory_b200 import _lib
_lib.lib()
torch.manual_seed(0)
r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
leaves = [t.requires_grad_(True) for t in (r(700, 264), r(520, 264), r(4, 72, 520), r(4, 72, 520), r(90, 264))]
ids, words = torch.randint(0, 4, (700, 2), device="cuda"), torch.randint(0, 90, (700,), device="cuda")
small, few = r(40, 2048), r(3000, 2048)
def step():
    x = leaves[0] + tb.embed(words, leaves[4])
    order = tb.sort_tokens(ids, 4)
    h = tb.gather_tokens(tb.linear(x, leaves[1], activation="gelu"), order)
    y = tb.return_tokens(tb.expert_linear(h, leaves[2], order.offsets, up=leaves[3], activation="silu"), order)
    return [y.detach(), tb.linear(small, few), tb.linear(small[:3], few)] + list(torch.autograd.grad(y.float().sum(), leaves))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outs, step()))
from tao_memory_b200.stream import check_device
assert check_device() == 0
print("ok")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stderr[-2000:]
