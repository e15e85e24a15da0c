"""``linear`` against 64 bits: every form of the product kernels, odd sizes, strides, refusals."""

import pytest
import torch

from _products import ACTS, Product, close

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def _inputs(rows, k, n, dtype, bias=False, residual=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    return (normal(rows, k), normal(n, k, scale=k ** -0.5), normal(n, scale=0.5) if bias else None,
            normal(rows, n) if residual else None, normal(rows, n))


def _check(x, w, b, res, dy, name, grad=True):
    from tao_memory_b200 import linear
    leaves = [None if t is None else t.detach().clone().requires_grad_(True) for t in (x, w, b, res)]
    want = Product(x, w, x.dtype, b, res, name=name)
    with torch.no_grad():
        y = linear(*leaves, activation=name)
    close(y, want.y, want.y_off, "y")
    if not grad:
        return
    again = linear(*leaves, activation=name)
    assert torch.equal(y, again.detach())
    used = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(again, used, dy))
    ref = want.backward(dy)
    for key, leaf in zip(("dx", "dw", "db", "dres"), leaves):
        if leaf is None:
            continue
        got = next(grads)
        assert got.dtype == x.dtype and got.shape == leaf.shape
        if key == "dres":
            assert torch.equal(got, dy)
        else:
            close(got, *ref[key], key)


# every tile: 16, 32 and 64 columns of few rows; 64, 128 and 256 outputs; with and without a split
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n", [(1, 64, 128), (1, 2048, 640), (2, 1, 1), (7, 65, 33), (16, 512, 130), (17, 96, 1000),
                                      (33, 4096, 257), (64, 130, 72), (65, 64, 64), (100, 2048, 200), (129, 63, 129),
                                      (300, 1001, 515), (1500, 200, 1200), (2500, 136, 2304), (1003, 72, 8),
                                      (200, 1300, 1300), (70, 4096, 1024), (4100, 264, 520), (640, 2304, 72)])
def test_sizes(rows, k, n, dtype):
    x, w, _, _, dy = _inputs(rows, k, n, dtype)
    _check(x, w, None, None, dy, None)


# pairs of blocks: forward, the input's and the weight's gradient, the last one split or not; whole and ragged tiles
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n,name", [(5100, 2050, 2600, "silu"), (5120, 2048, 2560, None), (4737, 2056, 2497, "gelu"),
                                           (20000, 770, 2300, None), (20001, 762, 2297, None), (16500, 768, 2304, "relu"),
                                           (1031, 3902, 4090, None), (1100, 4096, 4096, "gelu"), (3701, 4090, 4095, None)])
def test_pairs_of_blocks(rows, k, n, name, dtype):
    x, w, b, res, dy = _inputs(rows, k, n, dtype, True, True, seed=rows)
    _check(x, w, b, res, dy, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("rows,k,n", [(5, 72, 40), (64, 100, 129), (90, 256, 65), (1500, 64, 1200), (2500, 72, 2312)])
def test_epilogue(rows, k, n, name, dtype):
    for bias, residual in ((True, True), (True, False), (False, True)):
        x, w, b, res, dy = _inputs(rows, k, n, dtype, bias, residual, seed=n)
        _check(x, w, b, res, dy, name, grad=bias)


@pytest.mark.parametrize("wanted", [("w",), ("x",), ("b",), ("res",), ("x", "b")])
def test_some_gradients(wanted):
    from tao_memory_b200 import linear
    x, w, b, res, dy = _inputs(200, 96, 64, torch.bfloat16, True, True)
    all_ = {"x": x, "w": w, "b": b, "res": res}
    full = {k: t.detach().clone().requires_grad_(True) for k, t in all_.items()}
    part = {k: t.detach().clone().requires_grad_(k in wanted) for k, t in all_.items()}
    grads = [torch.autograd.grad(linear(*d.values(), activation="gelu"), [d[k] for k in wanted], dy) for d in (full, part)]
    assert all(torch.equal(a, c) for a, c in zip(*grads))


def test_gradient_against_differences():
    from tao_memory_b200 import linear
    x, w, b, res, dy = _inputs(90, 40, 56, torch.float16, True, True, seed=5)
    for name in ACTS:
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b, res)]
        grads = torch.autograd.grad(linear(*leaves, activation=name), leaves, dy)
        for i, g in enumerate(grads):
            at = [t.detach().double() for t in (x, w, b, res)]
            way = torch.randn(at[i].shape, device="cuda", dtype=torch.double, generator=torch.Generator("cuda").manual_seed(i))
            step = 1e-6
            sides = []
            for sign in (1, -1):
                moved = list(at)
                moved[i] = at[i] + sign * step * way
                sides.append((Product(moved[0], moved[1], torch.float16, moved[2], moved[3], name=name).y * dy.double()).sum())
            want = (sides[0] - sides[1]) / (2 * step)
            # the gradient's elements are off by a few half steps (2^-11) of themselves or of their terms
            assert (want - (g.double() * way).sum()).abs() <= 8 * 2.0 ** -11 * (g.double() * way).norm() + 1e-4


def test_strides_and_leading_axes():
    from tao_memory_b200 import linear
    g = torch.Generator(device="cuda").manual_seed(2)
    base = torch.randn(6, 40, 3 * 96, device="cuda", generator=g).bfloat16()
    w = torch.randn(2 * 80, 2 * 96, device="cuda", generator=g).bfloat16() * 0.1
    dy = torch.randn(6, 40, 80, device="cuda", generator=g).bfloat16()
    views = [base[..., 96:192], base[..., 1:97], base.flip(0)[..., :96], base.transpose(0, 1)[..., :96].transpose(0, 1),
             base[:, :1, :96].expand(6, 40, 96), base.transpose(1, 2)[:, :96, :].transpose(1, 2)]
    for x in views:
        for weight in (w[:80, 96:], w[1::2, 3:99], w[:, :80].T[:, :96], w[:1, :96].expand(80, 96)):
            res = base[..., 100:180]
            leaves = [t.detach().requires_grad_(True) for t in (x, weight)]
            y = linear(leaves[0], leaves[1], residual=res, activation="silu")
            want = Product(x.reshape(-1, 96), weight, torch.bfloat16, residual=res.reshape(-1, 80), name="silu")
            close(y.detach().reshape(-1, 80), want.y, want.y_off, "y")
            dx, dw = torch.autograd.grad(y, leaves, dy.transpose(0, 1).contiguous().transpose(0, 1))
            ref = want.backward(dy.reshape(-1, 80))
            close(dx.reshape(-1, 96), *ref["dx"], "dx")
            close(dw, *ref["dw"], "dw")
    y = linear(base[0, 0, :96], w[:80, :96])  # one token without a leading axis
    want = Product(base[0, :1, :96], w[:80, :96], torch.bfloat16)
    assert y.shape == (80,)
    close(y.unsqueeze(0), want.y, want.y_off)
    x = base[..., :96].detach().requires_grad_(True)
    linear(x, w[:80, :96]).sum().backward()  # a broadcast gradient
    ref = Product(base[..., :96].reshape(-1, 96), w[:80, :96], torch.bfloat16).backward(torch.ones(240, 80, device="cuda"))
    close(x.grad.reshape(-1, 96), *ref["dx"])


def test_no_rows():
    from tao_memory_b200 import linear
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w, b = (torch.ones(*s, device="cuda", dtype=torch.bfloat16, requires_grad=True) for s in ((32, 64), (32,)))
    y = linear(x, w, b, activation="silu")
    y.sum().backward()
    assert y.shape == (0, 32) and x.grad.shape == (0, 64) and (w.grad == 0).all() and (b.grad == 0).all()


@pytest.mark.parametrize("rows", [3, 50, 200])
def test_infinities_and_nan_stay_in_their_rows(rows):
    from tao_memory_b200 import linear
    x, w, _, _, dy = _inputs(rows, 100, 72, torch.bfloat16)
    clean = linear(x, w, activation="gelu_tanh")
    x[1, 5], x[2, 99] = float("nan"), float("inf")
    y = linear(x, w, activation="gelu_tanh")
    assert y[1].isnan().all() and not y[2].isfinite().all()
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[1] = keep[2] = False
    assert torch.equal(y[keep], clean[keep])


def test_residual_in_place_of_the_output():
    from tao_memory_b200 import _lib
    x, w, _, res, _ = _inputs(300, 128, 96, torch.bfloat16, residual=True)
    want = Product(x, w, torch.bfloat16, residual=res)
    p = _lib.TaoLinear(x=x.data_ptr(), x_row=128, x_col=1, w=w.data_ptr(), w_row=128, w_col=1, residual=res.data_ptr(), r_row=96,
                       rows=300, n=96, k=128, experts=1, y=res.data_ptr())
    _lib.on_device(0, _lib.lib().tao_linear, p)
    close(res, want.y, want.y_off)


def test_same_result_on_other_streams_at_once():
    from tao_memory_b200 import linear
    x, w, b, res, dy = _inputs(700, 768, 264, torch.bfloat16, True, True)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                y = linear(*leaves, activation="gelu")
                outs.append((y,) + torch.autograd.grad(y, leaves, dy) + (linear(x[:9], w),))
    torch.cuda.synchronize()
    for other in outs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(outs[0], other))


def test_captured_training_step():
    from tao_memory_b200 import linear
    x, w, b, _, dy = _inputs(300, 130, 96, torch.bfloat16, True)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = linear(*leaves, activation="silu")
        return (y.detach(), linear(x[:5].detach(), w.detach())) + torch.autograd.grad(y, leaves, dy)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.no_grad():
        x.mul_(0.75)
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(outs, step()))


def test_gradient_has_no_gradient():
    from tao_memory_b200 import linear
    x, w, _, _, _ = _inputs(3, 64, 32, torch.bfloat16)
    y = linear(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_refusals():
    from tao_memory_b200 import linear
    x, w, b, res, _ = _inputs(6, 64, 32, torch.bfloat16, True, True)
    for bad in (lambda: linear(x.float(), w.float()), lambda: linear(x, w.half()), lambda: linear(x[:, :60], w),
                lambda: linear(x, w[None]), lambda: linear(x, w, bias=b[:31]), lambda: linear(x, w, bias=b.float()),
                lambda: linear(x, w, residual=res[:5]), lambda: linear(x, w, residual=res.half()),
                lambda: linear(x, w, activation="tanh"), lambda: linear(x, w.cpu()), lambda: linear(x[:, :0], w[:, :0])):
        with pytest.raises(ValueError):
            bad()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(ValueError):
            linear(fwd.make_dual(x, x), w)


def test_no_wait_ran_out():
    from tao_memory_b200.stream import check_device
    assert check_device() == 0
