"""add_rms_norm and add_rms_norm_fp8 against the formulas in 64 bits.

Bounds: an output is rounded once from fp32, so it is off by at most the type's unit
roundoff u (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) of itself, plus what the fp32 arithmetic
before it loses: a few units of 2^-24 for a product and the reciprocal root (F = 32 units
bounds them with room), taken of the terms' magnitudes where they cancel."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALL = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25, torch.float32: 1e-37}  # half a subnormal step
F = 32 * 2.0 ** -24
EPS = 1e-5


def _inputs(rows, width, dtype, seed=0, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x = n(rows, width).to(dtype)
    res = (3 * n(rows, width) * torch.exp(n(width))).to(dtype) if residual else None
    return x, res, (1 + 0.3 * n(width)).to(dtype), n(rows, width).to(dtype), n(rows, width).to(dtype)


def _wide(x, w, res):
    s = x if res is None else (x.float() + res.float()).to(x.dtype)
    sd = s.double()
    r = (sd.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return s, sd, r, sd * r * (1 if w is None else w.double())


def _check(a, b, dtype, terms=None):
    terms = b.abs() if terms is None else terms
    bad = (a.double() - b).abs() > U[dtype] * b.abs() + F * terms + SMALL[dtype]
    assert not bad.any(), (int(bad.sum()), (a.double() - b).abs().max().item())


SHAPES = [(1, 1), (1, 64), (3, 7), (8, 768), (5, 1001), (2, 1024), (1185, 96), (1300, 768), (1201, 2048), (1190, 4100),
          (7, 8192), (1200, 8192), (3, 16384), (2, 65536), (2600, 480), (600, 2048), (1700, 640)]


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("residual", [True, False])
def test_forward(rows, width, dtype, residual):
    from tao_memory_b200 import add_rms_norm
    if dtype == torch.float32 and width > 32768:
        width //= 2
    x, res, w, _, _ = _inputs(rows, width, dtype, residual=residual)
    y, s = add_rms_norm(x, w, res, eps=EPS)
    ref_s, _, _, ref = _wide(x, w, res)
    assert torch.equal(s, ref_s) and y.dtype == dtype
    _check(y, ref, dtype)
    _check(add_rms_norm(x, None, res, eps=EPS)[0], _wide(x, None, res)[3], dtype)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows,width", [s for s in SHAPES if s[1] <= 16384])
@pytest.mark.parametrize("residual", [True, False])
def test_gradient(rows, width, dtype, residual):
    from tao_memory_b200 import add_rms_norm
    x, res, w, dy, ds = _inputs(rows, width, dtype, seed=1, residual=residual)
    leaves = [t.clone().requires_grad_(True) for t in (x, w) + ((res,) if residual else ())]
    y, s = add_rms_norm(leaves[0], leaves[1], leaves[2] if residual else None, eps=EPS)
    grads = torch.autograd.grad((y, s) if residual else y, leaves, (dy, ds) if residual else dy)
    _, sd, r, _ = _wide(x, w, res)
    n, g = sd * r, dy.double()
    wg = w.double() * g
    mean = (wg * n).mean(-1, keepdim=True)
    dx = r * (wg - n * mean) + (ds.double() if residual else 0)
    # the mean is a sum of terms that cancel: its loss goes by their magnitudes
    loss = (wg * n).abs().mean(-1, keepdim=True)
    terms = r * (wg.abs() + n.abs() * (loss + mean.abs())) + (ds.double().abs() if residual else 0)
    _check(grads[0], dx, dtype, terms)
    if residual:
        assert torch.equal(grads[2], grads[0])
    # a column's sum runs over at most a few dozen additions in each of its two stages
    _check(grads[1], (g * n).sum(0), dtype, 4 * (g * n).abs().sum(0))


def test_gradient_against_differences():
    """Central differences of the kernel's own forward in fp32, step h = 2^-6 along a random
    direction of unit size per element: truncation of order h^2 = 2.4e-4 of the gradient."""
    from tao_memory_b200 import add_rms_norm
    x, res, w, dy, ds = _inputs(33, 515, torch.float32, seed=2)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, res)]
    y, s = add_rms_norm(*leaves, eps=EPS)
    grads = torch.autograd.grad((y, s), leaves, (dy, ds))
    h = 2.0 ** -6
    for i in range(3):
        d = torch.randn_like(leaves[i])
        at = []
        for sign in (1, -1):
            args = [t.detach() + (sign * h * d if j == i else 0) for j, t in enumerate(leaves)]
            y, s = add_rms_norm(*args, eps=EPS)
            at.append((y.double() * dy.double()).sum() + (s.double() * ds.double()).sum())
        got = (at[0] - at[1]) / (2 * h)
        want = (grads[i].double() * d.double()).sum()
        size = grads[i].double().norm()
        assert (got - want).abs() <= 5e-3 * size, (i, got.item(), want.item(), size.item())


@pytest.mark.parametrize("use", ["y", "s"])
def test_gradient_of_one_output(use):
    from tao_memory_b200 import add_rms_norm
    x, res, w, dy, ds = _inputs(9, 200, torch.float32, seed=3)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, res)]
    y, s = add_rms_norm(*leaves, eps=EPS)
    if use == "s":
        s.backward(ds)
        assert torch.equal(leaves[0].grad, ds) and torch.equal(leaves[2].grad, ds) and leaves[1].grad is None
        return
    y.sum().backward()  # a broadcast gradient
    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    sd = ref[0] + ref[2]
    ((sd * (sd.square().mean(-1, keepdim=True) + EPS).rsqrt()) * ref[1]).sum().backward()
    for a, b in zip(leaves, ref):
        # the stream is rounded to fp32 before the norm; its gradient cancels to small values
        assert (a.grad.double() - b.grad).abs().max() <= 1e-5 * b.grad.abs().max() + 1e-6


def _check_fp8(q, scale, y, group):
    width = y.shape[-1]
    part = width if group is None else 128
    for i, c in enumerate(y.split(part, -1)):
        top = c.abs().amax(-1).clamp_min(1e-30)
        assert ((scale[..., i].double() - top / 448).abs() <= F * top / 448).all()
        v = c * (448 / top).unsqueeze(-1)
        # e4m3: unit roundoff 2^-4, half a subnormal step 2^-10, and the fp32 loss of v itself
        off = (q[..., i * part:(i + 1) * part].double() - v).abs()
        assert (off <= (2.0 ** -4 + F) * v.abs() + 2.0 ** -10).all()


@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows,width", [(1, 1), (4, 130), (9, 768), (3, 1001), (1300, 768), (1190, 2048), (1200, 5000),
                                        (2, 16384), (1700, 640), (600, 2048)])
def test_fp8(rows, width, dtype, group):
    from tao_memory_b200 import add_rms_norm_fp8
    x, res, w, _, _ = _inputs(rows, width, dtype, seed=4)
    q, scale, s = add_rms_norm_fp8(x, w, res, eps=EPS, group=group)
    ref_s, _, _, y = _wide(x, w, res)
    assert torch.equal(s, ref_s) and q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
    assert scale.shape == (rows, 1 if group is None else -(-width // 128))
    _check_fp8(q, scale, y, group)


def test_rows_of_zeros_and_without_numbers():
    from tao_memory_b200 import add_rms_norm, add_rms_norm_fp8
    x = torch.randn(4, 512, device="cuda", dtype=torch.bfloat16)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    y, _ = add_rms_norm(x, eps=EPS)
    q, scale, _ = add_rms_norm_fp8(x, eps=EPS)
    assert (y[1] == 0).all() and (q[1].float() == 0).all() and scale[1].item() > 0
    assert y[2].isnan().all() and q[2].float().isnan().all() and scale[2].isnan().all()
    # an infinity has r = 0: zeros, and a NaN in its own place
    assert y[3, 7].isnan() and (y[3, :7] == 0).all()
    ref = _wide(x[:1], None, None)[3]
    _check(y[:1], ref, torch.bfloat16)


def test_strides_offsets_and_leading_axes():
    from tao_memory_b200 import add_rms_norm, add_rms_norm_fp8
    base = torch.randn(6, 5, 300, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(96, device="cuda", dtype=torch.bfloat16)
    for x, res in ((base[:, 1, 3:99], base[:, 2, 8:104]),           # rows apart, one off its alignment
                   (base[:, :, 40:136], base[:, :, 104:200]),       # leading axes
                   (base.transpose(0, 2)[:96].permute(2, 1, 0), base[:, :, :96]),  # last axis not contiguous
                   (base[:1, 0, :96].expand(6, 96), base[:, 0, :96])):              # rows that are one row
        y, s = add_rms_norm(x, w, res, eps=EPS)
        ref_s, _, _, ref = _wide(x, w, res)
        assert torch.equal(s, ref_s) and y.shape == x.shape
        _check(y, ref, torch.bfloat16)
        q, scale, s = add_rms_norm_fp8(x, w, res, eps=EPS)
        assert torch.equal(s, ref_s)
        _check_fp8(q, scale, ref, None)
    empty = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y, _ = add_rms_norm(empty, w)
    y.sum().backward()
    assert y.shape == (0, 64) and (w.grad == 0).all()


def test_same_result_on_another_stream_and_again():
    from tao_memory_b200 import add_rms_norm
    x, res, w, dy, ds = _inputs(5000, 768, torch.bfloat16, seed=5)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, res)]
    outs = []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (torch.cuda.current_stream(), side, side):
        with torch.cuda.stream(stream):
            y, s = add_rms_norm(*leaves, eps=EPS)
            outs.append((y, s) + torch.autograd.grad((y, s), leaves, (dy, ds)))
    torch.cuda.synchronize()
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_gradient_has_no_gradient():
    from tao_memory_b200 import add_rms_norm
    x, _, w, _, _ = _inputs(3, 64, torch.float32, residual=False)
    y, _ = add_rms_norm(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_captured_training_step():
    from tao_memory_b200 import add_rms_norm
    x, res, w, dy, ds = _inputs(300, 256, torch.bfloat16, seed=6)
    leaves = [t.requires_grad_(True) for t in (x, w, res)]

    def step():
        y, s = add_rms_norm(*leaves, eps=EPS)
        return (y, s) + torch.autograd.grad((y, s), leaves, (dy, ds))

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.no_grad():
        x.mul_(1.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(outs, step()))


def test_refusals():
    from tao_memory_b200 import add_rms_norm, add_rms_norm_fp8
    x = torch.randn(4, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    for bad in (lambda: add_rms_norm(x.cpu()), lambda: add_rms_norm(x.double()), lambda: add_rms_norm(x, w[:32]),
                lambda: add_rms_norm(x, w.float()), lambda: add_rms_norm(x, w, x[:2]),
                lambda: add_rms_norm(x, w, x.float()), lambda: add_rms_norm(x[:, :0]),
                lambda: add_rms_norm_fp8(x, w, group=64), lambda: add_rms_norm(x.new_zeros(1, 65537)),
                lambda: add_rms_norm_fp8(x.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            bad()
