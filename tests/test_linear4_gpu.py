"""linear4 against the dequantised product in 64 bits.

Bound: y is rounded once (unit roundoff u: 2^-8 bf16, 2^-11 fp16; half a subnormal step of
fp16), and the fp32 sums before it lose at most D units of 2^-24 of the sum of the terms'
magnitudes, D the depth of the additions: 16 in a group (8 matrix instructions, which may
truncate), one a group of a warp's or block's run of k (at most 2304 / 128 at group 128, four
times that at 32, and a part of it where several share k), 8 to 16 such sums, and the scalings:
D = 64 for the sizes here.  One or two rows have exact group sums in whole numbers, of x to
2^-21 of the largest magnitude of its 128: for normal x at most 5 times the mean, 40 units."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
D = 64 * 2.0 ** -24


def _weight(n, k, group, zeros, dtype, seed=0):
    from tao_memory_b200 import Weight4
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), device="cuda", dtype=torch.uint8, generator=g)
    parts = -(-k // group)
    scales = ((torch.rand(n, parts, device="cuda", generator=g) + 0.1) * k ** -0.5 * 0.3).to(dtype)
    z = torch.randint(0, 16, (n, parts), device="cuda", dtype=torch.uint8, generator=g) if zeros else None
    at = torch.arange(k, device="cuda") // group
    wide = (codes.double() - (8 if z is None else z.double()[:, at])) * scales.double()[:, at]
    return Weight4.from_codes(codes, scales, z, group), wide


def _x(rows, k, act, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, device="cuda", generator=g)
    if act == "fp8":
        scale = x.abs().amax(-1, keepdim=True) / 448
        q = (x / scale).to(torch.float8_e4m3fn)
        return q, scale, q.float().double() * scale.double()
    x = x.to(act)
    return x, None, x.double()


def _check(y, xd, wide, bias=None):
    ref, terms = xd @ wide.T, xd.abs() @ wide.abs().T
    if bias is not None:
        ref, terms = ref + bias.double(), terms + bias.double().abs()
    small = 2.0 ** -25 if y.dtype == torch.float16 else 0
    bad = (y.double() - ref).abs() > U[y.dtype] * ref.abs() + D * terms + small
    assert not bad.any(), (int(bad.sum()), (y.double() - ref).abs().max().item())


SIZES = [(1, 1, 1), (1, 16, 128), (2, 17, 129), (3, 1999, 1001), (4, 40, 2048), (5, 768, 768), (7, 100, 72),
         (8, 2304, 768), (8, 33, 4104), (9, 64, 130), (15, 48, 1000), (16, 256, 1024), (17, 130, 264), (33, 64, 96),
         (64, 80, 640), (129, 24, 200)]


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16, "fp8"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_against_64_bits(rows, n, k, group, act):
    from tao_memory_b200 import linear4
    x, scale, xd = _x(rows, k, act)
    for zeros, bias in ((False, False), (True, True)):
        dtype = torch.bfloat16 if act == "fp8" and zeros else torch.float16 if act == "fp8" else act
        w, wide = _weight(n, k, group, zeros, dtype)
        b = torch.randn(n, device="cuda").to(dtype) if bias else None
        y = linear4(x, w, bias=b, x_scale=scale)
        assert y.shape == (rows, n) and y.dtype == dtype
        _check(y, xd, wide, b)


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16, "fp8"])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("rows,k", [(40, 1100), (64, 1152), (21, 1104)])
def test_all_of_k_in_one_block(rows, k, group, act):
    """More row tiles than the device takes at once: a block has nine runs of 128 k, more than its rings."""
    from tao_memory_b200 import linear4
    x, scale, xd = _x(rows, k, act)
    w, wide = _weight(18960, k, group, True, act if act != "fp8" else torch.bfloat16)
    _check(linear4(x, w, x_scale=scale), xd, wide)


@pytest.mark.parametrize("rows", [1, 8, 24])
def test_large(rows):
    from tao_memory_b200 import linear4
    w, wide = _weight(4099, 8192, 128, True, torch.bfloat16)
    x, _, xd = _x(rows, 8192, torch.bfloat16)
    _check(linear4(x, w), xd, wide)


def test_layout_round_trip_and_quantisation():
    from tao_memory_b200 import Weight4, linear4, quantize4
    codes = torch.randint(0, 16, (3, 37, 300), device="cuda", dtype=torch.uint8)
    scales = torch.rand(3, 37, 10, device="cuda").half()
    zeros = torch.randint(0, 16, (3, 37, 10), device="cuda", dtype=torch.uint8)
    back = Weight4.from_codes(codes, scales, zeros, group=32).to_codes()
    assert all(torch.equal(a, b) for a, b in zip(back, (codes, scales, zeros)))
    weight = torch.randn(96, 500, device="cuda") * 0.05
    weight[3, :64] = 0
    for zero in (False, True):
        w = quantize4(weight, group=64, zeros=zero)
        step = w.to_codes()[1].float().repeat_interleave(64, -1)[:, :500]
        # half a step, and what rounding the scale itself (2^-8) and, with zero points, the
        # zero point (half a step) moves the ends of the range by
        assert ((w.dequantize() - weight).abs() <= (1.06 if zero else 0.56) * step + 1e-9).all()
        assert (w.dequantize()[3, :64] == 0).all()
        x, _, xd = _x(3, 500, torch.bfloat16)
        _check(linear4(x, w), xd, w.dequantize().double())


def test_strides_streams_and_repeats():
    from tao_memory_b200 import linear4
    w, wide = _weight(200, 264, 64, True, torch.bfloat16)
    base = torch.randn(4, 6, 700, device="cuda", dtype=torch.bfloat16)
    views = (base[:, 2, 8:272], base[:, 2, 3:267], base[:, :, 100:364], base[:, 0, ::2][:, :264],
             base[:1, 0, :264].expand(4, 264), base[0, 0, :264])
    for x in views:
        y = linear4(x, w)
        assert y.shape == (*x.shape[:-1], 200)
        _check(y.reshape(-1, 200), x.reshape(-1, 264).double(), wide)
    out = torch.empty(4, 200, device="cuda", dtype=torch.bfloat16)
    x = views[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert linear4(x, w, out=out) is out
    torch.cuda.synchronize()
    assert torch.equal(out, linear4(x, w))
    assert linear4(x[:0], w).shape == (0, 200)


def test_rows_without_numbers_stay_alone():
    """A NaN or an infinity in one row reaches that row's outputs alone."""
    from tao_memory_b200 import linear4
    w, wide = _weight(64, 256, 128, False, torch.bfloat16)
    x, _, xd = _x(5, 256, torch.bfloat16)
    x[1, 9], x[3, 200] = float("nan"), float("inf")
    y = linear4(x, w)
    assert y[1].isnan().all() and not y[3].isfinite().any()
    keep = [0, 2, 4]
    _check(y[keep], xd[keep], wide)


def test_captured_in_a_graph():
    from tao_memory_b200 import linear4
    w, wide = _weight(96, 512, 128, False, torch.bfloat16)
    x, _, xd = _x(2, 512, torch.bfloat16)
    linear4(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = linear4(x, w)
    x.copy_(x * 2)
    graph.replay()
    _check(y, 2 * xd, wide)


def test_refusals():
    from tao_memory_b200 import Weight4, linear4, quantize4
    w, _ = _weight(64, 256, 128, False, torch.bfloat16)
    x, _, _ = _x(2, 256, torch.bfloat16)
    codes = torch.zeros(8, 64, device="cuda", dtype=torch.uint8)
    scales = torch.ones(8, 1, device="cuda", dtype=torch.bfloat16)
    ones = torch.ones(2, 1, device="cuda")
    for bad in (lambda: linear4(x.cpu(), w), lambda: linear4(x.half(), w), lambda: linear4(x[:, :128], w),
                lambda: linear4(x, w, x_scale=ones), lambda: linear4(x, w, bias=x[0]),
                lambda: linear4(x.to(torch.float8_e4m3fn), w, x_scale=ones[:1]),
                lambda: linear4(x, w, out=torch.empty(2, 64, device="cuda")), lambda: linear4(x, w.dequantize()),
                lambda: linear4(x.clone().requires_grad_(True), w), lambda: quantize4(codes),
                lambda: quantize4(x, group=48), lambda: Weight4.from_codes(codes, scales, group=16),
                lambda: Weight4.from_codes(codes + 16, scales), lambda: Weight4.from_codes(codes, scales.float()),
                lambda: Weight4.from_codes(codes, scales[:4]), lambda: Weight4.from_codes(codes, scales, scales)):
        with pytest.raises(ValueError):
            bad()
