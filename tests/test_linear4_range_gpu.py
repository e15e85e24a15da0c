"""linear4 on activations whose channels differ by orders of magnitude, against 64 bits.

Bound: that of test_linear4_gpu.py (one rounding of y, and D = 64 units of 2^-24 of the terms' magnitudes),
plus what one or two rows lose as fixed-point numbers: a row's 128 channels are whole multiples of
2^-26 to 2^-27 of their largest magnitude M, each rounded to the nearest, so x is off by at most 2^-27 M
and a sum by 2^-27 M times the sum of the 128 weights' magnitudes.  Under a zero weight a large
channel adds nothing to the terms, so that nothing else hides that loss."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
D = 64 * 2.0 ** -24


def _case(rows, n, k, group, dtype, big, seed=0):
    """Weights with zeros at every 64th channel (and one more), activations `big` there."""
    from tao_memory_b200 import Weight4
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), device="cuda", dtype=torch.uint8, generator=g)
    parts = -(-k // group)
    scales = ((torch.rand(n, parts, device="cuda", generator=g) + 0.1) * k ** -0.5).to(dtype)
    zeros = torch.randint(0, 16, (n, parts), device="cuda", dtype=torch.uint8, generator=g)
    at = torch.arange(k, device="cuda") // group
    large = torch.arange(5, k, 64, device="cuda")
    codes[:, large] = zeros[:, at[large]]
    wide = (codes.double() - zeros.double()[:, at]) * scales.double()[:, at]
    x = torch.randn(rows, k, device="cuda", generator=g)
    x[:, large] *= big
    return Weight4.from_codes(codes, scales, zeros, group), wide, x.to(dtype)


def _bound(xd, wide, dtype, rows, ref):
    off = U[dtype] * ref.abs() + D * (xd.abs() @ wide.abs().T) + (2.0 ** -25 if dtype == torch.float16 else 0)
    if rows <= 2:
        for b in range(0, xd.shape[1], 128):
            off = off + 2.0 ** -27 * xd[:, b:b + 128].abs().amax(-1, keepdim=True) * wide[:, b:b + 128].abs().sum(-1)
    return off


@pytest.mark.parametrize("dtype,big", [(torch.bfloat16, 1e3), (torch.bfloat16, 1e4), (torch.bfloat16, 1e5),
                                       (torch.float16, 1e3), (torch.float16, 1e4)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", [(1, 64, 256), (2, 100, 1000), (1, 4099, 4096), (2, 33, 8192), (3, 64, 1000),
                                      (12, 48, 1024), (20, 64, 512)])
def test_large_channels_under_zero_weights(rows, n, k, group, dtype, big):
    from tao_memory_b200 import linear4
    w, wide, x = _case(rows, n, k, group, dtype, big)
    xd = x.double()
    ref = xd @ wide.T
    y = linear4(x, w)
    bad = (y.double() - ref).abs() > _bound(xd, wide, dtype, rows, ref)
    assert not bad.any(), (int(bad.sum()), ((y.double() - ref).norm() / ref.norm()).item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_row_alone_and_among_others(dtype):
    """Both are within the bound of the same number, whatever form their row counts take."""
    from tao_memory_b200 import linear4
    w, wide, x = _case(24, 96, 1024, 64, dtype, 1e4, seed=1)
    xd = x.double()
    ref = xd @ wide.T
    all_rows = linear4(x, w).double()
    for count in (1, 2, 3, 9, 17):
        y = linear4(x[:count], w).double()
        off = _bound(xd[:count], wide, dtype, count, ref[:count]) + _bound(xd[:count], wide, dtype, 24, ref[:count])
        assert ((y - all_rows[:count]).abs() <= off).all()


@pytest.mark.parametrize("size", [0.0, 1e-41, 1e-38, 2.0 ** -101, 2.0 ** -99, 1e-20, 1e20, 3e35])
def test_one_row_of_any_magnitude(size):
    """From subnormal rows to rows whose products are near the type's largest."""
    from tao_memory_b200 import linear4
    w, wide, _ = _case(1, 64, 512, 128, torch.bfloat16, 1.0, seed=2)
    x = (torch.randn(2, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).double() * size)
    x = x.float().bfloat16()
    x[1, 128:256] *= 2.0 ** -60  # of another size than its neighbours
    xd = x.double()
    ref = xd @ wide.T
    y = linear4(x, w).double()
    # y's own subnormals are 2^-133 apart
    assert ((y - ref).abs() <= _bound(xd, wide, torch.bfloat16, 2, ref) + 2.0 ** -132).all()


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16, "fp8"])
@pytest.mark.parametrize("rows", [1, 2, 3, 9, 20])
def test_infinities_and_nans_are_those_of_the_sum(rows, act, group):
    """An infinity gives one of the weight's sign, none under a zero weight (infinity times zero is no
    number), and two of unlike sign give no number: as in a sum term by term.  Other rows are untouched."""
    from tao_memory_b200 import linear4
    dtype = torch.bfloat16 if act == "fp8" else act
    n, k, inf = 70, 1000, float("inf")
    w, wide, clean = _case(rows, n, k, group, dtype, 1.0, seed=4)
    for at, values in ((0, [(3, inf)]), (rows - 1, [(3, inf), (700, -inf)]), (0, [(5, -inf)]), (rows - 1, [(999, float("nan"))])):
        x = clean.clone()
        for c, v in values:
            x[at, c] = v
        scale = None
        if act == "fp8":  # has no infinities: a NaN in their place
            x = torch.where(x.isinf(), torch.full_like(x, float("nan")), x).to(torch.float8_e4m3fn)
            scale = torch.rand(rows, 1, device="cuda") + 0.5
        xd = x.to(torch.float32).double() * (1 if scale is None else scale.double())
        terms = xd[at] * wide  # [n, k]
        y = linear4(x, w, x_scale=scale)
        bad = ~xd[at].isfinite()
        want = terms[:, bad].sum(-1)  # decides over what is finite
        assert torch.equal(y[at].isnan(), want.isnan())
        assert torch.equal(y[at].isposinf(), want == inf) and torch.equal(y[at].isneginf(), want == -inf)
        others = [i for i in range(rows) if i != at]
        ref = xd[others] @ wide.T
        assert ((y[others].double() - ref).abs() <= _bound(xd[others], wide, dtype, rows, ref)).all()
