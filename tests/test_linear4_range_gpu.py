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
