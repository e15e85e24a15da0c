"""quantize4 of weights whose scales are below the smallest normal number."""
import pytest
import torch

from tao_memory_b200 import quantize4


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-30, 1e-37, 1e-38, 3e-39])
def test_the_error_is_half_a_step_and_zeros_stay(size, dtype, zeros):
    w = torch.randn(6, 96, generator=torch.Generator().manual_seed(1)) * size
    w[:, ::7] = 0
    w = w.to(dtype)
    q = quantize4(w, group=32, zeros=zeros)
    step = q.to_codes()[1].float().repeat_interleave(32, -1)
    # the scale's own rounding moves the ends (8 or 15 steps away) by 2^-8 of it, and by half of bf16's
    # subnormal spacing of 2^-133; a zero point's rounding moves all of a group by half a step
    slack = (1.06 if zeros else 0.56) * step + (15 if zeros else 8) * 2.0 ** -134
    assert ((q.dequantize() - w.float()).abs() <= slack).all()
    assert (q.dequantize()[:, ::7] == 0).all()
