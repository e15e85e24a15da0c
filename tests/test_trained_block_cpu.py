"""What TrainedBlock and TrainedDecoder refuse when they are made (no GPU needed)."""

import pytest
import torch

from tao_memory_b200.model import TrainedBlock, TrainedDecoder


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_types_the_attention_does_not_take(dtype):
    with pytest.raises(ValueError):
        TrainedBlock(2, 64, 96, device="cpu", dtype=dtype)
    block = TrainedBlock(2, 64, 96, device="cpu")
    assert all(p.dtype == torch.bfloat16 for n, p in block.named_parameters() if "fusion" not in n)
    with pytest.raises(ValueError):
        TrainedDecoder(50, [block], device="cpu", dtype=dtype)
    assert TrainedDecoder(50, [block], device="cpu").table.dtype == torch.bfloat16
