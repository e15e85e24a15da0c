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


@pytest.mark.parametrize("count", [0, 1, 3])
def test_states_of_another_number_of_blocks(count):
    """A prompt with too few went through as many blocks as it had states; with too many the rest stayed empty."""
    model = TrainedDecoder(50, [TrainedBlock(2, 64, 96, device="cpu") for _ in range(2)], device="cpu")
    with pytest.raises(ValueError, match="each of the 2 blocks"):
        model.prefill(torch.zeros(5, dtype=torch.int64), [None] * count)
    with pytest.raises(ValueError, match="each of the 2 blocks"):
        model.step(torch.zeros(2, dtype=torch.int64), [[None] * 2, [None] * count])
