"""One expert with as many rows as there may be: its weight's gradient is one tile whose sums take seconds."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_weight_gradient_of_2_to_the_30_rows():
    from tao_memory_b200 import _lib
    from tao_memory_b200.stream import check_device
    rows, n, k = 1 << 30, 8, 8
    if torch.cuda.mem_get_info()[0] < 5 * rows * n * 2 // 2:
        pytest.skip("the operands take 34 GB")
    x, dy = (torch.zeros(rows, 8, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    at = [0, 63, 64, 1 << 29, rows - 65, rows - 1]
    for i, r in enumerate(at):
        x[r], dy[r] = torch.arange(8, device="cuda") + i, 2.0 ** i
    offsets = torch.tensor([0, rows], device="cuda", dtype=torch.int32)
    dw = torch.empty(1, n, k, device="cuda", dtype=torch.bfloat16)
    p = _lib.TaoLinear(x=x.data_ptr(), x_row=k, x_col=1, offsets=offsets.data_ptr(), experts=1, rows=rows, n=n, k=k,
                       dy=dy.data_ptr(), dy_row=n, dw=dw.data_ptr())
    _lib.on_device(0, _lib.lib().tao_linear_gradient, p)
    assert check_device() == 0
    want = dy[at].double().T @ x[at].double()  # sums of whole numbers, exact in 32 bits
    assert torch.equal(dw[0], want.bfloat16())
