"""``tao_linear_gradient`` with some of its outputs alone, through the C interface, against 64 bits."""

import pytest
import torch

from _products import Product, close, half_step, lost, tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("outputs", [("db",), ("dx",), ("dw", "dup"), ("dx", "db"), ("dw", "dup", "db"), ()])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n", [(70, 40), (301, 67), (2000, 264)])
def test_gated(rows, n, dtype, outputs):
    """One expert with all but the last 9 rows; db is the sum of dz over all of them, which is 0 in rows of none."""
    from tao_memory_b200 import _lib
    lib, k, row = _lib.lib(), 72, -(-n // 16) * 16
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, w, up, dy = (torch.randn(*s, device="cuda", generator=g).to(dtype) for s in ((rows, k), (1, n, k), (1, n, k), (rows, n)))
    w, up = w * 0.125, up * 0.125
    offsets = torch.tensor([0, rows - 9], device="cuda", dtype=torch.int32)
    y, kept = torch.empty_like(dy), torch.empty(3, rows, row, device="cuda", dtype=dtype)
    plane = kept.stride(0) * 2
    room = torch.empty(1 << 22, device="cuda", dtype=torch.uint8)
    at = room.data_ptr() + -room.data_ptr() % 256
    fields = dict(x=x.data_ptr(), x_row=k, x_col=1, w=w.data_ptr(), w_row=k, w_col=1, w_expert=n * k, up=up.data_ptr(), up_row=k,
                  up_col=1, up_expert=n * k, offsets=offsets.data_ptr(), rows=rows, n=n, k=k, experts=1,
                  type=int(dtype == torch.float16), activation=2, z=kept.data_ptr(), u=kept.data_ptr() + plane,
                  low=kept.data_ptr() + 2 * plane, z_row=row, workspace=at, workspace_bytes=(1 << 22) - 256)
    _lib.on_device(0, lib.tao_linear, _lib.TaoLinear(y=y.data_ptr(), **fields))
    got = {name: torch.full(s, float("nan"), device="cuda", dtype=dtype)
           for name, s in dict(dx=x.shape, dw=w.shape, dup=up.shape, db=(n,)).items() if name in outputs}
    p = _lib.TaoLinear(dy=dy.data_ptr(), dy_row=n, **fields, **{name: t.data_ptr() for name, t in got.items()})
    assert lib.tao_linear_workspace_bytes(p, 1) <= (1 << 22) - 256
    _lib.on_device(0, lib.tao_linear_gradient, p)
    ref = Product(x[:-9], w[0], dtype, up=up[0], name="silu").backward(dy[:-9])
    for name, t in got.items():
        if name == "dx":
            assert (t[-9:] == 0).all()
            t = t[:-9]
        close(t.reshape(ref[name][0].shape), *ref[name], name)


@pytest.mark.parametrize("act", [None, "relu"])
def test_experts_without_a_gate_db_alone(act):
    """db takes all rows, those of no expert too (their argument is 0)."""
    from tao_memory_b200 import _lib
    rows, n, k, dtype = 500, 88, 64, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(4)
    z, dy = (torch.randn(rows, n, device="cuda", generator=g).to(dtype) for _ in range(2))
    db, room = torch.empty(n, device="cuda", dtype=dtype), torch.empty(1 << 18, device="cuda", dtype=torch.uint8)
    offsets = torch.tensor([0, 300, 400], device="cuda", dtype=torch.int32)
    p = _lib.TaoLinear(offsets=offsets.data_ptr(), experts=2, rows=rows, n=n, k=k, type=0, activation=0 if act is None else 1,
                       z=z.data_ptr(), z_row=n, dy=dy.data_ptr(), dy_row=n, db=db.data_ptr(),
                       workspace=room.data_ptr() + -room.data_ptr() % 256, workspace_bytes=(1 << 18) - 256)
    _lib.on_device(0, _lib.lib().tao_linear_gradient, p)
    dz = dy.double() if act is None else dy.double() * (z > 0)
    off = lost(16 * rows) * dz.abs().sum(0)
    want = dz.sum(0)
    close(db, want, off + half_step(dtype) * (want.abs() + off) + tiny(dtype))
