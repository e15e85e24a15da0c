"""``tao_linear``'s kept argument in rows that reach into each other is refused (no GPU needed)."""

import pytest

from tao_memory_b200 import _lib
from test_trained_ops_cpu import DX, DY, EXPERTS, ROOM, Z, _described


@pytest.mark.parametrize("z_row", [0, 1, 31, -32])
@pytest.mark.parametrize("form", [dict(activation=2), dict(EXPERTS, activation=1)])
def test_rows_of_z_that_are_too_short(form, z_row):
    lib = _lib.lib()
    assert lib.tao_linear(_described(z=Z, z_row=z_row, **form), None) == _lib.TAO_ERR_ARG
    assert lib.tao_linear(_described(z=Z, z_row=z_row), None) == _lib.TAO_ERR_ARG  # it is written without an activation too
    p = _described(z=Z, z_row=z_row, dy=DY, dy_row=32, dx=DX, y=None, workspace=ROOM, workspace_bytes=1 << 16, **form)
    assert lib.tao_linear_gradient(p, None) == _lib.TAO_ERR_ARG
    none = _described(z=Z, z_row=z_row, dy=DY, dy_row=32, y=None)  # not read: nothing is refused
    assert lib.tao_linear_gradient(none, None) == _lib.TAO_OK
