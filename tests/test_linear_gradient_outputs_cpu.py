"""``tao_linear_gradient`` where no output is asked for: nothing is launched (no GPU needed)."""

import pytest

from tao_memory_b200 import _lib
from test_trained_ops_cpu import DY, EXPERTS, GATED, LOW, U, Z, _described


@pytest.mark.parametrize("form", [dict(), dict(activation=2, z=Z, z_row=32), dict(EXPERTS), dict(EXPERTS, activation=1, z=Z, z_row=32),
                                  dict(GATED, z=Z, u=U, low=LOW, z_row=32), dict(GATED, z=Z, u=U, low=LOW, z_row=32, activation=2)])
def test_no_output(form):
    lib = _lib.lib()
    p = _described(dy=DY, dy_row=32, y=None, **form)
    assert lib.tao_linear_workspace_bytes(p, 1) == 0
    assert lib.tao_linear_gradient(p, None) == _lib.TAO_OK
    for name in ("dy",) + (("z",) if "activation" in form or "up" in form else ()):  # still looked at
        assert lib.tao_linear_gradient(_described(**{**dict(dy=DY, dy_row=32, y=None), **form, name: None}), None) == _lib.TAO_ERR_ARG
