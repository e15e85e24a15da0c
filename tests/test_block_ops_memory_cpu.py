"""The block operators' memory, as far as no GPU is needed to see it: what the C entries refuse
before any CUDA call."""
import ctypes

from tao_memory_b200 import _lib


def _layer(**k):
    return _lib.TaoExperts(**{**dict(router=1 << 20, gate=1 << 20, up=1 << 20, down=1 << 20, gate_expert=64,
                                     gate_row=8, up_expert=64, up_row=8, down_expert=64, down_row=8, width=8, inner=8,
                                     experts=2, top_k=1, group=0, renormalize=1), **k})


def _experts(x, out, tokens=1, stride=8):
    return _lib.lib().tao_expert_layer(ctypes.byref(_layer()), x, stride, tokens, out, None, None, 1 << 21, 1 << 20,
                                       None)


def test_an_expert_layers_out_starts_on_8_bytes():
    # the sums' kernel stores 8 bytes at a time
    for offset in (1, 2, 4, 6, 10):
        assert _experts(16, (1 << 22) + offset) == _lib.TAO_ERR_ARG, offset
        assert b"8 bytes" in _lib.lib().tao_last_error()
