"""CPU-side checks of the block operators: the 4-bit layout the header describes, quantisation,
and the C entries' refusals before any CUDA call."""
import ctypes
import random

import pytest
import torch

from tao_memory_b200 import Weight4, _lib, quantize4


@pytest.mark.parametrize("n,k,group", [(37, 300, 32), (16, 128, 128), (1, 1, 64), (50, 257, 64)])
def test_layout_is_the_headers(n, k, group):
    g = torch.Generator().manual_seed(0)
    parts = -(-k // group)
    codes = torch.randint(0, 16, (2, n, k), generator=g, dtype=torch.uint8)
    scales = torch.rand(2, n, parts, generator=g).bfloat16()
    zeros = torch.randint(0, 16, (2, n, parts), generator=g, dtype=torch.uint8)
    w = Weight4.from_codes(codes, scales, zeros, group)
    assert all(torch.equal(a, b) for a, b in zip(w.to_codes(), (codes, scales, zeros)))
    tiles, blocks, per = -(-n // 16), -(-k // 128), 128 // group
    laid = w.codes.view(2, tiles, blocks, 2, 32, 16)
    ls, lz = (t.view(2, tiles, blocks, 8, per, 2) for t in (w.scales, w.zeros))
    rng = random.Random(1)
    for _ in range(2000):
        e, tile, b, h, lane, byte, half = (rng.randrange(m) for m in (2, tiles, blocks, 2, 32, 16, 2))
        g_, t, i, f, low = lane // 4, lane % 4, byte // 8, byte // 4 % 2, byte % 4
        row, col = 16 * tile + g_ + 8 * half, 128 * b + 64 * h + 32 * i + 8 * t + 4 * f + (0, 2, 1, 3)[low]
        want = int(codes[e, row, col]) if row < n and col < k else 0
        assert int(laid[e, tile, b, h, lane, byte]) >> (4 * half) & 15 == want
        j = rng.randrange(per)
        part = b * per + j
        inside = row < n and part < parts
        assert float(ls[e, tile, b, g_, j, half]) == (float(scales[e, row, part]) if inside else 0)
        assert int(lz[e, tile, b, g_, j, half]) == (int(zeros[e, row, part]) if inside else 0)


@pytest.mark.parametrize("zeros", [False, True])
def test_quantisation_error_is_half_a_step(zeros):
    w = torch.randn(24, 200, generator=torch.Generator().manual_seed(2)) * 0.1
    q = quantize4(w, group=32, zeros=zeros)
    step = q.to_codes()[1].float().repeat_interleave(32, -1)[:, :200]
    # the scale's own rounding (2^-8) moves the ends, a zero point's rounding all of a group
    assert ((q.dequantize() - w).abs() <= (1.06 if zeros else 0.56) * step).all()


def test_refusals_without_gpu():
    lib, arg = _lib.lib(), _lib.TAO_ERR_ARG
    norm = lambda **k: lib.tao_add_rms_norm(*{**dict(x=16, xs=8, r=None, rs=0, w=None, rows=1, width=8, type=0,
                                                     eps=1e-6, s=None, y=16, stream=None), **k}.values())
    assert norm(type=3) == arg and norm(width=0) == arg and norm(width=65537) == arg and norm(rows=-1) == arg
    assert norm(x=None) == arg and norm(r=16) == arg and norm(rows=0, x=None) == _lib.TAO_OK
    assert lib.tao_add_rms_norm_fp8(16, 8, None, 0, None, 1, 8, 0, 1e-6, 64, None, 16, 16, None) == arg
    size = lib.tao_add_rms_norm_workspace_bytes(100, 768, 0)
    assert size > 0 and lib.tao_add_rms_norm_workspace_bytes(100, 768, 7) == 0
    assert lib.tao_add_rms_norm_backward(16, 8, None, 0, 16, 8, None, 100, 768, 0, 1e-6, 16, 16, 16, size - 1,
                                         None) == arg
    product = lambda **k: lib.tao_linear4(*{**dict(x=16, xs=128, xt=0, xscale=None, codes=16, scales=16, zeros=None,
                                                   group=128, type=0, bias=None, rows=1, n=16, k=128, y=16,
                                                   stream=None), **k}.values())
    assert product(group=16) == arg and product(type=2) == arg and product(xt=1) == arg and product(codes=None) == arg
    assert product(n=0) == arg and product(k=65537) == arg and product(rows=-1) == arg
    assert product(scales=24) == arg and b"16 bytes" in lib.tao_last_error()
    assert product(rows=0, x=None) == _lib.TAO_OK
    layer = lambda **k: _lib.TaoExperts(**{**dict(router=16, gate=16, up=16, down=16, gate_expert=64, gate_row=8,
                                                  up_expert=64, up_row=8, down_expert=64, down_row=8, width=8,
                                                  inner=8, experts=2, top_k=1, group=0, renormalize=1), **k})

    def run(l, tokens=1, ws=256, size=1 << 20):
        return lib.tao_expert_layer(ctypes.byref(l), 16, 8, tokens, 16, None, None, ws, size, None)

    for bad in (dict(width=12), dict(inner=0), dict(experts=513), dict(top_k=3), dict(top_k=0), dict(group=16),
                dict(gate=None), dict(group=32), dict(gate_row=4), dict(down=20)):
        assert run(layer(**bad)) == arg, bad
    assert run(layer(), size=256) == arg and run(layer(), tokens=-1) == arg and run(layer(), tokens=0) == _lib.TAO_OK
    assert lib.tao_expert_workspace_bytes(ctypes.byref(layer()), 64) > 0
    assert lib.tao_expert_workspace_bytes(ctypes.byref(layer(experts=0)), 64) == 0
    assert lib.tao_expert_check(None, 0, None, None) == arg
