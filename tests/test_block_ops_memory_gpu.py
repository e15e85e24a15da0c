"""The block operators' memory on the device: outputs that are views."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _layer(width=64, inner=32, experts=4, top_k=2, seed=0):
    from tao_memory_b200 import ExpertWeights
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: (torch.randn(*s, device="cuda", generator=g) * s[-1] ** -0.5).bfloat16()
    return ExpertWeights(n(experts, width), n(experts, inner, width), n(experts, inner, width),
                         n(experts, width, inner), top_k=top_k)


@pytest.mark.parametrize("tokens", [1, 5, 70])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 4, 8])
def test_an_expert_layers_out_may_be_any_contiguous_view(tokens, offset):
    from tao_memory_b200 import expert_layer
    layer = _layer()
    x = torch.randn(tokens, 64, device="cuda").bfloat16()
    want = expert_layer(x, layer)
    room = torch.full((tokens * 64 + 16,), 7.0, device="cuda", dtype=torch.bfloat16)
    out = room[offset:offset + tokens * 64].view(tokens, 64)
    assert expert_layer(x, layer, out=out) is out
    assert torch.equal(out, want)
    assert (room[:offset] == 7).all() and (room[offset + tokens * 64:] == 7).all()


@pytest.mark.parametrize("rows", [1, 2, 5, 40])
@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_a_products_out_may_be_any_contiguous_view(rows, offset):
    from tao_memory_b200 import linear4, quantize4
    w = quantize4(torch.randn(50, 192, device="cuda").bfloat16())
    x = torch.randn(rows, 192, device="cuda").bfloat16()
    room = torch.full((rows * 50 + 16,), 7.0, device="cuda", dtype=torch.bfloat16)
    out = room[offset:offset + rows * 50].view(rows, 50)
    assert linear4(x, w, out=out) is out
    assert torch.equal(out, linear4(x, w))
    assert (room[:offset] == 7).all() and (room[offset + rows * 50:] == 7).all()
