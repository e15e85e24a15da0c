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


def test_a_products_out_over_its_activations_is_refused():
    from tao_memory_b200 import linear4, quantize4
    w = quantize4(torch.randn(128, 128, device="cuda").bfloat16())
    room = torch.randn(9, 128, device="cuda").bfloat16()
    kept = room.clone()
    for x, out in ((room[:4], room[:4]), (room[:4], room[3:7]), (room[2:6], room[:4]), (room[:8:2], room[1:5])):
        with pytest.raises(ValueError, match="overlap"):
            linear4(x, w, out=out)
    assert torch.equal(room, kept)
    assert torch.equal(linear4(room[:4], w, out=room[4:8]), linear4(kept[:4], w))


def test_a_products_out_beside_its_activations():
    """What lies next to x, and between rows that are apart, is free."""
    from tao_memory_b200 import linear4, quantize4
    w = quantize4(torch.randn(64, 128, device="cuda").bfloat16())
    room = torch.randn(4096, device="cuda").bfloat16()
    kept = room.clone()
    rows = lambda t, stride: t.as_strided((2, 128), (stride, 1), 1024)
    for stride, at in ((128, 1024 - 128), (128, 1024 + 256), (1024, 1024 + 128), (1024, 2048 - 128), (1024, 2048 + 128),
                       (0, 1024 + 128), (0, 1024 - 128)):
        room.copy_(kept)
        out = room[at:at + 128].view(2, 64)
        assert torch.equal(linear4(rows(room, stride), w, out=out), linear4(rows(kept, stride), w)), (stride, at)
    room.copy_(kept)
    x, bias = room[:256].view(2, 128), room[256:320]
    assert torch.equal(linear4(x, w, bias=bias, out=room[320:448].view(2, 64)), linear4(x, w, bias=bias))
    with pytest.raises(ValueError, match="overlap"):
        linear4(x, w, bias=bias, out=room[300:428].view(2, 64))


@pytest.mark.parametrize("tokens", [3, 64, 65, 200])
def test_an_expert_layers_out_over_its_tokens(tokens):
    from tao_memory_b200 import expert_layer
    layer = _layer()
    x = torch.randn(tokens, 64, device="cuda").bfloat16()
    want = expert_layer(x, layer)
    same = x.clone()
    assert torch.equal(expert_layer(same, layer, out=same), want)
    for shift, off in ((1, 1), (1, 0), (0, 1)):
        room = torch.zeros(tokens + 2, 64, device="cuda", dtype=torch.bfloat16)
        room[shift:shift + tokens] = x
        out = room[off:off + tokens]
        if shift == off or tokens <= 64:
            assert torch.equal(expert_layer(room[shift:shift + tokens], layer, out=out), want)
        else:
            with pytest.raises(ValueError, match="overlap"):
                expert_layer(room[shift:shift + tokens], layer, out=out)
            assert torch.equal(room[shift:shift + tokens], x)


def test_a_copied_or_loaded_weight_outlives_its_original():
    import copy
    import io
    from tao_memory_b200 import linear4, quantize4
    w = quantize4(torch.randn(96, 256, device="cuda").bfloat16(), zeros=True)
    x = torch.randn(3, 256, device="cuda").bfloat16()
    want = linear4(x, w)
    file = io.BytesIO()
    torch.save(w, file)
    file.seek(0)
    others = [copy.deepcopy(w), torch.load(file, weights_only=False)]
    for t in (w.codes, w.scales, w.zeros):
        t.zero_()  # what the original's memory holds no longer matters
    for other in others:
        assert torch.equal(linear4(x, other), want)
    file.seek(0)
    with pytest.raises(ValueError):
        linear4(x, torch.load(file, weights_only=False, map_location="cpu"))


@pytest.mark.parametrize("four", [False, True])
def test_expert_weights_are_copied_and_loaded(four):
    import copy
    import io
    from tao_memory_b200 import ExpertWeights, expert_layer, quantize4
    layer = _layer()
    if four:
        layer = ExpertWeights(layer.router, *(quantize4(w, 32, zeros=True) for w in (layer.gate, layer.up, layer.down)),
                              top_k=2, renormalize=False)
    x = torch.randn(5, 64, device="cuda").bfloat16()
    want = expert_layer(x, layer)
    file = io.BytesIO()
    torch.save(layer, file)
    file.seek(0)
    others = [copy.deepcopy(layer), torch.load(file, weights_only=False)]
    tensors = [t for w in (layer.gate, layer.up, layer.down) for t in ((w.codes, w.scales, w.zeros) if four else (w,))]
    for t in [layer.router, *tensors]:
        t.zero_()
    for other in others:
        assert (other.top_k, other.renormalize) == (layer.top_k, layer.renormalize)
        assert torch.equal(expert_layer(x, other), want)
    file.seek(0)
    with pytest.raises(ValueError):  # a layer is on a GPU
        torch.load(file, weights_only=False, map_location="cpu")


def test_expert_weights_follow_their_tensors():
    """A tensor of a layer cannot be exchanged; one whose memory was (as modules do) is found there."""
    from tao_memory_b200 import expert_layer
    layer, other = _layer(seed=1), _layer(seed=2)
    x = torch.randn(5, 64, device="cuda").bfloat16()
    want, moved = expert_layer(x, other), expert_layer(x, layer)
    for name in ("router", "gate", "up", "down"):
        with pytest.raises(AttributeError):
            setattr(layer, name, getattr(other, name))
    assert torch.equal(expert_layer(x, layer), moved)
    for name in ("router", "gate", "up", "down"):
        getattr(layer, name).data = getattr(other, name).clone()
    assert torch.equal(expert_layer(x, layer), want)
