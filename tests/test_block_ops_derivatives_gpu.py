"""Derivatives that the block operators do not have are refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu


def _n(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda").to(dtype)


def _dual(t):
    return fw.make_dual(t, torch.ones_like(t))


def test_the_norm_has_no_forward_mode_derivative():
    from tao_memory_b200 import add_rms_norm, add_rms_norm_fp8
    x, w, r = (_n(3, 64, dtype=torch.float32) for _ in range(3))
    w = w[0].contiguous()
    for norm in (add_rms_norm, add_rms_norm_fp8):
        with fw.dual_level():
            plain = norm(x, w, r)
            for args in ((_dual(x), w, r), (x, _dual(w), r), (x, w, _dual(r))):
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                        norm(*args)
        assert all(torch.equal(a, b) for a, b in zip(plain, norm(x, w, r)))
        assert len(norm(_n(2, 64))) > 1  # nothing is left of the level


def test_products_and_experts_have_no_forward_mode_derivative():
    from tao_memory_b200 import ExpertWeights, expert_layer, linear4, quantize4
    w, x, bias = quantize4(_n(32, 64)), _n(3, 64), _n(32)
    q, scale = x.to(torch.float8_e4m3fn), torch.ones(3, 1, device="cuda")
    router, gate, up, down = _n(4, 64), _n(4, 32, 64), _n(4, 32, 64), _n(4, 64, 32)
    layer = ExpertWeights(router, gate, up, down, top_k=2)
    with fw.dual_level():
        linear4(x, w, bias), linear4(q, w, x_scale=scale), expert_layer(x, layer)
        duals = ExpertWeights(_dual(router), gate, up, down, top_k=2), ExpertWeights(router, gate, up, _dual(down), top_k=2)
        for call in (lambda: linear4(_dual(x), w), lambda: linear4(x, w, _dual(bias)),
                     lambda: linear4(q, w, x_scale=_dual(scale)), lambda: expert_layer(_dual(x), layer),
                     lambda: expert_layer(x, duals[0]), lambda: expert_layer(x, duals[1])):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    call()


def test_products_and_experts_refuse_whatever_asks_for_a_gradient():
    from tao_memory_b200 import ExpertWeights, Weight4, expert_layer, linear4, quantize4
    w, x, bias = quantize4(_n(32, 64)), _n(3, 64), _n(32)
    q, scale = x.to(torch.float8_e4m3fn), torch.ones(3, 1, device="cuda")
    router, gate, up, down = _n(4, 64), _n(4, 32, 64), _n(4, 32, 64), _n(4, 64, 32)
    leaf = lambda t: t.clone().requires_grad_(True)
    codes, scales, _ = w.to_codes()
    learned = Weight4.from_codes(codes, leaf(scales))
    layers = [ExpertWeights(*(leaf(t) if i == j else t for j, t in enumerate((router, gate, up, down))), top_k=2)
              for i in range(4)]
    four = [quantize4(t) for t in (gate, up, down)]
    layers.append(ExpertWeights(router, four[0], Weight4.from_codes(four[1].to_codes()[0], leaf(four[1].to_codes()[1])),
                                four[2], top_k=2))
    calls = [lambda: linear4(leaf(x), w), lambda: linear4(x, w, leaf(bias)), lambda: linear4(x, learned),
             lambda: linear4(q, w, x_scale=leaf(scale)), lambda: expert_layer(leaf(x), layers[0])]
    calls += [lambda layer=layer: expert_layer(x, layer) for layer in layers]
    for call in calls:
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad():
            assert not call().requires_grad
    with torch.inference_mode():
        assert all(call().shape[0] == 3 for call in calls)
