"""The trained block's operators within autograd: gradients of some operands, again, of nothing, with what is saved
kept elsewhere, under checkpoints and without gradients."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _all(seed=0, tokens=150):
    """(name, call, leaves) of each operator."""
    from tao_memory_b200 import embed, expert_linear, gather_tokens, linear, return_tokens, sort_tokens
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g).bfloat16()

    ids = torch.randint(-1, 5, (tokens, 3), device="cuda", generator=g)
    words = torch.randint(-1, 40, (tokens,), device="cuda", generator=g)
    order = sort_tokens(ids, 5)
    return [
        ("linear", lambda x, w, b, r: linear(x, w, b, r, activation="gelu"), [normal(tokens, 72), normal(50, 72), normal(50), normal(tokens, 50)]),
        ("odd linear", lambda x, w, b: linear(x, w, b), [normal(tokens, 71), normal(33, 71), normal(33)]),
        ("experts", lambda x, w, u: expert_linear(x, w, order.offsets, up=u, activation="silu"),
         [normal(3 * tokens, 64), normal(5, 40, 64), normal(5, 40, 64)]),
        ("plain experts", lambda x, w: expert_linear(x, w, order.offsets, activation="relu"), [normal(3 * tokens, 64), normal(5, 40, 64)]),
        ("gather", lambda x: gather_tokens(x, order), [normal(tokens, 40)]),
        ("return", lambda ys, w: return_tokens(ys, order, w), [normal(3 * tokens, 40), torch.rand(tokens, 3, device="cuda", generator=g)]),
        ("embed", lambda t: embed(words, t, 2.0), [normal(40, 48)]),
    ]


NAMES = ["linear", "odd linear", "experts", "plain experts", "gather", "return", "embed"]


def _case(name, **kw):
    return next((call, leaves) for n, call, leaves in _all(**kw) if n == name)


def _grads(call, leaves, wanted=None):
    leaves = [t.detach().clone().requires_grad_(wanted is None or i in wanted) for i, t in enumerate(leaves)]
    y = call(*leaves)
    dy = torch.linspace(-1, 1, y.numel(), device="cuda").view(y.shape).to(y.dtype)
    return y.detach(), torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)


@pytest.mark.parametrize("name", NAMES)
def test_each_operand_alone(name):
    call, leaves = _case(name)
    y, full = _grads(call, leaves)
    for i in range(len(leaves)):
        z, (one,) = _grads(call, leaves, {i})
        assert torch.equal(y, z) and torch.equal(one, full[i])


@pytest.mark.parametrize("name", NAMES)
def test_a_graph_used_twice_and_accumulated(name):
    call, leaves = _case(name)
    leaves = [t.detach().clone().requires_grad_(True) for t in leaves]
    y = call(*leaves)
    dy = torch.ones_like(y)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    second = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    for _ in range(2):
        call(*leaves).backward(dy)
    assert all(torch.equal(t.grad, (g + g)) for t, g in zip(leaves, first))


@pytest.mark.parametrize("name", NAMES)
def test_what_is_saved_may_be_kept_elsewhere(name):
    from torch.utils.checkpoint import checkpoint
    call, leaves = _case(name)
    y, full = _grads(call, leaves)
    with torch.autograd.graph.save_on_cpu():
        z, other = _grads(call, leaves)
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(full, other))
    z, other = _grads(lambda *t: checkpoint(call, *t, use_reentrant=False), leaves)
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(full, other))


@pytest.mark.parametrize("name", NAMES)
def test_without_gradients(name):
    call, leaves = _case(name)
    y, _ = _grads(call, leaves)
    with torch.no_grad():
        z = call(*[t.requires_grad_(True) for t in leaves])
    assert torch.equal(y, z) and not z.requires_grad
    with torch.inference_mode():
        assert torch.equal(y, call(*[t.clone() for t in leaves]))


@pytest.mark.parametrize("name", NAMES)
def test_no_tokens(name):
    call, leaves = _case(name, tokens=0)
    y, grads = _grads(call, leaves)
    assert y.numel() == 0
    for t, g in zip(leaves, grads):
        assert g.shape == t.shape and (g == 0).all()


@pytest.mark.parametrize("name", NAMES)
def test_changes_in_place_are_noticed(name):
    call, leaves = _case(name)
    leaves = [t.detach().clone().requires_grad_(True) for t in leaves]
    y = call(*leaves)
    if name in ("gather", "embed"):  # nothing of the rows is needed for their gradient
        return
    with torch.no_grad():
        leaves[0].mul_(2)
    with pytest.raises(RuntimeError):
        y.sum().backward()
