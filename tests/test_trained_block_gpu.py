"""TrainedBlock and TrainedDecoder: the block's parts in their order, its gradients against a composition in plain
torch operations around the same attention, prompts and decoding against whole sequences, the example."""
import os
import runpy

import pytest
import torch
from torch.nn import functional as F

pytestmark = pytest.mark.gpu


def _block(experts, heads=2, width=64, inner=96, seed=3, **kw):
    from tao_memory_b200.model import TrainedBlock
    from tao_memory_b200.presets import index_only_page_memo
    torch.manual_seed(seed)
    block = TrainedBlock(heads, width, inner, experts, config=index_only_page_memo(), **kw)
    with torch.no_grad():
        for p in (block.fusion_a, block.fusion_b):
            p.normal_(0, 0.02)
    return block


class _Round(torch.autograd.Function):
    """To bf16 and back; its gradient is rounded too."""

    @staticmethod
    def forward(ctx, x):
        return x.bfloat16().double()

    @staticmethod
    def backward(ctx, g):
        return g.bfloat16().double()


def _plain(block, x, stream, ids=None):
    """The block in 64 bits with the kernels' roundings between its parts; parameters are looked up by name."""
    import tao_memory_b200 as tb
    rnd = _Round.apply
    p = {k: v.detach().double().requires_grad_(True) for k, v in block.named_parameters()}

    def norm(s, w):
        return rnd(s * (s.square().mean(-1, keepdim=True) + block.eps).rsqrt() * w)

    s = x if stream is None else rnd(x + stream)
    raw_q, raw_k, v = rnd(norm(s, p["norms.0"]) @ p["qkv"].T).unflatten(-1, (3, block.heads, block.width)).unbind(2)
    q, k = (rnd(t * (t.square().mean(-1, keepdim=True) + block.eps).rsqrt()) for t in (raw_q, raw_k))
    low = [t.bfloat16() for t in (q, k, v, raw_q, raw_k)]
    att = tb.tao_attention(*low[:3], raw_q=low[3], raw_k=low[4], fusion_a=p["fusion_a"].float(),
                           fusion_b=p["fusion_b"].float(), alpha=block.alpha, config=block.config).double()
    o = rnd(att.flatten(-2) @ p["out"].T)
    s = rnd(o + s)
    h = norm(s, p["norms.1"])
    if not block.experts:
        mid = rnd(F.gelu(h @ p["first"].T + p["first_bias"]))
        return p, rnd(mid @ p["second"].T + p["second_bias"] + s), None
    rows = h.flatten(0, 1)
    probs = torch.softmax(rnd(rows @ p["router"].T), -1)
    weights = probs.gather(1, ids)
    weights = weights / weights.sum(-1, keepdim=True)
    out = 0
    for e in range(block.experts):
        mid = rnd(F.silu(rows @ p["gate"][e].T) * (rows @ p["up"][e].T))
        out = out + (weights * (ids == e)).sum(-1, keepdim=True) * rnd(mid @ p["down"][e].T)
    return p, rnd(out).view(h.shape), s


@pytest.mark.parametrize("experts,first", [(0, True), (0, False), (5, True), (5, False)])
def test_block_and_its_gradients(experts, first):
    block = _block(experts)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, stream, dy, ds = (torch.randn(2, 1100, 128, device="cuda", generator=g).bfloat16() for _ in range(4))
    x.requires_grad_(True), stream.requires_grad_(True)
    stream = None if first else stream
    chosen = []
    if experts:
        route = block.route
        block.route = lambda h: chosen.append(route(h)) or chosen[-1]
    y, s = block(x, stream)
    outs, ups = ([y], [dy]) if s is None else ([y, s], [dy, ds])
    leaves = dict(block.named_parameters(), x=x)
    if stream is not None:
        leaves["stream"] = stream
    grads = torch.autograd.grad(outs, list(leaves.values()), ups)
    wide = [None if t is None else t.detach().double().requires_grad_(True) for t in (x, stream)]
    p, ref, ref_s = _plain(block, *wide, chosen[0][0] if experts else None)
    refs = [ref] if ref_s is None else [ref, ref_s]
    p["x"] = wide[0]
    if stream is not None:
        p["stream"] = wide[1]
    wants = torch.autograd.grad(refs, [p[k] for k in leaves], [t.double() for t in ups])
    # both sides round at the same places; where their sums differ, a value may fall to the other side: one step
    # (2^-7) of few values.  The kernels' gradients keep the activation's argument and dz in bf16 too, and some go
    # on through about eight roundings, of random sign, of 2^-8 at most each.
    for a, b in zip(outs, refs):
        assert (a.detach().double() - b.detach()).norm() <= 2.0 ** -7 * b.detach().norm()
    for name, a, b in zip(leaves, grads, wants):
        assert a.shape == leaves[name].shape and a.dtype == leaves[name].dtype
        assert (a.double() - b).norm() <= 8 ** 0.5 * 2.0 ** -8 * b.norm(), name


def test_decoder_is_its_parts_and_pads():
    import tao_memory_b200 as tb
    from tao_memory_b200.model import TrainedDecoder
    blocks = [_block(4, seed=5), _block(0, seed=6)]
    model = TrainedDecoder(50, blocks)
    ids = torch.randint(0, 50, (2, 300), device="cuda")
    ids[1, 200:] = -1
    logits = model(ids)
    x, s = blocks[0](tb.embed(ids, model.table, 128 ** 0.5))
    x, s = blocks[1](x, s)
    assert s is None
    assert torch.equal(logits, tb.linear(tb.add_rms_norm(x, model.norm, s)[0], model.table))
    other = ids.clone()
    other[1, 200:] = 77  # also none
    assert torch.equal(logits, model(other))
    logits[0].float().square().mean().backward()
    grads = [p.grad.clone() for p in model.parameters()]
    assert all(g is not None and torch.isfinite(g).all() for g in grads)


@pytest.mark.parametrize("experts", [0, 4])
def test_prompt_and_steps_against_the_whole_sequence(experts):
    """Logits of a prompt and of the tokens after it, of two requests together, against whole sequences below the
    768 tokens of the attention's exact window (there streaming and training read the same keys): the same weights
    through the few rows' and the many rows' kernels and two attention kernels, by the logits' median."""
    import tao_memory_b200 as tb
    from tao_memory_b200.model import TrainedDecoder
    from tao_memory_b200.presets import index_only_page_memo
    model = TrainedDecoder(64, [_block(experts, seed=8), _block(experts, seed=9)])
    ids = torch.randint(0, 64, (2, 330), device="cuda")
    with torch.no_grad():
        whole = model(ids)
    requests = [tb.RequestStates(2, index_only_page_memo()) for _ in range(2)]
    last = torch.cat([model.prefill(row[:320], r.layers) for row, r in zip(ids, requests)])
    for t in range(320, 330):
        off = (last.float() - whole[:, t - 1].float()).norm(dim=-1) / whole[:, t - 1].float().norm(dim=-1)
        assert off.median() <= 5e-2
        last = model.step(ids[:, t], [r.layers for r in requests])


def test_example_runs():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_blocks.py")
    model, loss, last = runpy.run_path(path)["main"](vocab=90, heads=2, batch=2, tokens=901, steps=2, new=3)
    assert torch.isfinite(loss) and torch.isfinite(last.float()).all()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
