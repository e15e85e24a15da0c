"""ServedBlock: the block's parts in their order, bit by bit against the same calls made one by
one, and the whole against a plain composition in fp32 around the operator's own attention."""
import os
import runpy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _block(heads=2, width=64, inner=96, experts=6, top_k=2):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_blocks.py")
    example = runpy.run_path(path)
    return example["make_block"](heads, width, inner, experts, top_k, seed=7), example["main"]


def _state(tb):
    from tao_memory_b200.presets import index_only_page_memo
    return tb.new_state(0, index_only_page_memo())


@pytest.mark.parametrize("tokens,first", [(1, True), (3, False)])
def test_step_is_its_parts(tokens, first):
    import tao_memory_b200 as tb
    from tao_memory_b200.model import split_norm
    block, _ = _block()
    torch.manual_seed(1)
    states = [[_state(tb) for _ in range(tokens)] for _ in range(2)]
    prompts = [torch.randn(830, 128, device="cuda").bfloat16() for _ in range(tokens)]
    for same in states:
        for state, prompt in zip(same, prompts):
            block.prefill(prompt, None, state)
    x = torch.randn(tokens, 128, device="cuda").bfloat16()
    stream = None if first else torch.randn(tokens, 128, device="cuda").bfloat16()
    y, s = block.step(x, stream, states[0])
    with torch.no_grad():
        h, s1 = tb.add_rms_norm(x, block.norms[0], stream)
        q, k, v, raw_q, raw_k = split_norm(tb.linear4(h, block.qkv).view(tokens, 1, -1), 2, 64)
        att, _ = tb.tao_attention_decode_batch(q, k, v, raw_q=raw_q, raw_k=raw_k, fusion_a=block.fusion_a,
                                               fusion_b=block.fusion_b, alpha=block.alpha, states=states[1])
        o = tb.linear4(att.view(tokens, 128), block.out)
        h2, s2 = tb.add_rms_norm(o, block.norms[1], s1)
        z, ids, weights = tb.expert_layer(h2, block.experts, return_routing=True)
    assert torch.equal(s, s2) and torch.equal(y, z)
    # each part against its plain form on the same input: one bf16 rounding (2^-8) and fp32 sums
    plain = lambda t, w: t.float() * (t.float().square().mean(-1, keepdim=True) + block.eps).rsqrt() * w.float()
    near = lambda a, b: ((a.float() - b).norm() <= 2.0 ** -8 * b.norm())
    assert torch.equal(s1, x if first else x + stream) and near(h, plain(s1, block.norms[0]))
    assert near(o, att.view(tokens, 128).float() @ block.out.dequantize().T)
    assert torch.equal(s2, o + s1) and near(h2, plain(s2, block.norms[1]))
    gate, up, down = (w.dequantize() for w in (block.experts.gate, block.experts.up, block.experts.down))
    want = torch.zeros_like(h2, dtype=torch.float32)
    for t in range(tokens):
        for e, p in zip(ids[t].tolist(), weights[t]):
            a = h2[t].float()
            want[t] += p * (down[e] @ (torch.nn.functional.silu(gate[e] @ a) * (up[e] @ a)))
    assert near(z, want)


def test_prefill_then_step_equals_steps():
    """A prompt taken as one chunk and token by token: the same states and outputs up to the
    rounding of the attention's two kernels (bf16, |a-b| <= 5e-2 of the outputs' scale)."""
    import tao_memory_b200 as tb
    block, _ = _block()
    torch.manual_seed(2)
    x = torch.randn(40, 128, device="cuda").bfloat16()
    a, b = _state(tb), _state(tb)
    ya, _ = block.prefill(x, None, a)
    yb = torch.cat([block.step(x[i:i + 1], None, [b])[0] for i in range(40)])
    assert a.position == b.position == 40
    # a token whose routing is nearly tied may take another expert: rare, so by the median
    off = (ya.float() - yb.float()).norm(dim=-1) / yb.float().norm(dim=-1)
    assert off.median() <= 5e-2


def test_example_runs():
    _, main = _block()
    out = main(requests=2, prompt=900, tokens=4, heads=2)
    assert out.shape == (2, 128) and torch.isfinite(out.float()).all()


def test_refusals():
    from tao_memory_b200.model import ServedBlock
    block, _ = _block()
    args = (block.fusion_a, block.fusion_b, 0.5)
    for bad in (lambda: ServedBlock(2, 64, block.out, block.out, block.norms, block.experts, *args),
                lambda: ServedBlock(2, 64, block.qkv, block.out, block.norms[:1], block.experts, *args),
                lambda: ServedBlock(1, 64, block.qkv, block.out, block.norms, block.experts, *args)):
        with pytest.raises(ValueError):
            bad()
