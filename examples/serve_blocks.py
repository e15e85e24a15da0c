"""A few requests through a small served model: two ``ServedBlock`` (residual norms, 4-bit
projections, Tao attention, 4-bit experts), prompts prefilled one by one, then decoded together.

    python examples/serve_blocks.py
"""

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from tao_memory_b200 import ExpertWeights, RequestStates, quantize4
from tao_memory_b200.model import ServedBlock
from tao_memory_b200.presets import index_only_page_memo
from tao_memory_b200.stream import check_device


def make_block(heads, width, inner, experts, top_k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    channels = heads * width

    def weight(*shape):
        return (torch.randn(*shape, device="cuda", generator=g) * shape[-1] ** -0.5).bfloat16()

    layer = ExpertWeights(weight(experts, channels), quantize4(weight(experts, inner, channels)),
                          quantize4(weight(experts, inner, channels)), quantize4(weight(experts, channels, inner)),
                          top_k=top_k)
    fusion = [0.02 * torch.randn(heads, width, 3, device="cuda", generator=g) for _ in range(2)]
    norms = [torch.ones(channels, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    return ServedBlock(heads, width, quantize4(weight(3 * channels, channels)), quantize4(weight(channels, channels)),
                       norms, layer, *fusion, alpha=0.5)


def main(requests=4, prompt=1000, tokens=16, heads=12, width=64):
    blocks = [make_block(heads, width, inner=512, experts=8, top_k=2, seed=i) for i in range(2)]
    states = [RequestStates(len(blocks), index_only_page_memo()) for _ in range(requests)]
    torch.manual_seed(0)
    last = []
    for request in states:
        x, stream = torch.randn(prompt, heads * width, device="cuda").bfloat16(), None
        for block, state in zip(blocks, request.layers):
            x, stream = block.prefill(x, stream, state)
        last.append((x + stream)[-1:])
    x = torch.cat(last)
    for _ in range(tokens):
        stream = None
        for layer, block in enumerate(blocks):
            x, stream = block.step(x, stream, [request[layer] for request in states])
        x = x + stream  # in place of the model's head and embedding
        x = x / x.float().square().mean(-1, keepdim=True).sqrt().to(x.dtype)
    check_device()
    print(f"{requests} requests at position {states[0].positions[0]}, output rms {x.float().square().mean().sqrt():.4f}")
    return x


if __name__ == "__main__":
    main()
