"""A small decoder trained for a few steps and decoded from as it is: an embedding, a block with experts and a
dense one around the Tao attention, all in bf16 with the library's kernels, forward and backward.

    python examples/train_blocks.py
"""

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from tao_memory_b200 import RequestStates
from tao_memory_b200.model import TrainedBlock, TrainedDecoder
from tao_memory_b200.presets import index_only_page_memo
from tao_memory_b200.stream import check_device


def make_model(vocab, heads, width, inner, experts, top_k, seed=0):
    torch.manual_seed(seed)
    config = index_only_page_memo()
    return TrainedDecoder(vocab, [TrainedBlock(heads, width, inner, experts, top_k, config=config),
                                  TrainedBlock(heads, width, inner, config=config)])


def loss_of(model, ids):
    """Cross entropy of each next token; ids [batch, tokens], -1 is padding."""
    logits = model(ids[:, :-1])
    return torch.nn.functional.cross_entropy(logits.float().flatten(0, 1), ids[:, 1:].flatten(), ignore_index=-1)


def main(vocab=1000, heads=4, width=64, batch=2, tokens=1025, steps=4, new=8):
    model = make_model(vocab, heads, width, inner=512, experts=8, top_k=2)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    ids = (torch.rand(batch, tokens, device="cuda") ** 4 * vocab).long()
    ids[-1, -tokens // 5:] = -1
    for step in range(steps):
        loss = loss_of(model, ids)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        print(f"step {step}: loss {loss.item():.4f}")
    states = [RequestStates(len(model.blocks), index_only_page_memo()) for _ in range(batch)]
    last = torch.cat([model.prefill(row[:tokens // 2], request.layers) for row, request in zip(ids, states)])
    said = []
    for _ in range(new):
        said.append(last.argmax(-1))
        last = model.step(said[-1], [request.layers for request in states])
    check_device()
    print("continued with", torch.stack(said, 1).tolist())
    return model, loss, last


if __name__ == "__main__":
    main()
