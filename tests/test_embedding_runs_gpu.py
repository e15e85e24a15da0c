"""The embedding's gradient at the edges of its runs of 16 sorted tokens: one run and two (the first that are joined), words
that are exactly one run or meet on a run's border, and words of as many runs as one warp joins and one more."""

import math

import pytest
import torch

from _products import close, half_step, tiny

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(ids, vocab, width, dtype, scale=1.0, seed=0):
    from tao_memory_b200 import embed
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = ids.cuda()
    table = torch.zeros(vocab, width, device="cuda", dtype=dtype, requires_grad=True)
    dy = torch.randn(len(ids), width, device="cuda", generator=g).to(dtype)
    got, = torch.autograd.grad(embed(ids, table, scale), table, dy)
    has = (ids >= 0) & (ids < vocab)
    sums, sizes = (torch.zeros(vocab, width, device="cuda", dtype=torch.double) for _ in range(2))
    sums.index_add_(0, ids[has], dy[has].double())
    sizes.index_add_(0, ids[has], dy[has].double().abs())
    # a word of m tokens lies in up to m / 16 + 2 runs: 15 additions in one, then one for each other run (up to nine) or
    # those of a 32nd of the runs and 31 more, and the scaling; 2^-24 of the terms' magnitudes each
    runs = int(torch.bincount(ids[has], minlength=1).max()) // 16 + 2
    steps = 16 + (runs if runs <= 10 else math.ceil(runs / 32) + 32)
    off = abs(scale) * sizes * steps * 2.0 ** -24
    want, u = sums * scale, half_step(dtype)
    close(got, want, off + u * (want.abs() + off) + tiny(dtype), (len(ids), vocab, width))
    assert (got[sizes[:, 0] == 0] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [64, 33])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 143, 144, 145, 160, 161])
def test_one_word_and_two_that_meet(n, width, dtype):
    at = torch.arange(n)
    _check(torch.zeros(n, dtype=torch.long), 3, width, dtype)
    for border in (1, 15, 16, 17, 32, n - 16, n - 1):
        if 0 < border < n:
            _check((at >= border).long() * 2, 3, width, dtype, scale=0.5, seed=border)
            _check((at >= border).long() * 3, 3, width, dtype)  # the second is padding, behind all words


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [15, 16, 17, 32, 48, 144, 160, 176])
def test_words_of_whole_runs(length, dtype):
    """Every word as long as the next; of 16 tokens each is a run of its own and none is joined."""
    for n in (16 * length, 20 * length, 20 * length + 5):
        ids = torch.arange(n) // length
        _check(ids, int(ids.max()) + 2, 72, dtype)
        order = torch.randperm(n, generator=torch.Generator().manual_seed(n))
        _check(ids[order], int(ids.max()) + 2, 72, dtype, scale=3.0)


def test_words_of_two_lengths_by_turns():
    """One of 1 to 20 runs, then one that brings the next to any place of a run."""
    for runs in (1, 2, 8, 9, 10, 20):
        for rest in (1, 8, 15, 16):
            lengths = torch.tensor([16 * runs, rest] * 9)
            ids = torch.repeat_interleave(torch.arange(18), lengths)
            _check(ids, 18, 40, torch.bfloat16)
