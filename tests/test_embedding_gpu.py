"""``embed`` and its gradient against 64 bits."""

import pytest
import torch

from _products import close, half_step, tiny

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(ids, table, scale, dy):
    from tao_memory_b200 import embed
    dtype, u = table.dtype, half_step(table.dtype)
    vocab, width = table.shape
    leaf = table.detach().requires_grad_(True)
    y = embed(ids, leaf, scale)
    assert y.shape == (*ids.shape, width) and y.dtype == dtype
    flat = ids.flatten().long()
    has = (flat >= 0) & (flat < vocab)
    want = torch.where(has.unsqueeze(-1), table.detach().double()[flat.clamp(0, vocab - 1)] * scale, 0.0)
    close(y.detach().reshape(-1, width), want, (u + 2.0 ** -23) * want.abs() + tiny(dtype), "y")
    got, = torch.autograd.grad(y, leaf, dy)
    sums, sizes = (torch.zeros(vocab, width, device="cuda", dtype=torch.double) for _ in range(2))
    rows = dy.double().reshape(-1, width)
    sums.index_add_(0, flat[has], rows[has])
    sizes.index_add_(0, flat[has], rows[has].abs())
    most = int(torch.bincount(flat[has]).max()) if has.any() else 1
    off = abs(scale) * sizes * (min(most, 64) + most / 64 + 3) * 2.0 ** -24  # runs of 64, then the runs
    want = sums * scale
    assert got.shape == table.shape and got.dtype == dtype
    close(got, want, off + u * (want.abs() + off) + tiny(dtype), "dtable")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 50000, 64), (5, 7, 768), (64, 3, 130), (65, 3, 130), (1000, 511, 257),
                                           (3000, 512, 72), (8192, 40, 64), (8193, 40, 64), (20000, 70000, 96),
                                           (5000, 300000, 8), (700, 128, 4104)])
def test_sizes(n, vocab, width, dtype):
    g = torch.Generator(device="cuda").manual_seed(n)
    table, dy = (torch.randn(s, width, device="cuda", generator=g).to(dtype) for s in (vocab, n))
    for id_type in (torch.int64, torch.int32):
        ids = torch.randint(0, vocab, (n,), device="cuda", generator=g).to(id_type)
        _check(ids, table, 1.0 if id_type == torch.int64 else 2.5, dy)


@pytest.mark.parametrize("share", [0.02, 0.5, 0.98, 1.0])
def test_one_word_many_times(share):
    """Ids that go on over many runs, from their first token to their last, and padding."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n, vocab, width = 10000, 900, 200
    table, dy = (torch.randn(s, width, device="cuda", generator=g).bfloat16() for s in (vocab, n))
    for word in (0, 450, vocab - 1, -1):
        ids = torch.randint(0, vocab, (n,), device="cuda", generator=g)
        ids[torch.rand(n, device="cuda", generator=g) < share] = word
        _check(ids, table, 1.0, dy)
    sorted_ids = torch.arange(n, device="cuda") // 64  # every word a whole run
    _check(sorted_ids, table, 1.0, dy)


@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 768), (torch.float16, 301), (torch.float32, 260)])
@pytest.mark.parametrize("least,most", [(100, 200), (130, 400), (300, 900), (16, 5000)])
def test_long_words_one_after_the_other(least, most, dtype, width):
    """Words of many lengths, so that their first and last tokens lie anywhere among the runs that join them."""
    g = torch.Generator(device="cuda").manual_seed(least)
    vocab = 120
    lengths = torch.randint(least, most + 1, (vocab,), device="cuda", generator=g)
    lengths[::3] = lengths[::3] // 16 * 16  # and on their borders
    ids = torch.repeat_interleave(torch.arange(vocab, device="cuda"), lengths)
    ids = ids[torch.randperm(len(ids), device="cuda", generator=g)]
    table, dy = (torch.randn(s, width, device="cuda", generator=g).to(dtype) for s in (vocab, len(ids)))
    _check(ids, table, 1.0, dy)
    _check(torch.cat([ids, ids.new_full((777,), vocab)]), table, 1.0, torch.cat([dy, dy[:777]]))


def test_shapes_and_views():
    table = torch.randn(300, 200, device="cuda").bfloat16()
    ids = torch.randint(-2, 110, (6, 10), device="cuda")
    for t in (table[:100, 8:72], table[::3, 3:67], table.T[:100, :64], table[:1, :64].expand(100, 64)):
        dy = torch.randn(10, 6, 64, device="cuda").bfloat16().transpose(0, 1)
        _check(ids, t, 0.5, dy)
        _check(ids.T, t, 0.5, dy.transpose(0, 1))
    from tao_memory_b200 import embed
    leaf = table.clone().requires_grad_(True)
    y = embed(ids[:, :0], leaf)
    y.sum().backward()
    assert y.shape == (6, 0, 200) and (leaf.grad == 0).all()
    one = embed(torch.tensor(7, device="cuda"), table)
    assert torch.equal(one, table[7])
    leaf.grad = None
    embed(ids, leaf).sum().backward()  # a broadcast gradient
    counts = torch.bincount(ids[(ids >= 0)].flatten(), minlength=300)
    assert torch.equal(leaf.grad, counts.bfloat16().unsqueeze(1).expand(300, 200))


def test_ids_that_are_none():
    from tao_memory_b200 import embed
    table = torch.randn(10, 64, device="cuda")
    ids = torch.tensor([-1, 10, 2 ** 40 + 3, -2 ** 50, 9, 2 ** 32], device="cuda")
    y = embed(ids, table)
    assert (y[[0, 1, 2, 3, 5]] == 0).all() and torch.equal(y[4], table[9])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1, 5, 8])
@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 3, 5), (2, 700, 129), (4096, 600, 64), (4097, 33, 7), (40000, 300000, 24),
                                           (9, 40001, 1031)])
def test_gradient_fills_the_table_and_no_more(n, vocab, width, offset, dtype):
    """Every row of a table that held NaN, from any element on, and nothing before or behind it."""
    from tao_memory_b200 import _lib
    from tao_memory_b200.norm import TYPES as CODES
    g = torch.Generator(device="cuda").manual_seed(n)
    ids = torch.randint(-1, vocab, (n,), device="cuda", generator=g)
    dy = torch.ones(n, width, device="cuda", dtype=dtype)
    held = torch.full((offset + vocab * width + 16,), float("nan"), device="cuda", dtype=dtype)
    table = held[offset:offset + vocab * width]
    size = _lib.lib().tao_embed_gradient_workspace_bytes(n, vocab, width)
    room = torch.empty(size, dtype=torch.uint8, device="cuda")
    _lib.on_device(0, _lib.lib().tao_embed_gradient, ids.data_ptr(), 8, n, dy.data_ptr(), width, vocab, width, CODES[dtype],
                   1.0, table.data_ptr(), room.data_ptr(), size)
    counts = torch.bincount(ids[ids >= 0], minlength=vocab).to(dtype)  # whole numbers up to 256: exact, or rounded once
    assert torch.equal(table.view(vocab, width), counts.unsqueeze(1).expand(vocab, width))
    assert held[:offset].isnan().all() and held[offset + vocab * width:].isnan().all()


def test_refusals():
    from tao_memory_b200 import embed
    table, ids = torch.randn(10, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: embed(ids.float(), table), lambda: embed(ids.cpu(), table), lambda: embed(ids, table.double()),
                lambda: embed(ids, table[0]), lambda: embed(ids, table[:0]), lambda: embed(ids.to(torch.int16), table)):
        with pytest.raises(ValueError):
            bad()
    y = embed(ids, table.requires_grad_(True))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), table, create_graph=True)


def test_same_result_again_captured_and_on_other_streams():
    from tao_memory_b200 import embed
    g = torch.Generator(device="cuda").manual_seed(4)
    table = torch.randn(5000, 128, device="cuda", generator=g).bfloat16().requires_grad_(True)
    ids = (torch.rand(20000, device="cuda", generator=g) ** 8 * 5000).long()
    dy = torch.randn(20000, 128, device="cuda", generator=g).bfloat16()

    def step():
        y = embed(ids, table, 3.0)
        return (y.detach(),) + torch.autograd.grad(y, table, dy)  # no eager graph outlives a captured one's start

    first = step()
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            outs.append(step())
    torch.cuda.synchronize()
    for other in outs:
        assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    ids.copy_(ids.flip(0) // 2)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, step()))
