"""Tokens sorted by expert and back, and the experts' products over them, against 64 bits."""

import pytest
import torch

from _products import ACTS, Product, close, half_step, tiny

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _ids(tokens, k, experts, none=0.0, dtype=torch.int64, seed=0, skew=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    like = torch.randn(tokens, experts, device="cuda", generator=g) + skew * torch.randn(experts, device="cuda", generator=g)
    ids = like.topk(min(k, experts), -1).indices
    if k > experts:
        ids = torch.cat((ids, ids[:, :1].expand(tokens, k - experts)), 1)
    gone = torch.rand(tokens, k, device="cuda", generator=g) < none
    far = torch.where(torch.rand(tokens, k, device="cuda", generator=g) < 0.5, -1, experts + 5)
    return torch.where(gone, far, ids).to(dtype)


def _order(ids, experts):
    flat = ids.flatten().long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    by, pairs = torch.sort(key, stable=True)
    places = torch.empty_like(pairs)
    places[pairs] = torch.arange(pairs.numel(), device=ids.device)
    return pairs, places.view(ids.shape), torch.searchsorted(by, torch.arange(experts + 1, device=ids.device))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (1, 8, 64), (5, 3, 7), (64, 8, 64), (1000, 2, 512), (1024, 4, 40), (1025, 4, 5), (1024, 8, 40),
                                              (1025, 8, 5), (3001, 3, 512), (40000, 4, 129), (70000, 8, 64), (9000, 1, 1)])
def test_order(tokens, k, experts, dtype):
    from tao_memory_b200 import sort_tokens
    for none, skew in ((0.0, 1.0), (0.3, 0.0), (1.0, 0.0), (0.01, 30.0)):
        ids = _ids(tokens, k, experts, none, dtype, seed=tokens, skew=skew)
        order = sort_tokens(ids, experts)
        pairs, places, offsets = _order(ids, experts)
        assert torch.equal(order.pairs.long(), pairs) and torch.equal(order.places.long(), places)
        assert torch.equal(order.offsets.long(), offsets)
        assert order.pairs.dtype == order.places.dtype == order.offsets.dtype == torch.int32
        assert (order.tokens, order.top_k, order.experts) == (tokens, k, experts)


def test_order_of_views_and_of_nothing():
    from tao_memory_b200 import gather_tokens, return_tokens, sort_tokens
    ids = _ids(500, 8, 30)
    for view in (ids[::3, 1::2], ids.T[:4], ids[:, :1]):
        assert torch.equal(sort_tokens(view, 30).pairs, sort_tokens(view.contiguous(), 30).pairs)
    order = sort_tokens(ids[:0], 30)
    assert order.pairs.numel() == 0 and (order.offsets == 0).all() and order.offsets.shape == (31,)
    x = torch.empty(0, 64, device="cuda")
    assert gather_tokens(x, order).shape == (0, 64) and return_tokens(x, order).shape == (0, 64)
    huge = torch.tensor([[2 ** 33 + 1, 1], [-2 ** 40, 0]], device="cuda")
    assert sort_tokens(huge, 2).offsets.tolist() == [0, 1, 2]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,experts,width", [(1, 1, 4, 64), (3, 2, 2, 1), (64, 8, 64, 768), (77, 3, 9, 130),
                                                    (500, 4, 12, 1001), (33, 11, 40, 4104), (2000, 2, 100, 72)])
@pytest.mark.parametrize("weighted", ["fp32", "same", None])
def test_gather_and_return(tokens, k, experts, width, dtype, weighted):
    from tao_memory_b200 import gather_tokens, return_tokens, sort_tokens
    ids = _ids(tokens, k, experts, none=0.1, seed=width)
    order = sort_tokens(ids, experts)
    pairs, places, offsets = _order(ids, experts)
    g = torch.Generator(device="cuda").manual_seed(7)
    x, dy = (torch.randn(tokens, width, device="cuda", generator=g).to(dtype) for _ in range(2))
    ys, dxs = (torch.randn(tokens * k, width, device="cuda", generator=g).to(dtype) for _ in range(2))
    w = None
    if weighted:
        w = torch.rand(tokens, k, device="cuda", generator=g).to(torch.float32 if weighted == "fp32" else dtype)
    for t in (x, ys, w):
        if t is not None:
            t.requires_grad_(True)
    xs, y = gather_tokens(x, order), return_tokens(ys, order, w)
    assert torch.equal(xs.detach(), x.detach()[pairs // k])
    has = (ids >= 0) & (ids < experts)
    wide = torch.where(has, torch.ones_like(has).double() if w is None else w.detach().double(), 0.0)
    at = ys.detach().double()[places]
    u, f = half_step(dtype), 2.0 ** -24
    want = (wide.unsqueeze(-1) * at).sum(1)
    off = (k + 1) * f * (wide.unsqueeze(-1) * at).abs().sum(1)
    close(y.detach(), want, off + u * (want.abs() + off) + tiny(dtype), "y")
    leaves = [t for t in (x, ys, w) if t is not None]
    grads = torch.autograd.grad((xs, y), leaves, (dxs, dy))
    want = dxs.double()[places].sum(1)
    off = k * f * dxs.double()[places].abs().sum(1)
    close(grads[0], want, off + u * (want.abs() + off) + tiny(dtype), "dx")
    want = torch.zeros(tokens * k, width, device="cuda", dtype=torch.double)
    want[places.flatten()] = (wide.unsqueeze(-1) * dy.double().unsqueeze(1)).view(-1, width)
    close(grads[1], want, (u + f) * want.abs() + tiny(dtype), "dys")
    if w is not None:
        terms = torch.where(has.unsqueeze(-1), at * dy.double().unsqueeze(1), 0.0)
        want, uw = terms.sum(-1), half_step(w.dtype)
        off = (width + 1) * f * terms.abs().sum(-1)
        close(grads[2], want, off + uw * (want.abs() + off) + tiny(w.dtype), "dw")


def test_rows_apart_and_off_their_alignment():
    from tao_memory_b200 import gather_tokens, return_tokens, sort_tokens
    ids = _ids(60, 3, 8)
    order = sort_tokens(ids, 8)
    base = torch.randn(180, 400, device="cuda").bfloat16()
    for view in (base[:, 8:264], base[:, 3:99], base.T[:180, :180], base[:1, :64].expand(180, 64), base.flip(0)[:, :128]):
        plain = view.contiguous()
        assert torch.equal(gather_tokens(view[:60], order), gather_tokens(plain[:60], order))
        assert torch.equal(return_tokens(view, order), return_tokens(plain, order))


def test_pairs_of_no_expert_do_not_count():
    from tao_memory_b200 import return_tokens, sort_tokens
    ids = _ids(40, 4, 6, none=0.5)
    order = sort_tokens(ids, 6)
    ys = torch.randn(160, 32, device="cuda")
    ys[int(order.offsets[-1]):] = float("nan")
    w = torch.rand(40, 4, device="cuda")
    w[~((ids >= 0) & (ids < 6))] = float("nan")
    ys.requires_grad_(True), w.requires_grad_(True)
    y = return_tokens(ys, order, w)
    dys, dw = torch.autograd.grad(y, (ys, w), torch.randn_like(y))
    assert not y.isnan().any() and not dys.isnan().any() and not dw.isnan().any()
    assert (dys[int(order.offsets[-1]):] == 0).all()


def test_orders_made_elsewhere_and_what_is_refused():
    """An order of a caller's own (places outside of the pairs are passed over), and the Python calls' refusals."""
    from tao_memory_b200 import TokenOrder, expert_linear, gather_tokens, return_tokens, sort_tokens
    ids = _ids(50, 3, 7)
    made = sort_tokens(ids, 7)
    order = TokenOrder(made.pairs, made.places.clone(), made.offsets)
    order.places[3, 1], order.places[4, 0] = -5, 2 ** 31 - 1
    ys = torch.randn(150, 40, device="cuda")
    full, part = return_tokens(ys, made), return_tokens(ys, order)
    keep = torch.ones(50, dtype=torch.bool, device="cuda")
    keep[3] = keep[4] = False
    assert torch.equal(full[keep], part[keep]) and not torch.equal(full[3], part[3])
    x = torch.randn(50, 40, device="cuda")
    same = gather_tokens(x, order) == gather_tokens(x, made)
    missed = made.places[[3, 4], [1, 0]].long()
    same[missed] = True
    assert same.all()
    for kept in (-1, -2 ** 31, 0, 2 ** 31 - 1):  # the number of pairs that have an expert is held within them
        offsets = made.offsets.clone()
        offsets[-1] = kept
        leaf = ys.clone().requires_grad_(True)
        y = return_tokens(leaf, TokenOrder(made.pairs, made.places, offsets))
        dys, = torch.autograd.grad(y.sum(), leaf)
        assert torch.equal(y.detach(), full if kept > 0 else torch.zeros_like(full))
        assert (dys == (1 if kept > 0 else 0)).all()
    w, offsets = torch.randn(7, 8, 40, device="cuda").bfloat16(), made.offsets
    rows = ys.bfloat16()
    for bad in (lambda: sort_tokens(ids.float(), 7), lambda: sort_tokens(ids[0], 7), lambda: sort_tokens(ids, 0),
                lambda: sort_tokens(ids, 513), lambda: sort_tokens(ids[:, :0], 7), lambda: gather_tokens(x[:49], made),
                lambda: gather_tokens(x.double(), made), lambda: gather_tokens(x, made.places), lambda: return_tokens(x, made),
                lambda: return_tokens(ys, made, torch.ones(50, 2, device="cuda")),
                lambda: return_tokens(ys, made, torch.ones(50, 3, device="cuda").half()),
                lambda: return_tokens(ys, made, torch.ones(50, 3)), lambda: return_tokens(ys[:, :0], made),
                lambda: TokenOrder(made.pairs, made.places.long(), offsets), lambda: TokenOrder(made.pairs, made.places.T, offsets),
                lambda: TokenOrder(made.pairs[:9], made.places, offsets),
                lambda: expert_linear(rows, w, offsets.long()), lambda: expert_linear(rows, w, offsets[1:]),
                lambda: expert_linear(rows, w[0], offsets), lambda: expert_linear(rows, w.half(), offsets),
                lambda: expert_linear(rows[:, 1:], w, offsets), lambda: expert_linear(rows, w, offsets, up=w[:, 1:]),
                lambda: expert_linear(rows, w, offsets, activation="tanh"), lambda: expert_linear(ys, w.float(), offsets),
                lambda: expert_linear(rows[None], w, offsets)):
        with pytest.raises(ValueError):
            bad()


def test_what_was_saved_is_not_changed_in_between():
    from tao_memory_b200 import return_tokens, sort_tokens
    order = sort_tokens(_ids(20, 2, 4), 4)
    ys = torch.randn(40, 8, device="cuda", requires_grad=True)
    y = return_tokens(ys, order, torch.ones(20, 2, device="cuda"))
    order.places.add_(0)
    with pytest.raises(RuntimeError):
        y.sum().backward()


# -- the experts' products ----------------------------------------------------
def _check_experts(x, w, up, offsets, name, dy, grad=True):
    from tao_memory_b200 import expert_linear
    leaves = [None if t is None else t.detach().clone().requires_grad_(True) for t in (x, w, up)]
    with torch.no_grad():
        y = expert_linear(leaves[0], leaves[1], offsets, up=leaves[2], activation=name)
    used = [t for t in leaves if t is not None]
    got = {}
    if grad:
        again = expert_linear(leaves[0], leaves[1], offsets, up=leaves[2], activation=name)
        assert torch.equal(y, again.detach())
        got = dict(zip(("dx", "dw") + (() if up is None else ("dup",)), torch.autograd.grad(again, used, dy)))
    limits = offsets.tolist()
    assert (y[limits[-1]:] == 0).all()
    for e in range(w.shape[0]):
        at = slice(limits[e], limits[e + 1])
        if limits[e] == limits[e + 1]:
            assert all((got[k][e] == 0).all() for k in ("dw", "dup") if k in got)
            continue
        want = Product(x[at], w[e], x.dtype, up=None if up is None else up[e], name=name)
        close(y[at], want.y, want.y_off, "y")
        if grad:
            ref = want.backward(dy[at])
            close(got["dx"][at], *ref["dx"], "dx")
            for key in ("dw", "dup"):
                if key in got:
                    close(got[key][e], *ref[key], key)
    if grad:
        assert (got["dx"][limits[-1]:] == 0).all()


def _experts_case(counts, none, k, n, dtype, gated, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    offsets = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    rows, e = sum(counts) + none, len(counts)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    return (normal(rows, k), normal(e, n, k, scale=k ** -0.5), normal(e, n, k, scale=k ** -0.5) if gated else None, offsets,
            normal(rows, n))


COUNTS = [([1], 0), ([0, 5, 0, 0], 0), ([3, 0, 200, 64, 1], 9), ([300, 129, 0, 128, 127], 70), ([0, 0, 0], 4),
          ([2] * 40, 3), ([700, 1], 0), ([65, 63, 16, 17], 200)]


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("counts,none", COUNTS + [([30, 50, 41, 0], 8), ([90, 33, 64, 1], 0), ([70] * 5, 0)])
def test_experts(counts, none, gated, dtype):
    for k, n in ((64, 64), (136, 264), (1000, 130), (33, 7)):
        x, w, up, offsets, dy = _experts_case(counts, none, k, n, dtype, gated, seed=k)
        _check_experts(x, w, up, offsets, "silu" if gated else None, dy)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("gated", [True, False])
def test_experts_activations(name, gated):
    for counts in ([90, 0, 7], [200, 300]):
        _check_experts(*_experts_case(counts, 5, 72, 136, torch.bfloat16, gated)[:4], name,
                       _experts_case(counts, 5, 72, 136, torch.bfloat16, gated)[4])


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dtype", TYPES[:2])
def test_experts_by_pairs_of_blocks(dtype, gated):
    """Experts of many rows, some whose last pair has one block's rows or fewer, one without any, rows of none."""
    x, w, up, offsets, dy = _experts_case([2600, 0, 1300, 2501, 130, 1], 77, 1032, 2600, dtype, gated, seed=3)
    _check_experts(x, w, up, offsets, "silu" if gated else None, dy)


def test_512_experts():
    g = torch.Generator().manual_seed(1)
    counts = torch.randint(0, 9, (512,), generator=g).tolist()
    for gated in (True, False):
        x, w, up, offsets, dy = _experts_case(counts, 11, 64, 72, torch.bfloat16, gated)
        _check_experts(x, w, up, offsets, "silu" if gated else None, dy)


def test_strides_of_experts():
    x, w, up, offsets, dy = _experts_case([60, 0, 41, 9], 3, 96, 80, torch.bfloat16, True)
    both = torch.cat((w, up), 1)  # gate and up in one tensor
    wide = torch.cat((x, x), 1)
    _check_experts(wide[:, 96:], both[:, :80], both[:, 80:], offsets, "silu", dy)
    _check_experts(wide[:, 1:97], both.transpose(0, 1)[:80].transpose(0, 1), both[:, 80:], offsets, "silu", dy)
    _check_experts(x, w.transpose(1, 2).contiguous().transpose(1, 2), up[:1].expand(4, 80, 96), offsets, "silu", dy)


@pytest.mark.parametrize("counts", [[40, 21, 1], [300, 77, 129]])
def test_rows_keep_to_their_expert(counts):
    """An infinite row changes neither another expert's rows nor its weights' gradient."""
    from tao_memory_b200 import expert_linear
    x, w, up, offsets, dy = _experts_case(counts, 20, 64, 72, torch.bfloat16, True)

    def all_(x, dy):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, up)]
        y = expert_linear(leaves[0], leaves[1], offsets, up=leaves[2], activation="silu")
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    clean = all_(x, dy)
    first, end = counts[0], sum(counts)
    bad_x, bad_dy = x.clone(), dy.clone()
    bad_x[first:first + counts[1]] = float("inf")
    bad_dy[first:first + counts[1]] = float("nan")
    bad_x[end:], bad_dy[end:] = float("nan"), float("inf")
    for i, (a, b) in enumerate(zip(clean, all_(bad_x, bad_dy))):
        if i < 2:  # rows
            assert torch.equal(a[:first], b[:first]) and torch.equal(a[first + counts[1]:], b[first + counts[1]:])
        else:
            assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("bad", [[0, -5, 20, 30], [0, 20, 10, 30], [7, 9, 2 ** 30, 5], [0, 10, 500, 2 ** 31 - 1],
                                 [0, -2 ** 31, 3, 3]])
def test_offsets_that_are_none(bad):
    """Offsets out of order are held between their neighbours and the rows: nothing out of range is read or written."""
    from tao_memory_b200 import expert_linear
    x, w, up, _, dy = _experts_case([30, 30, 30], 0, 64, 72, torch.bfloat16, True)
    offsets = torch.tensor(bad, device="cuda", dtype=torch.int32)
    held, last = [0], 0
    for v in bad[1:]:
        last = max(last, min(max(v, 0), 90))
        held.append(last)
    for t in (offsets, torch.tensor(held, device="cuda", dtype=torch.int32)):
        leaves = [v.detach().clone().requires_grad_(True) for v in (x, w, up)]
        y = expert_linear(leaves[0], leaves[1], t, up=leaves[2], activation="silu")
        outs = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
        if t is offsets:
            first = outs
    assert all(torch.equal(a, b) for a, b in zip(first, outs))


# -- together ---------------------------------------------------------------------
def _layer(x, ids, p, gate, up, down, experts):
    from tao_memory_b200 import expert_linear, gather_tokens, return_tokens, sort_tokens
    order = sort_tokens(ids, experts)
    h = expert_linear(gather_tokens(x, order), gate, order.offsets, up=up, activation="silu")
    return return_tokens(expert_linear(h, down, order.offsets), order, p)


def _layer_inputs(tokens, width, inner, experts, k, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).bfloat16()

    ids = _ids(tokens, k, experts, none=0.1, seed=seed)
    p = torch.rand(tokens, k, device="cuda", generator=g)
    return (normal(tokens, width), ids, p, normal(experts, inner, width, scale=width ** -0.5),
            normal(experts, inner, width, scale=width ** -0.5), normal(experts, width, inner, scale=inner ** -0.5), experts)


def test_a_layer_of_experts():
    """The four together against 64 bits, token by token's choices."""
    x, ids, p, gate, up, down, experts = _layer_inputs(300, 128, 96, 10, 3)
    leaves = [t.requires_grad_(True) for t in (x, p, gate, up, down)]
    y = _layer(x, ids, p, gate, up, down, experts)
    dy = torch.randn_like(y)
    grads = torch.autograd.grad(y, leaves, dy)
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    ref = torch.zeros(300, 128, device="cuda", dtype=torch.double)
    for e in range(experts):
        share = (wide[1] * (ids == e)).sum(-1, keepdim=True)
        h = torch.nn.functional.silu(wide[0] @ wide[2][e].T) * (wide[0] @ wide[3][e].T)
        ref = ref + share * (h @ wide[4][e].T)
    # h, the experts' outputs and y are rounded (2^-8 each at most, of random sign: rms 2^-8 / sqrt 3), the gradient's
    # rows five times more; the norm of the error is below sqrt(8) roundings' maximum
    limit = 8 ** 0.5 * 2.0 ** -8
    assert (y.double() - ref).norm() <= limit * ref.norm()
    for a, b in zip(grads, torch.autograd.grad(ref, wide, dy.double())):
        assert (a.double() - b).norm() <= limit * b.norm()


def test_a_captured_layer_and_on_other_streams():
    x, ids, p, gate, up, down, experts = _layer_inputs(2000, 128, 64, 12, 2)
    leaves = [t.requires_grad_(True) for t in (x, p, gate, up, down)]
    dy = torch.randn(2000, 128, device="cuda").bfloat16()

    def step():
        y = _layer(x, ids, p, gate, up, down, experts)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)  # no eager graph outlives a captured one's start

    first = step()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(step())
    torch.cuda.synchronize()
    for other in outs:
        assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        ids.copy_(_ids(2000, 2, experts, none=0.3, seed=9))  # other choices in the same graph
        x.mul_(1.25)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, step()))


def test_no_wait_ran_out():
    from tao_memory_b200.stream import check_device
    assert check_device() == 0
