"""expert_layer against the routed sum in 64 bits.

Bound: out is rounded once (2^-8); before it the fp32 sums lose at most D = 64 units of 2^-24
of their terms' magnitudes in each of the products (see test_linear4_gpu), h has 2^-16 of
itself, and expf and the divisions a few units: with T the sum over the chosen experts of
weight * |down| (|dh|max), where |dh| <= (D + 2^-16) |h| terms: silu's slope is at most 1.1, so
dh <= 1.1 D (|gate| |x|) |up x| + D |silu| (|up| |x|) + 2^-16 |h|.  The routing weights add
2 D of the logits' magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 64 * 2.0 ** -24


def _layer(width, inner, experts, top_k, kind="bf16", group=128, zeros=False, renormalize=True, seed=0):
    from tao_memory_b200 import ExpertWeights, quantize4
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    router = (2 * n(experts, width) * width ** -0.5).bfloat16()
    ws = [(n(experts, inner, width) * width ** -0.5).bfloat16(), (n(experts, inner, width) * width ** -0.5).bfloat16(),
          (n(experts, width, inner) * inner ** -0.5).bfloat16()]
    if kind == "4bit":
        ws = [quantize4(w, group, zeros) for w in ws]
        wide = [w.dequantize().double() for w in ws]
    else:
        wide = [w.double() for w in ws]
    return ExpertWeights(router, *ws, top_k=top_k, renormalize=renormalize), router, wide


def _ref(x, router, wide, top_k, renormalize):
    """(out, bound before the rounding, ids, weights) in 64 bits."""
    xd, rd = x.double(), router.double()
    logits = xd @ rd.T
    p = torch.softmax(logits, -1)
    order = torch.sort(p, dim=-1, descending=True, stable=True)
    ids, w = order.indices[:, :top_k], order.values[:, :top_k]
    if renormalize:
        w = w / w.sum(-1, keepdim=True)
    slack = 2 * D * (xd.abs() @ rd.abs().T).amax(-1)
    out, off = torch.zeros_like(xd), torch.zeros_like(xd)
    for e in range(router.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        gate, up, down = (m[e] for m in wide)
        a, b = xd[t] @ gate.T, xd[t] @ up.T
        s = a * torch.sigmoid(a)
        h = s * b
        dh = (1.1 * D * (xd[t].abs() @ gate.abs().T) * b.abs() + D * s.abs() * (xd[t].abs() @ up.abs().T)
              + 2.0 ** -16 * h.abs())
        share = w[t, j].unsqueeze(-1)
        y = h @ down.T
        out.index_add_(0, t, share * y)
        terms = dh @ down.abs().T + D * (h.abs() @ down.abs().T) + (slack[t] + D).unsqueeze(-1) * y.abs()
        off.index_add_(0, t, share * terms)
    return out, off, ids, w


def _run(x, layer, router, wide):
    from tao_memory_b200 import expert_layer
    out, ids, w = expert_layer(x, layer, return_routing=True)
    ref, off, rid, rw = _ref(x.reshape(-1, x.shape[-1]), router, wide, layer.top_k, layer.renormalize)
    assert torch.equal(ids.reshape(rid.shape).long(), rid)
    assert ((w.reshape(rw.shape).double() - rw).abs() <= 1e-4 * rw).all()
    bad = (out.reshape(ref.shape).double() - ref).abs() > 2.0 ** -8 * ref.abs() + off + 1e-30
    assert not bad.any(), (int(bad.sum()), (out.reshape(ref.shape).double() - ref).abs().max().item())
    return out


SIZES = [  # tokens, width, inner, experts, top_k
    (1, 8, 8, 1, 1), (1, 64, 128, 4, 2), (2, 72, 136, 5, 5), (3, 776, 1000, 10, 3), (1, 2048, 1024, 16, 8),
    (8, 256, 64, 33, 4), (9, 128, 96, 7, 1), (17, 512, 520, 3, 2), (64, 256, 128, 128, 8), (64, 96, 64, 2, 2),
    (65, 128, 64, 12, 4), (130, 64, 40, 300, 16), (5, 40, 2056, 512, 16)]


@pytest.mark.parametrize("kind,group,zeros", [("bf16", 128, False), ("4bit", 32, True), ("4bit", 64, False),
                                              ("4bit", 128, True)])
@pytest.mark.parametrize("tokens,width,inner,experts,top_k", SIZES)
def test_against_64_bits(tokens, width, inner, experts, top_k, kind, group, zeros):
    layer, router, wide = _layer(width, inner, experts, top_k, kind, group, zeros, renormalize=tokens % 2 == 1)
    x = torch.randn(tokens, width, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).bfloat16()
    _run(x, layer, router, wide)


def test_every_token_to_the_same_experts():
    """All 64 tokens take the same two of 40 experts, the others none."""
    layer, router, wide = _layer(128, 64, 40, 2)
    x = torch.randn(1, 128, device="cuda").bfloat16() + 0.01 * torch.randn(64, 128, device="cuda").bfloat16()
    _run(x.bfloat16(), layer, router, wide)


def test_ties_go_to_the_lowest_expert():
    from tao_memory_b200 import ExpertWeights, expert_layer
    layer, router, wide = _layer(64, 32, 70, 6)
    router = router[:1].expand(70, 64).contiguous()
    router[40] = 0
    ws = [w.bfloat16() for w in wide]
    layer = ExpertWeights(router, *ws, top_k=6)
    x = torch.randn(3, 64, device="cuda").bfloat16()
    x[2] = 0  # every logit is 0
    _, ids, w = expert_layer(x, layer, return_routing=True)
    logit = (x.double() @ router[0].double())
    for t in range(3):
        want = [40, 0, 1, 2, 3, 4] if logit[t] < 0 else [0, 1, 2, 3, 4, 5]
        assert ids[t].tolist() == want
    assert (w[2] == 1 / 6).all() or (w[2] - 1 / 6).abs().max() < 1e-7


def test_rows_without_numbers_stay_alone():
    layer, router, wide = _layer(256, 128, 16, 4)
    from tao_memory_b200 import expert_layer
    x = torch.randn(6, 256, device="cuda").bfloat16()
    clean = expert_layer(x[[0, 2, 3, 5]], layer)
    x[1, 3], x[4, 9] = float("nan"), float("inf")
    out, ids, w = expert_layer(x, layer, return_routing=True)
    assert torch.equal(out[[0, 2, 3, 5]], clean)
    assert out[1].isnan().all() and w[1].isnan().all() and not out[4].isfinite().any()
    assert ((ids >= 0) & (ids < 16)).all()


def test_views_streams_graph_and_repeats():
    from tao_memory_b200 import ExpertWeights, expert_layer
    layer, router, wide = _layer(264, 72, 9, 3)
    # gate and up as halves of one tensor; the others off their alignment
    fused = torch.cat((wide[0], wide[1]), 1).bfloat16()
    odd = torch.empty(9 * 264 * 72 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(9, 264, 72)
    odd.copy_(wide[2])
    layer = ExpertWeights(router, fused[:, :72], fused[:, 72:], odd, top_k=3)
    assert layer.gate.data_ptr() == fused.data_ptr()
    base = torch.randn(4, 3, 600, device="cuda").bfloat16()
    for x in (base[:, 1, 8:272], base[:, 1, 5:269], base[:, :, 16:280], base[:, 0, ::2][:, :264], base[0, 0, :264],
              base[:1, 0, :264].expand(4, 264)):
        _run(x, layer, router, wide)
    x = base[:, 1, 8:272]
    first = expert_layer(x, layer)
    assert expert_layer(x[:0], layer).shape == (0, 264)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        outs = [expert_layer(x, layer) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)
    graph = torch.cuda.CUDAGraph()
    xs = x.contiguous()
    with torch.cuda.graph(graph):
        y = expert_layer(xs, layer)
    for seed in range(3):
        xs.copy_(torch.randn(4, 264, device="cuda"))
        graph.replay()
        assert torch.equal(y, expert_layer(xs, layer))
    from tao_memory_b200.stream import check_device
    assert check_device() == 0


def test_layers_of_different_size_share_a_workspace():
    small, r1, w1 = _layer(64, 32, 4, 2)
    large, r2, w2 = _layer(1032, 520, 24, 6, seed=1)
    for tokens in (1, 40, 3):
        for layer, router, wide in ((small, r1, w1), (large, r2, w2)):
            x = torch.randn(tokens, layer.width, device="cuda").bfloat16()
            _run(x, layer, router, wide)


def test_an_error_word_is_reported_once():
    """The host's side of an expired wait: the word is set here by hand."""
    from tao_memory_b200 import _lib, expert_layer
    from tao_memory_b200.experts import _Room
    from tao_memory_b200.stream import check_device
    layer, router, wide = _layer(64, 32, 4, 2)
    x = torch.randn(2, 64, device="cuda").bfloat16()
    out = expert_layer(x, layer)
    room = _Room.get(x.device, torch.cuda.current_stream().cuda_stream, 1)
    room[:4] = torch.tensor([1, 0, 0, 0], dtype=torch.uint8)
    with pytest.raises(_lib.TaoError):
        check_device()
    assert check_device() == 0 and (room == 0).all()
    assert torch.equal(expert_layer(x, layer), out)


def test_refusals():
    from tao_memory_b200 import ExpertWeights, expert_layer, quantize4
    layer, router, wide = _layer(64, 32, 4, 2)
    gate, up, down = (w.bfloat16() for w in wide)
    x = torch.randn(2, 64, device="cuda").bfloat16()
    q = [quantize4(w, 32) for w in (gate, up, down)]
    for bad in (lambda: expert_layer(x.float(), layer), lambda: expert_layer(x.cpu(), layer),
                lambda: expert_layer(x[:, :32], layer), lambda: expert_layer(x, gate),
                lambda: expert_layer(x, layer, out=x[:1]), lambda: expert_layer(x.clone().requires_grad_(True), layer),
                lambda: ExpertWeights(router, gate, up, down, top_k=5),
                lambda: ExpertWeights(router, gate, up, down, top_k=0),
                lambda: ExpertWeights(router, gate, up, gate, top_k=2),
                lambda: ExpertWeights(router.float(), gate, up, down, top_k=2),
                lambda: ExpertWeights(router, q[0], up, down, top_k=2),
                lambda: ExpertWeights(router, q[0], q[1], quantize4(down, 64), top_k=2),
                lambda: ExpertWeights(router, q[0], q[1], quantize4(down, 32, zeros=True), top_k=2),
                lambda: ExpertWeights(router[:, :60], gate[..., :60], up[..., :60], down[:, :60], top_k=2),
                lambda: ExpertWeights(router.repeat(129, 1), *(w.repeat(129, 1, 1) for w in (gate, up, down)),
                                      top_k=2)):
        with pytest.raises(ValueError):
            bad()
