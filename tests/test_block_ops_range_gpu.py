"""The block operators at the ends of the sizes they take, against 64 bits.

Bounds as in the operators' own tests: one rounding of the output (U), and fp32 sums before it that lose at
most as many units of 2^-24 of their terms' magnitudes as the longest chain of additions has, 512 for products
of 65536 channels (64 blocks of up to 4 groups in a warp, 16 products a group, and the sums of up to 128 warps).
The norm's row of 65536 is at most 64 additions a thread, 10 more across them, and the few units of the
products and the root: 128."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALL = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25, torch.float32: 1e-37}
EPS = 1e-5


def _near(got, want, terms, dtype, units):
    bad = (got.double() - want).abs() > U[dtype] * want.abs() + units * 2.0 ** -24 * terms + SMALL[dtype]
    assert not bad.any(), (int(bad.sum()), (got.double() - want).abs().max().item())


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16, "fp8"])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 16, 17, 70])
@pytest.mark.parametrize("n,k", [(40, 49408), (24, 65536), (3, 65535)])
def test_products_of_the_longest_rows(n, k, rows, group, act):
    """From about 49000 channels on nine and more rows take the form of up to eight."""
    from tao_memory_b200 import Weight4, linear4
    dtype = torch.bfloat16 if act == "fp8" else act
    g = torch.Generator(device="cuda").manual_seed(k + rows)
    codes = torch.randint(0, 16, (n, k), device="cuda", dtype=torch.uint8, generator=g)
    parts = -(-k // group)
    scales = ((torch.rand(n, parts, device="cuda", generator=g) + 0.1) * k ** -0.5).to(dtype)
    zeros = torch.randint(0, 16, (n, parts), device="cuda", dtype=torch.uint8, generator=g)
    at = torch.arange(k, device="cuda") // group
    wide = (codes.double() - zeros.double()[:, at]) * scales.double()[:, at]
    x = torch.randn(rows, k, device="cuda", generator=g)
    scale = None
    if act == "fp8":
        scale = x.abs().amax(-1, keepdim=True) / 448
        x = (x / scale).to(torch.float8_e4m3fn)
    else:
        x = x.to(act)
    xd = x.float().double() * (1 if scale is None else scale.double())
    y = linear4(x, Weight4.from_codes(codes, scales, zeros, group), x_scale=scale)
    _near(y, xd @ wide.T, xd.abs() @ wide.abs().T, dtype, 512)


@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 65536), (torch.float16, 65528), (torch.bfloat16, 65535),
                                         (torch.bfloat16, 16392), (torch.float16, 16385), (torch.float32, 32768),
                                         (torch.float32, 32767), (torch.float32, 16388)])
@pytest.mark.parametrize("rows", [1, 5, 200])
def test_gradient_of_the_widest_rows(rows, width, dtype):
    from tao_memory_b200 import add_rms_norm
    g = torch.Generator(device="cuda").manual_seed(width)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, res, w = n(rows, width).to(dtype), (3 * n(rows, width)).to(dtype), (1 + 0.3 * n(width)).to(dtype)
    dy, ds = n(rows, width).to(dtype), n(rows, width).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, res)]
    y, s = add_rms_norm(x, w, res, eps=EPS)
    dx, dw, dres = torch.autograd.grad((y, s), leaves, (dy, ds))
    want_s = (x.detach().float() + res.detach().float()).to(dtype)
    assert torch.equal(s, want_s) and torch.equal(dx, dres)
    sd, wd, gd = want_s.double(), w.detach().double(), dy.double()
    r = (sd.square().mean(-1, keepdim=True) + EPS).rsqrt()
    m = sd * r
    _near(y.detach(), m * wd, (m * wd).abs(), dtype, 128)
    wg = wd * gd
    mean, loss = (wg * m).mean(-1, keepdim=True), (wg * m).abs().mean(-1, keepdim=True)
    _near(dx, r * (wg - m * mean) + ds.double(), r * (wg.abs() + m.abs() * (loss + mean.abs())) + ds.double().abs(),
          dtype, 128)
    _near(dw, (gd * m).sum(0), (gd * m).abs().sum(0), dtype, 128)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("tokens,width,inner,experts,top_k", [(1, 32768, 256, 3, 2), (9, 256, 32776, 2, 2),
                                                              (2, 20008, 1000, 4, 1)])
def test_experts_of_many_channels(tokens, width, inner, experts, top_k, four):
    """The sums of up to 32776 channels run over 64 blocks of a warp and more (512 units, as the products');
    h is held to 2^-16."""
    from tao_memory_b200 import ExpertWeights, expert_layer, quantize4
    g = torch.Generator(device="cuda").manual_seed(width)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    router = (2 * n(experts, width) * width ** -0.5).bfloat16()
    ws = [(n(experts, inner, width) * width ** -0.5).bfloat16(), (n(experts, inner, width) * width ** -0.5).bfloat16(),
          (n(experts, width, inner) * inner ** -0.5).bfloat16()]
    if four:
        ws = [quantize4(w, 64, True) for w in ws]
    gate, up, down = (w.dequantize().double() if four else w.double() for w in ws)
    x = n(tokens, width).bfloat16()
    out, ids, share = expert_layer(x, ExpertWeights(router, *ws, top_k=top_k), return_routing=True)
    xd, d = x.double(), 512 * 2.0 ** -24
    p = torch.softmax(xd @ router.double().T, -1)
    order = torch.sort(p, dim=-1, descending=True, stable=True)
    assert torch.equal(ids.long(), order.indices[:, :top_k])
    want = order.values[:, :top_k] / order.values[:, :top_k].sum(-1, keepdim=True)
    assert ((share.double() - want).abs() <= 1e-4 * want).all()
    ref, off = torch.zeros_like(xd), torch.zeros_like(xd)
    slack = 2 * d * (xd.abs() @ router.double().abs().T).amax(-1)
    for e in range(experts):
        t, j = (ids == e).nonzero(as_tuple=True)
        a, b = xd[t] @ gate[e].T, xd[t] @ up[e].T
        s = a * torch.sigmoid(a)
        h = s * b
        dh = 1.1 * d * (xd[t].abs() @ gate[e].abs().T) * b.abs() + d * s.abs() * (xd[t].abs() @ up[e].abs().T)
        dh += 2.0 ** -16 * h.abs()
        y, part = h @ down[e].T, want[t, j].unsqueeze(-1)
        ref.index_add_(0, t, part * y)
        off.index_add_(0, t, part * (dh @ down[e].abs().T + d * (h.abs() @ down[e].abs().T)
                                     + (slack[t] + d).unsqueeze(-1) * y.abs()))
    bad = (out.double() - ref).abs() > 2.0 ** -8 * ref.abs() + off + 1e-30
    assert not bad.any(), (int(bad.sum()), (out.double() - ref).abs().max().item())


@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 65536), (torch.float16, 65535), (torch.float32, 32768),
                                         (torch.float32, 32767), (torch.bfloat16, 20001)])
@pytest.mark.parametrize("rows", [1, 160])
def test_e4m3_of_the_widest_rows(rows, width, dtype, group):
    from tao_memory_b200 import add_rms_norm_fp8
    g = torch.Generator(device="cuda").manual_seed(width + rows)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, res, w = n(rows, width).to(dtype), (3 * n(rows, width)).to(dtype), (1 + 0.3 * n(width)).to(dtype)
    q, scale, s = add_rms_norm_fp8(x, w, res, eps=EPS, group=group)
    want_s = (x.float() + res.float()).to(dtype)
    assert torch.equal(s, want_s)
    sd = want_s.double()
    y = sd * (sd.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
    lost = 128 * 2.0 ** -24
    for i, c in enumerate(y.split(width if group is None else 128, -1)):
        top = c.abs().amax(-1).clamp_min(1e-30)
        assert ((scale[..., i].double() - top / 448).abs() <= lost * top / 448).all()
        v = c * (448 / top).unsqueeze(-1)
        at = i * (width if group is None else 128)
        # e4m3: unit roundoff 2^-4 and half a subnormal step 2^-10
        assert ((q[..., at:at + c.shape[-1]].double() - v).abs() <= (2.0 ** -4 + lost) * v.abs() + 2.0 ** -10).all()


def test_operators_on_two_streams_at_once():
    """Calls on two streams share no workspace: every result is that of the call alone."""
    from tao_memory_b200 import ExpertWeights, add_rms_norm, expert_layer, linear4, quantize4
    from tao_memory_b200.stream import check_device
    g = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: (torch.randn(*s, device="cuda", generator=g) * s[-1] ** -0.5).bfloat16()
    layer = ExpertWeights(n(16, 512), n(16, 256, 512), n(16, 256, 512), n(16, 512, 256), top_k=4)
    w4 = quantize4(n(512, 512))
    xs = [torch.randn(rows, 512, device="cuda", generator=g).bfloat16() for rows in (3, 40)]
    weight = torch.ones(512, device="cuda", dtype=torch.bfloat16)

    def block(x):
        h, s = add_rms_norm(x, weight, x)
        return expert_layer(linear4(h, w4), layer), s

    want = [block(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(25):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(block(xs[i]))
    torch.cuda.synchronize()
    assert check_device() == 0
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
