"""Cases of the operators around the attention in a served or trained block: the root-mean-square
norm with the residual's addition (also with an 8-bit output, and its gradient), the product of a
few rows with 4-bit weights, and the mixture-of-experts layer for a few tokens.

Each case is computed in plain form here (`own` false: elementary torch operations in 32 bits,
rounded once) or by the package's entry points (`own` true), and in 64 bits by `exact`.

Definitions (D = width, all sums over the last axis):

* norm: s = x + residual rounded to the stream's type (the next block reads it), r = rsqrt(mean s^2 + eps),
  y = s r w.  8 bits: per row or per 128 channels scale = max(max |y|, 1e-30) / 448 and
  q = e4m3(y 448 / max(max |y|, 1e-30)).  Gradient with n = s r: dx = ds + r (w dy - n mean(w dy n)), dw = sum over rows of dy n.
* product: y = x W^T + b with W[n][k] = (code[n][k] - zero[n][k / group]) scale[n][k / group]; x in
  16 bits, or in e4m3 with one scale a row.
* experts: p = softmax(x R^T); the top_k largest p (ties to the lowest index), optionally divided by
  their sum; out = sum over them of p down_e(silu(gate_e x) * (up_e x)).
"""

import math

import torch

own = False

EPS = 1e-6
E4M3_MAX, TINY = 448.0, 1e-30
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# -- cases ---------------------------------------------------------------
def _norm(name, rows, width, dtype="bf16", out="same", residual=True, grad=False):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "out": out,
            "residual": residual, "grad": grad}


def _product(name, rows, k, n, group=128, zeros=False, bias=False, act="bf16"):
    return {"name": name, "op": "product", "rows": rows, "k": k, "n": n, "group": group, "zeros": zeros,
            "bias": bias, "act": act}


def _experts(name, tokens, width, inner, experts, top_k, weights="bf16", group=128, zeros=False, renorm=True):
    return {"name": name, "op": "experts", "tokens": tokens, "width": width, "inner": inner, "experts": experts,
            "top_k": top_k, "weights": weights, "group": group, "zeros": zeros, "renorm": renorm}


def listed():
    return [
        # eight requests decode one token each at 12 heads of 64
        _norm("norm 8x768", 8, 768),
        # a 16K-token prompt at 16 heads of 128, quantised for an 8-bit product, one scale a row
        _norm("norm fp8 16384x2048", 16384, 2048, out="fp8"),
        # the training step: batch 4 of 8192 tokens at 12 heads of 64, forward and backward
        _norm("norm train 32768x768", 32768, 768, grad=True),
        # a ragged batch of a model in 32 bits whose width no vector divides, forward and backward
        _norm("norm train fp32 1003x1001", 1003, 1001, dtype="fp32", grad=True, residual=False),
        # one token through the fused projection of 16 heads of 128
        _product("product 1x2048x6144", 1, 2048, 6144),
        # eight requests through a large projection with zero points
        _product("product 8x8192x8192", 8, 8192, 8192, group=64, zeros=True, bias=True),
        # three draft tokens, odd sizes, small groups, fp16
        _product("product fp16 3x1001x1999", 3, 1001, 1999, group=32, zeros=True, act="fp16"),
        # the 64 requests of the serving mix, activations already in 8 bits
        _product("product fp8 64x2048x6144", 64, 2048, 6144, act="fp8"),
        # one token through 64 experts
        _experts("experts 1 of 64", 1, 2048, 1024, 64, 8),
        # eight requests, 4-bit experts
        _experts("experts 4-bit 8 of 64", 8, 2048, 1024, 64, 8, weights="4bit"),
        # the 64 requests of the serving mix: nearly every expert is read
        _experts("experts 64 of 128", 64, 2048, 768, 128, 8),
        # a small layer of few experts with odd sizes, 4-bit with zero points
        _experts("experts 4-bit 5 of 10", 5, 776, 1000, 10, 3, weights="4bit", group=32, zeros=True, renorm=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high, multiple=1):
    """Log-uniform; of any remainder half of the time, else a multiple of 64."""
    v = _log(rng, low, high)
    step = multiple if rng.random() < 0.5 else max(multiple, 64)
    v = max(multiple, min(high, v) // step * step)
    return v + multiple if v == 3072 else v


def draw(rng):
    op = rng.choice(("norm", "product", "experts"))
    if op == "norm":
        width = _size(rng, 64, 8192)
        rows = _log(rng, 1, min(32768, (1 << 24) // width))
        rows += rows == 3072
        grad = rng.random() < 0.5
        case = _norm("", rows, width, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                     out="same" if grad else rng.choice(("same", "fp8", "fp8 by 128")),
                     residual=rng.random() < 0.75, grad=grad)
    elif op == "product":
        k = _size(rng, 64, 16384)
        n = _size(rng, 64, min(16384, (1 << 26) // k))
        case = _product("", _log(rng, 1, 64), k, n, group=rng.choice((32, 64, 128)), zeros=rng.random() < 0.5,
                        bias=rng.random() < 0.3, act=rng.choice(("bf16", "bf16", "fp16", "fp8")))
    else:
        width = _size(rng, 256, 4096, 8)
        inner = _size(rng, 128, 2048, 8)
        experts = _log(rng, 4, max(4, min(128, (1 << 27) // (width * inner))))
        case = _experts("", _log(rng, 1, 64), width, inner, experts, rng.randint(1, min(8, experts)),
                        weights=rng.choice(("bf16", "4bit")), group=rng.choice((32, 64, 128)),
                        zeros=rng.random() < 0.5, renorm=rng.random() < 0.7)
    del case["name"]
    return case


# -- inputs --------------------------------------------------------------
def _codes(normal, uniform, batch, n, k, group, zeros):
    """4-bit codes [.., n, k] of roughly normal weights, their scales [.., n, groups] and zero points."""
    groups = -(-k // group)
    codes = normal(*batch, n, k).mul_(2.6).add_(8).round_().clamp_(0, 15).to(torch.uint8)
    scales = (uniform(*batch, n, groups) + 0.5) * (0.4 / math.sqrt(k))
    zero = (uniform(*batch, n, groups) * 5 + 6).to(torch.uint8) if zeros else None
    return codes, scales, zero


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=dev, dtype=dtype, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=g)

    st = {"case": case}
    if case["op"] == "norm":
        dt, rows, width = TYPES[case["dtype"]], case["rows"], case["width"]
        # a residual stream: channels of different size, some of them much larger
        channel = torch.exp(0.5 * normal(width)) * (1 + 20 * (uniform(width) > 0.995))
        st["x"] = (normal(rows, width) * 0.5).to(dt)
        st["residual"] = (normal(rows, width) * channel).to(dt) if case["residual"] else None
        st["weight"] = (1 + 0.2 * normal(width)).to(dt)
        if case["grad"]:
            st["dy"] = normal(rows, width).to(dt)
            st["ds"] = normal(rows, width).to(dt) if case["residual"] else None
            for key in ("x", "residual", "weight"):
                if st[key] is not None:
                    st[key].requires_grad_(True)
        return st
    if case["op"] == "product":
        rows, k, n = case["rows"], case["k"], case["n"]
        dt = TYPES["fp16" if case["act"] == "fp16" else "bf16"]
        x = normal(rows, k)
        st["x_scale"] = None
        if case["act"] == "fp8":
            st["x_scale"] = x.abs().amax(-1, keepdim=True) / E4M3_MAX
            st["x"] = (x / st["x_scale"]).to(torch.float8_e4m3fn)
        else:
            st["x"] = x.to(dt)
        codes, scales, zeros = _codes(normal, uniform, (), n, k, case["group"], case["zeros"])
        st["codes"], st["scales"], st["zeros"] = codes, scales.to(dt), zeros
        st["bias"] = normal(n).to(dt) if case["bias"] else None
        if own:
            from tao_memory_b200 import Weight4
            st["weight"] = Weight4.from_codes(codes, st["scales"], zeros, group=case["group"])
        return st
    d, f, e = case["width"], case["inner"], case["experts"]
    st["x"] = normal(case["tokens"], d).to(torch.bfloat16)
    st["router"] = (normal(e, d) * (2 / math.sqrt(d))).to(torch.bfloat16)
    shapes = {"gate": (f, d), "up": (f, d), "down": (d, f)}
    for name, (n, k) in shapes.items():
        if case["weights"] == "4bit":
            codes, scales, zeros = _codes(normal, uniform, (e,), n, k, case["group"], case["zeros"])
            st[name] = (codes, scales.to(torch.bfloat16), zeros)
        else:
            st[name] = normal(e, n, k, dtype=torch.bfloat16).mul_(1 / math.sqrt(k))
    if own:
        from tao_memory_b200 import ExpertWeights, Weight4
        w = [Weight4.from_codes(*st[n], group=case["group"]) if case["weights"] == "4bit" else st[n] for n in shapes]
        st["layer"] = ExpertWeights(st["router"], *w, top_k=case["top_k"], renormalize=case["renorm"])
    return st


# -- the plain form ------------------------------------------------------
def _plain_norm(st):
    case = st["case"]
    x, res, w = (None if st[k] is None else st[k].detach() for k in ("x", "residual", "weight"))
    s = x if res is None else (x.float() + res.float()).to(x.dtype)
    sf, wf = s.float(), w.float()
    r = torch.rsqrt((sf * sf).mean(-1, keepdim=True) + EPS)
    y = sf * r * wf
    out = {} if res is None else {"s": s}
    if case["out"] != "same":
        part = case["width"] if case["out"] == "fp8" else 128
        groups = -(-case["width"] // part)
        pad = torch.nn.functional.pad(y, (0, groups * part - case["width"])).view(-1, groups, part)
        top = pad.abs().amax(-1, keepdim=True).clamp_min(TINY)
        q = (pad * (E4M3_MAX / top)).view(y.shape[0], -1)[:, :case["width"]]
        return {**out, "q": q.to(torch.float8_e4m3fn), "scale": (top / E4M3_MAX).squeeze(-1)}
    out["y"] = y.to(x.dtype)
    if case["grad"]:
        n = sf * r
        g = st["dy"].float()
        wg = wf * g
        dx = r * (wg - n * (wg * n).mean(-1, keepdim=True))
        if st["ds"] is not None:
            dx = dx + st["ds"].float()
        out["dx"] = dx.to(x.dtype)
        out["dw"] = (g * n).sum(0).to(w.dtype)
    return out


def _weights(codes, scales, zeros, group):
    """The 4-bit weights in 32 bits."""
    k = codes.shape[-1]
    s = scales.float().repeat_interleave(group, -1)[..., :k]
    if zeros is None:
        return (codes.float() - 8) * s
    return (codes.float() - zeros.float().repeat_interleave(group, -1)[..., :k]) * s


def _plain_product(st):
    x = st["x"].float()
    if st["x_scale"] is not None:
        x = x * st["x_scale"]
    y = x @ _weights(st["codes"], st["scales"], st["zeros"], st["case"]["group"]).T
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.to(st["scales"].dtype)


def _route(x, router, case):
    p = torch.softmax(x @ router.T, -1)
    top, ids = torch.sort(p, dim=-1, descending=True, stable=True)
    top, ids = top[:, :case["top_k"]], ids[:, :case["top_k"]]
    return (top / top.sum(-1, keepdim=True) if case["renorm"] else top), ids


def _plain_experts(st):
    case = st["case"]
    x = st["x"].float()
    top, ids = _route(x, st["router"].float(), case)
    tokens, k = ids.shape

    def of(name, picked):
        w = st[name]
        if case["weights"] == "4bit":
            codes, scales, zeros = (None if t is None else t if picked is None else t[picked] for t in w)
            return _weights(codes, scales, zeros, case["group"])
        return (w if picked is None else w[picked]).float()

    if tokens * k <= case["experts"]:  # fewer pairs than experts: read the chosen experts alone
        pick = ids.reshape(-1)
        xs = x.repeat_interleave(k, 0).unsqueeze(-1)
        h = torch.nn.functional.silu(of("gate", pick) @ xs) * (of("up", pick) @ xs)
        y = (of("down", pick) @ h).view(tokens, k, -1)
        return (y * top.unsqueeze(-1)).sum(1).to(torch.bfloat16)
    share = torch.zeros(tokens, case["experts"], device=x.device).scatter_(1, ids, top).T.unsqueeze(-1)
    h = torch.nn.functional.silu(x @ of("gate", None).transpose(1, 2)) * (x @ of("up", None).transpose(1, 2))
    return (h * share @ of("down", None).transpose(1, 2)).sum(0).to(torch.bfloat16)


# -- the package's entry points ------------------------------------------
def _own_norm(st):
    import tao_memory_b200 as tb
    case = st["case"]
    if case["out"] != "same":
        q, scale, s = tb.add_rms_norm_fp8(st["x"], st["weight"], st["residual"], eps=EPS,
                                          group=None if case["out"] == "fp8" else 128)
        out = {"q": q, "scale": scale}
    else:
        y, s = tb.add_rms_norm(st["x"], st["weight"], st["residual"], eps=EPS)
        out = {"y": y.detach()}
    if st["residual"] is not None:
        out["s"] = s.detach()
    if case["grad"]:
        if st["residual"] is None:
            out["dx"], out["dw"] = torch.autograd.grad(y, (st["x"], st["weight"]), st["dy"])
        else:
            out["dx"], _, out["dw"] = torch.autograd.grad((y, s), (st["x"], st["residual"], st["weight"]),
                                                          (st["dy"], st["ds"]))
    return out


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"norm": _plain_norm, "product": _plain_product, "experts": _plain_experts}[op](state)
    if op == "norm":
        return _own_norm(state)
    import tao_memory_b200 as tb
    if op == "product":
        return tb.linear4(state["x"], state["weight"], bias=state["bias"], x_scale=state["x_scale"])
    return tb.expert_layer(state["x"], state["layer"])


# -- work ----------------------------------------------------------------
def _weight_bytes(count, n, k, bits4, group, zeros):
    if not bits4:
        return 2.0 * count * n * k
    return count * n * (0.5 * k + -(-k // group) * (2.5 if zeros else 2.0))


def work(case):
    if case["op"] == "norm":
        b = 4 if case["dtype"] == "fp32" else 2
        size, two = case["rows"] * case["width"], 2 if case["residual"] else 1
        rows_bytes = size * b * two + size * (b * (two - 1) + (b if case["out"] == "same" else 1))
        flops = 5.0 * size
        if case["grad"]:  # dy, ds and the stream in, dx out
            rows_bytes += size * b * (4 if case["residual"] else 3)
            flops += 10.0 * size
        if case["out"] != "same":
            rows_bytes += 4 * case["rows"] * (1 if case["out"] == "fp8" else -(-case["width"] // 128))
        return {"bytes": rows_bytes + case["width"] * b * (2 if case["grad"] else 1), "flops": flops}
    if case["op"] == "product":
        rows, k, n = case["rows"], case["k"], case["n"]
        bytes_ = _weight_bytes(1, n, k, True, case["group"], case["zeros"]) + rows * n * 2
        bytes_ += rows * (k + 4 if case["act"] == "fp8" else 2 * k) + (2 * n if case["bias"] else 0)
        return {"bytes": bytes_, "flops": 2.0 * rows * k * n}
    t, d, f, e, k = (case[n] for n in ("tokens", "width", "inner", "experts", "top_k"))
    active = e * (1 - (1 - k / e) ** t)  # expected number of experts that some token chose
    bits4 = case["weights"] == "4bit"
    bytes_ = 2.0 * e * d + 4.0 * t * d
    for n, m in ((f, d), (f, d), (d, f)):
        bytes_ += _weight_bytes(active, n, m, bits4, case["group"], case["zeros"])
    return {"bytes": bytes_, "flops": 2.0 * t * e * d + 6.0 * t * k * d * f}


# -- 64 bits -------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        x, w = st["x"].detach(), st["weight"].detach().double()
        s = x.double()
        out = {}
        if case["residual"]:
            out["s"] = x.double() + st["residual"].detach().double()
            s = out["s"].to(torch.float32).to(x.dtype).double()
        r = (s.square().sum(-1, keepdim=True) / case["width"] + EPS).pow(-0.5)
        n = s * r
        if case["out"] != "same":
            part = case["width"] if case["out"] == "fp8" else 128
            tops = [(c.abs().amax(-1, keepdim=True).clamp_min(TINY), c) for c in (n * w).split(part, -1)]
            out["q"] = torch.cat([c * E4M3_MAX / t for t, c in tops], -1)
            out["scale"] = torch.cat([t for t, _ in tops], -1) / E4M3_MAX
            return out
        out["y"] = n * w
        if case["grad"]:
            dn = st["dy"].double() * w
            dx = (dn - n * (dn * n).sum(-1, keepdim=True) / case["width"]) * r
            out["dx"] = dx if st["ds"] is None else dx + st["ds"].double()
            out["dw"] = torch.einsum("rd,rd->d", st["dy"].double(), n)
        return out

    def wide(codes, scales, zeros):
        z = torch.full_like(scales, 8).double() if zeros is None else zeros.double()
        at = torch.arange(codes.shape[-1], device=codes.device) // case["group"]
        return (codes.double() - z[..., at]) * scales.double()[..., at]

    if case["op"] == "product":
        x = st["x"].to(torch.float32).double()
        if st["x_scale"] is not None:
            x = x * st["x_scale"].double()
        y = torch.einsum("rk,nk->rn", x, wide(st["codes"], st["scales"], st["zeros"]))
        return y if st["bias"] is None else y + st["bias"].double()
    x = st["x"].double()
    logits = torch.einsum("td,ed->te", x, st["router"].double())
    p = (logits - logits.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    chosen = torch.topk(p, case["top_k"], -1).indices
    share = torch.zeros_like(p).scatter_(1, chosen, p.gather(1, chosen))
    if case["renorm"]:
        share = share / share.sum(-1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        at = share[:, e].nonzero().flatten()
        if at.numel():
            gate, up, down = (wide(*(None if t is None else t[e] for t in st[n])) if case["weights"] == "4bit"
                              else st[n][e].double() for n in ("gate", "up", "down"))
            a = x[at] @ gate.T
            out[at] += share[at, e:e + 1] * ((a / (1 + (-a).exp()) * (x[at] @ up.T)) @ down.T)
    return out
