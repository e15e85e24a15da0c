"""Cases of the operators that train a decoder block around the attention and take its prompts: the
product with bias, activation and residual in 16 bits, tokens sorted by expert and back, the experts'
products over the sorted tokens, and the embedding; each with its gradient.

Each case is computed in plain form here (`own` false: elementary torch operations in 32 bits,
rounded once) or by the package's entry points (`own` true), and in 64 bits by `exact`.

Definitions:

* linear: y = act(x W^T + b) + residual.  With z = x W^T + b and dz = dy act'(z): dx = dz W, dW = dz^T x,
  db = sum of dz over the rows, and the residual's gradient is dy.
* tokens: every token has k experts (an id outside 0..E-1 is none: a padded token's).  Its pairs (token,
  choice) are sorted by expert, stably, those of no expert last.  pairs[p] = the pair at place p, places =
  its inverse, offsets[e] = the first place of expert e; xs[p] = x[token of pairs[p]] and
  y[t] = sum over t's pairs with an expert of w ys[place].  Gradients: dx[t] = sum over t's pairs of
  dxs[place], dys[place] = w dy[t], dw = dy[t] . ys[place] (pairs of no expert: zero).
* experts: the rows offsets[e] to offsets[e + 1] go through expert e: y = act(x W_e^T) (x U_e^T), or
  x W_e^T alone; rows of no expert give zeros.  Gradients of x, W and U by the same formulas.
* embed: y = scale table[id] (an id outside the table gives zeros); dtable[v] = scale sum of dy over the
  tokens whose id is v.
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# -- cases ---------------------------------------------------------------
def _linear(name, rows, k, n, dtype="bf16", act="", bias=False, residual=False, grad=False):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "grad": grad}


def _tokens(name, tokens, width, experts, top_k, dtype="bf16", padded=0, grad=False):
    return {"name": name, "op": "tokens", "tokens": tokens, "width": width, "experts": experts, "top_k": top_k,
            "dtype": dtype, "padded": padded, "grad": grad}


def _experts(name, tokens, k, n, experts, top_k, dtype="bf16", act="silu", padded=0, grad=False):
    return {"name": name, "op": "experts", "tokens": tokens, "k": k, "n": n, "experts": experts, "top_k": top_k,
            "dtype": dtype, "act": act, "padded": padded, "grad": grad}


def _embed(name, tokens, vocab, width, dtype="bf16", scale=1.0, grad=False):
    return {"name": name, "op": "embed", "tokens": tokens, "vocab": vocab, "width": width, "dtype": dtype,
            "scale": scale, "grad": grad}


def listed():
    return [
        # one token through the fused projection of 16 heads of 128
        _linear("linear 1x2048x6144", 1, 2048, 6144),
        # 24 requests decode one token each: a wide projection back into the residual stream
        _linear("linear 24x8192x2048 residual", 24, 8192, 2048, residual=True),
        # a 16K-token prompt at 16 heads of 128 through the first half of a dense feed-forward layer
        _linear("linear gelu 16384x2048x8192", 16384, 2048, 8192, act="gelu", bias=True),
        # the training step: batch 4 of 8192 tokens at 12 heads of 64 through the fused projection
        _linear("linear train 32768x768x2304", 32768, 768, 2304, grad=True),
        # a ragged batch of odd sizes in fp16 with all of the epilogue, forward and backward
        _linear("linear train fp16 1003x1001x515", 1003, 1001, 515, dtype="fp16", act="silu", bias=True, residual=True,
                grad=True),
        # the 64 requests of the serving mix to 8 of 64 experts and back
        _tokens("tokens 64x2048, 8 of 64", 64, 2048, 64, 8),
        # the training step's tokens to 4 of 64 experts and back, forward and backward
        _tokens("tokens train 32768x768, 4 of 64", 32768, 768, 64, 4, grad=True),
        # 96 tokens of a padded batch, 8 of 128 experts: a few rows an expert
        _experts("experts 96x2048x768, 8 of 128", 96, 2048, 768, 128, 8, padded=5),
        # a 4K-token prompt through the gated half of 64 experts
        _experts("experts 4096x2048x1024, 8 of 64", 4096, 2048, 1024, 64, 8),
        # a training step through the gated half of 16 experts, forward and backward
        _experts("experts train 8192x768x1536, 2 of 16", 8192, 768, 1536, 16, 2, grad=True),
        # eight requests decode one token each
        _embed("embed 8 of 32768x2048", 8, 32768, 2048),
        # the training step: batch 4 of 8192 tokens, forward and backward
        _embed("embed train 32768 of 65536x768", 32768, 65536, 768, scale=math.sqrt(768), grad=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high, multiple=1):
    """Log-uniform; of any remainder half of the time, else a multiple of 64."""
    step = multiple if rng.random() < 0.5 else max(multiple, 64)
    return max(multiple, min(high, _log(rng, low, high)) // step * step)


def draw(rng):
    op = rng.choice(("linear", "linear", "tokens", "experts", "embed"))
    grad = rng.random() < 0.5
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "linear":
        k = _size(rng, 64, 8192)
        n = _size(rng, 64, 8192)
        case = _linear("", _log(rng, 1, min(32768, (1 << 38) // (k * n * (3 if grad else 1)))), k, n, dtype=dtype,
                       act=rng.choice(("", "relu", "silu", "gelu", "gelu_tanh")), bias=rng.random() < 0.4,
                       residual=rng.random() < 0.4, grad=grad)
    elif op == "tokens":
        experts = _log(rng, 4, 512)
        top_k = rng.randint(1, min(8, experts))
        width = _size(rng, 64, 8192)
        tokens = _log(rng, 1, min(32768, (1 << 27) // (width * top_k)))
        case = _tokens("", tokens, width, experts, top_k, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                       padded=rng.choice((0, tokens // 7)), grad=grad)
    elif op == "experts":
        k = _size(rng, 128, 4096, 8)
        n = _size(rng, 128, 4096, 8)
        experts = _log(rng, 4, max(4, min(128, (1 << 28) // (k * n))))
        top_k = rng.randint(1, min(8, experts))
        tokens = _log(rng, 1, min(8192, (1 << 36) // (k * n * top_k * (3 if grad else 1))))
        case = _experts("", tokens, k, n, experts, top_k, dtype=dtype, act=rng.choice(("", "silu", "silu", "gelu_tanh")),
                        padded=rng.choice((0, tokens // 7)), grad=grad)
    else:
        width = _size(rng, 64, 4096)
        vocab = _log(rng, 64, min(131072, (1 << 27) // width))
        case = _embed("", _log(rng, 1, min(32768, (1 << 26) // width)), vocab, width,
                      dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), scale=rng.choice((1.0, math.sqrt(width))),
                      grad=grad)
    del case["name"]
    return case


# -- inputs --------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=dev, dtype=dt if math.prod(shape) > 1 << 24 else torch.float32,
                            generator=g) * scale).to(dt)

    def ids(tokens, experts, top_k, padded):
        """Choices of a router that prefers some experts; the last tokens are padding."""
        like = torch.randn(tokens, experts, device=dev, generator=g) + 0.7 * torch.randn(experts, device=dev, generator=g)
        top, at = torch.topk(torch.softmax(like, -1), top_k, -1)
        if padded:
            at[-padded:] = -1
        return at, top / top.sum(-1, keepdim=True)

    st, leaves = {"case": case}, ()
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        st["x"] = normal(rows, k)
        st["weight"] = normal(n, k, scale=1 / math.sqrt(k))
        st["bias"] = normal(n, scale=0.3) if case["bias"] else None
        st["residual"] = normal(rows, n) if case["residual"] else None
        leaves = ("x", "weight", "bias", "residual")
        if case["grad"]:
            st["dy"] = normal(rows, n)
    elif case["op"] == "tokens":
        t, d, k = case["tokens"], case["width"], case["top_k"]
        st["x"] = normal(t, d)
        st["ids"], st["w"] = ids(t, case["experts"], k, case["padded"])
        st["ys"] = normal(t * k, d)
        leaves = ("x", "ys", "w")
        if case["grad"]:
            st["dxs"], st["dy"] = normal(t * k, d), normal(t, d)
    elif case["op"] == "experts":
        t, k, n, e, top = case["tokens"], case["k"], case["n"], case["experts"], case["top_k"]
        at, _ = ids(t, e, top, case["padded"])
        counts = torch.bincount(at.flatten() + 1, minlength=e + 1)[1:]
        st["offsets"] = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
        st["most"] = int(counts.max())  # rows of the fullest expert: the room that the plain form gives each
        st["x"] = normal(t * top, k)
        st["weight"] = normal(e, n, k, scale=1 / math.sqrt(k))
        st["up"] = normal(e, n, k, scale=1 / math.sqrt(k)) if case["act"] else None
        leaves = ("x", "weight", "up")
        if case["grad"]:
            st["dy"] = normal(t * top, n)
    else:
        t, v, d = case["tokens"], case["vocab"], case["width"]
        # words by their rank: a few come very often, most never
        rank = torch.rand(t, device=dev, generator=g).double()
        word = ((v + 1.0) ** rank - 1).long().clamp_(0, v - 1)
        st["ids"] = torch.randperm(v, device=dev, generator=g)[word]
        st["table"] = normal(v, d, scale=0.02)
        leaves = ("table",)
        if case["grad"]:
            st["dy"] = normal(t, d)
    if case["grad"]:
        for key in leaves:
            if st[key] is not None:
                st[key].requires_grad_(True)
    return st


# -- the plain form ------------------------------------------------------
def _act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_linear(st):
    case = st["case"]
    x, w, b, res = (None if st[k] is None else st[k].detach().float() for k in ("x", "weight", "bias", "residual"))
    dt = st["x"].dtype
    z = x @ w.T
    if b is not None:
        z = z + b
    y = _act(z, case["act"])
    out = {"y": (y if res is None else y + res).to(dt)}
    if case["grad"]:
        dz = st["dy"].float() * _act_slope(z, case["act"])
        out["dx"], out["dw"] = (dz @ w).to(dt), (dz.T @ x).to(dt)
        if b is not None:
            out["db"] = dz.sum(0).to(dt)
        if res is not None:
            out["dres"] = st["dy"]
    return out


def _plain_tokens(st):
    case = st["case"]
    x, ys, w = st["x"].detach(), st["ys"].detach(), st["w"].detach()
    ids, e, k = st["ids"], case["experts"], case["top_k"]
    flat = ids.reshape(-1)
    has = (flat >= 0) & (flat < e)
    by, pairs = torch.sort(torch.where(has, flat, e), stable=True)
    places = torch.empty_like(pairs)
    places[pairs] = torch.arange(pairs.numel(), device=pairs.device)
    offsets = torch.searchsorted(by, torch.arange(e + 1, device=by.device))
    weight = torch.where(has.view(-1, k), w, 0)
    at = places.view(-1, k)
    out = {"pairs": pairs.to(torch.int32), "places": at.to(torch.int32), "offsets": offsets.to(torch.int32),
           "xs": x[pairs // k], "y": (ys.float()[at] * weight.unsqueeze(-1)).sum(1).to(x.dtype)}
    if case["grad"]:
        dy = st["dy"].float()
        out["dx"] = st["dxs"].float()[at].sum(1).to(x.dtype)
        dys = torch.empty_like(ys)
        dys[places] = (weight.unsqueeze(-1) * dy.unsqueeze(1)).to(x.dtype).view(-1, x.shape[1])
        out["dys"] = dys
        out["dw"] = torch.where(has.view(-1, k), (ys.float()[at] * dy.unsqueeze(1)).sum(-1), 0)
    return out


def _plain_experts(st):
    case = st["case"]
    x, w, up = (None if st[k] is None else st[k].detach() for k in ("x", "weight", "up"))
    offsets, e, dt = st["offsets"].long(), case["experts"], x.dtype
    # the rows of each expert, filled up to those of the fullest
    at = offsets[:-1, None] + torch.arange(st["most"], device=x.device)
    inside = (at < offsets[1:, None]).unsqueeze(-1)
    at = at.clamp_max(x.shape[0] - 1)
    of = torch.searchsorted(offsets[1:], torch.arange(x.shape[0], device=x.device), right=True)
    row = torch.arange(x.shape[0], device=x.device) - offsets[of]
    kept, of = (of < e).unsqueeze(-1), of.clamp_max(e - 1)
    row = row.clamp_max(st["most"] - 1)

    def padded(t):
        return torch.where(inside, t[at].float(), 0)

    def rows(t):
        return torch.where(kept, t[of, row], 0).to(dt)

    xs = padded(x)
    z = xs @ w.float().transpose(1, 2)
    if up is None:
        out = {"y": rows(z)}
    else:
        u = xs @ up.float().transpose(1, 2)
        out = {"y": rows(_act(z, case["act"]) * u)}
    if case["grad"]:
        dy = padded(st["dy"])
        dz = dy if up is None else dy * u * _act_slope(z, case["act"])
        dx = dz @ w.float()
        out["dw"] = (dz.transpose(1, 2) @ xs).to(dt)
        if up is not None:
            du = dy * _act(z, case["act"])
            dx = dx + du @ up.float()
            out["dup"] = (du.transpose(1, 2) @ xs).to(dt)
        out["dx"] = rows(dx)
    return out


def _plain_embed(st):
    case, table = st["case"], st["table"].detach()
    out = {"y": (table[st["ids"]].float() * case["scale"]).to(table.dtype)}
    if case["grad"]:
        sums = torch.zeros(table.shape, device=table.device, dtype=torch.float32)
        sums.index_add_(0, st["ids"], st["dy"].float())
        out["dtable"] = (sums * case["scale"]).to(table.dtype)
    return out


# -- the package's entry points ------------------------------------------
def _own_linear(st):
    import tao_memory_b200 as tb
    case = st["case"]
    y = tb.linear(st["x"], st["weight"], bias=st["bias"], residual=st["residual"], activation=case["act"] or None)
    out = {"y": y.detach()}
    if case["grad"]:
        names = {"dx": "x", "dw": "weight", "db": "bias", "dres": "residual"}
        names = {k: v for k, v in names.items() if st[v] is not None}
        out.update(zip(names, torch.autograd.grad(y, [st[v] for v in names.values()], st["dy"])))
    return out


def _own_tokens(st):
    import tao_memory_b200 as tb
    case = st["case"]
    order = tb.sort_tokens(st["ids"], case["experts"])
    xs = tb.gather_tokens(st["x"], order)
    y = tb.return_tokens(st["ys"], order, st["w"])
    out = {"pairs": order.pairs, "places": order.places, "offsets": order.offsets, "xs": xs.detach(), "y": y.detach()}
    if case["grad"]:
        out["dx"], out["dys"], out["dw"] = torch.autograd.grad((xs, y), (st["x"], st["ys"], st["w"]),
                                                               (st["dxs"], st["dy"]))
    return out


def _own_experts(st):
    import tao_memory_b200 as tb
    case = st["case"]
    y = tb.expert_linear(st["x"], st["weight"], st["offsets"], up=st["up"], activation=case["act"] or None)
    out = {"y": y.detach()}
    if case["grad"]:
        names = {"dx": "x", "dw": "weight", "dup": "up"}
        names = {k: v for k, v in names.items() if st[v] is not None}
        out.update(zip(names, torch.autograd.grad(y, [st[v] for v in names.values()], st["dy"])))
    return out


def _own_embed(st):
    import tao_memory_b200 as tb
    y = tb.embed(st["ids"], st["table"], scale=st["case"]["scale"])
    out = {"y": y.detach()}
    if st["case"]["grad"]:
        out["dtable"], = torch.autograd.grad(y, st["table"], st["dy"])
    return out


_PLAIN = {"linear": _plain_linear, "tokens": _plain_tokens, "experts": _plain_experts, "embed": _plain_embed}
_OWN = {"linear": _own_linear, "tokens": _own_tokens, "experts": _own_experts, "embed": _own_embed}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# -- work ----------------------------------------------------------------
def work(case):
    size = 4.0 if case["dtype"] == "fp32" else 2.0
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        once = m * k + n * k + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        flops = 2.0 * m * k * n
        if case["grad"]:  # dy in; dx, dw and db out
            once += m * n + m * k + n * k + (n if case["bias"] else 0)
            flops *= 3
        return {"bytes": size * once, "flops": flops}
    if case["op"] == "tokens":
        t, d, k = case["tokens"], case["width"], case["top_k"]
        bytes_ = size * d * (2 * t + 2 * t * k) + t * k * (8 + 4 + 8)  # x, xs, ys, y; ids, weights, the order
        flops = 2.0 * t * k * d
        if case["grad"]:  # dxs, dy in; dx, dys, dw out (ys is read above)
            bytes_ += size * d * (2 * t + 2 * t * k) + 4.0 * t * k
            flops *= 3.5
        return {"bytes": bytes_, "flops": flops}
    if case["op"] == "experts":
        t, k, n, e, top = (case[i] for i in ("tokens", "k", "n", "experts", "top_k"))
        pairs, two = (t - case["padded"]) * top, 2 if case["act"] else 1
        active = e * (1 - (1 - top / e) ** (t - case["padded"]))  # expected number of experts with rows
        bytes_ = size * (two * active * n * k + pairs * (k + n)) + 4 * (e + 1)
        flops = 2.0 * two * pairs * k * n
        if case["grad"]:  # dy in; dx, dw and dup out
            bytes_ += size * (pairs * (k + n) + two * e * n * k)
            flops *= 3
        return {"bytes": bytes_, "flops": flops}
    t, v, d = case["tokens"], case["vocab"], case["width"]
    bytes_ = 8.0 * t + size * 2 * t * d
    if case["grad"]:
        bytes_ += size * (t * d + v * d)
    return {"bytes": bytes_, "flops": 1.0 * t * d * (2 if case["grad"] else 1)}


# -- 64 bits -------------------------------------------------------------
def _exact_act(z, name):
    """(act(z), act'(z)) in 64 bits."""
    if not name:
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).double()
    if name == "silu":
        s = 1 / (1 + (-z).exp())
        return z * s, s + z * s * (1 - s)
    if name == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * (-z.square() / 2).exp() / math.sqrt(2 * math.pi)
    q = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z.pow(3))
    s = 1 / (1 + (-q).exp())
    return z * s, s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z.square())


def exact(case, seed):
    st = {k: v.detach() if torch.is_tensor(v) else v for k, v in prepare(case, seed).items()}
    if case["op"] == "linear":
        x, w = st["x"].double(), st["weight"].double()
        z = torch.einsum("mk,nk->mn", x, w)
        if st["bias"] is not None:
            z += st["bias"].double()
        y, slope = _exact_act(z, case["act"])
        out = {"y": y if st["residual"] is None else y + st["residual"].double()}
        if case["grad"]:
            dz = slope * st["dy"].double()
            out["dx"], out["dw"] = torch.einsum("mn,nk->mk", dz, w), torch.einsum("mn,mk->nk", dz, x)
            if st["bias"] is not None:
                out["db"] = dz.sum(0)
            if st["residual"] is not None:
                out["dres"] = st["dy"].double()
        return out
    if case["op"] == "tokens":
        e, k = case["experts"], case["top_k"]
        ids = st["ids"].flatten().cpu().numpy()
        key = ids.copy()
        key[(ids < 0) | (ids >= e)] = e
        order = key.argsort(kind="stable")
        dev = st["x"].device
        pairs = torch.from_numpy(order).to(dev)
        token = pairs // k
        w = torch.where((st["ids"] >= 0) & (st["ids"] < e), st["w"].double(), 0.0).flatten()[pairs]
        ys = st["ys"].double()
        y = torch.zeros(st["x"].shape, dtype=torch.float64, device=dev).index_add_(0, token, w[:, None] * ys)
        out = {"pairs": None, "places": None, "offsets": None, "xs": st["x"].double()[token], "y": y}
        if case["grad"]:
            dy = st["dy"].double()
            out["dx"] = torch.zeros_like(y).index_add_(0, token, st["dxs"].double())
            out["dys"] = w[:, None] * dy[token]
            dw = torch.zeros(pairs.numel(), dtype=torch.float64, device=dev)
            dw[pairs] = torch.einsum("pd,pd->p", dy[token], ys) * (st["ids"].flatten()[pairs] >= 0)
            out["dw"] = dw.view(-1, k)
        return out
    if case["op"] == "experts":
        x, limits = st["x"].double(), st["offsets"].tolist()
        y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=x.device)
        out = {"y": y}
        if case["grad"]:
            out["dw"] = torch.zeros(st["weight"].shape, dtype=torch.float64, device=x.device)
            if st["up"] is not None:
                out["dup"] = torch.zeros_like(out["dw"])
            out["dx"] = torch.zeros_like(x)
        for e in range(case["experts"]):
            at = slice(limits[e], limits[e + 1])
            if limits[e] == limits[e + 1]:
                continue
            w = st["weight"][e].double()
            a, slope = _exact_act(x[at] @ w.T, case["act"])
            u = x[at] @ st["up"][e].double().T if st["up"] is not None else 1.0
            y[at] = a * u
            if case["grad"]:
                dy = st["dy"][at].double()
                dz = dy * u * slope
                out["dx"][at] = dz @ w
                out["dw"][e] = dz.T @ x[at]
                if st["up"] is not None:
                    out["dx"][at] += (dy * a) @ st["up"][e].double()
                    out["dup"][e] = (dy * a).T @ x[at]
        return out
    one = st["table"].double()
    out = {"y": one.index_select(0, st["ids"]) * case["scale"]}
    if case["grad"]:
        out["dtable"] = torch.zeros_like(one).index_put_((st["ids"],), st["dy"].double() * case["scale"], accumulate=True)
    return out
