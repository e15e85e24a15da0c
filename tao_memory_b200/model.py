"""Model-side neighbours of the operator: the caller's fused Q/K/V projection and the
RMS normalisation of the exact-local q and k (reference examples/common.py:6-20,
``ProjectedInputs``), with the same names and semantics.

The projection is a plain GEMM (``F.linear``, cuBLAS); the split into the five
operands and the two RMS norms run in one library kernel forward and one backward
(``tao_qkv_split_norm``), so the operator receives contiguous q, k, v, raw_q and raw_k
without five separate elementwise passes.  Positional transforms stay the caller's.

``ServedBlock`` is a whole decoder block around the operator as it is served: residual
norms, 4-bit projections and a mixture-of-experts layer (``add_rms_norm``, ``linear4``,
``expert_layer``) on both sides of the streaming attention.  ``TrainedBlock`` and
``TrainedDecoder`` are the block and a small model in training, in 16 bits (``embed``,
``linear``, tokens sorted by expert and ``expert_linear``), which also take prompts and
decode as they are.
"""

import torch
from torch import nn
from torch.nn import functional as F

from . import _lib
from .embedding import embed
from .experts import expert_layer
from .linear import expert_linear, linear
from .linear4 import linear4
from .norm import add_rms_norm
from .operator import DEFAULT_CONFIG, tao_attention, tao_attention_decode_batch, tao_attention_prefill
from .tokens import gather_tokens, return_tokens, sort_tokens

_BF16 = torch.bfloat16
# F.rms_norm's default eps: the epsilon of its fp32 compute type (also for bf16 inputs)
RMS_EPS = float(torch.finfo(torch.float32).eps)


class _SplitNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, projected, heads, width):
        rows = projected.numel() // (3 * heads * width)
        shape = (*projected.shape[:-1], heads, width)
        outs = [torch.empty(shape, dtype=_BF16, device=projected.device) for _ in range(5)]
        q, k, v, raw_q, raw_k = outs
        stream = torch.cuda.current_stream(projected.device).cuda_stream
        _lib.check(_lib.lib().tao_qkv_split_norm(projected.data_ptr(), rows, heads, width, RMS_EPS, q.data_ptr(),
                                                 k.data_ptr(), v.data_ptr(), raw_q.data_ptr(), raw_k.data_ptr(),
                                                 stream))
        ctx.save_for_backward(raw_q, raw_k)
        ctx.dims = (rows, heads, width, projected.shape)
        return q, k, v, raw_q, raw_k

    @staticmethod
    def backward(ctx, dq, dk, dv, d_raw_q, d_raw_k):
        raw_q, raw_k = ctx.saved_tensors
        rows, heads, width, shape = ctx.dims
        grads = [torch.zeros_like(raw_q) if g is None else g.to(_BF16).contiguous()
                 for g in (dq, dk, dv, d_raw_q, d_raw_k)]
        d_proj = torch.empty(shape, dtype=_BF16, device=raw_q.device)
        stream = torch.cuda.current_stream(raw_q.device).cuda_stream
        _lib.check(_lib.lib().tao_qkv_split_norm_backward(raw_q.data_ptr(), raw_k.data_ptr(),
                                                          *(g.data_ptr() for g in grads), rows, heads, width,
                                                          RMS_EPS, d_proj.data_ptr(), stream))
        return d_proj, None, None


def split_norm(projected, heads, width):
    """[..., 3 * heads * width] bf16 CUDA -> (q, k, v, raw_q, raw_k), each [..., heads, width]."""
    if projected.dtype != _BF16 or not projected.is_cuda:
        raise ValueError("split_norm takes a bf16 CUDA projection (no CPU fallback)")
    if projected.shape[-1] != 3 * heads * width:
        raise ValueError("the projection's last dimension must be 3 * heads * width")
    return _SplitNorm.apply(projected.contiguous(), heads, width)


class ProjectedInputs(nn.Module):
    """Caller-owned projections feeding the operator (examples/common.py:6-20):
    x [B, T, heads * width] -> q, k, v, raw_q, raw_k [B, T, heads, width]; fusion_a and
    fusion_b are the pointwise gate's parameters."""

    def __init__(self, heads=2, width=64):
        super().__init__()
        self.heads, self.width = heads, width
        self.projection = nn.Linear(heads * width, 3 * heads * width, bias=False)
        self.fusion_a = nn.Parameter(torch.zeros(heads, width, 3))
        self.fusion_b = nn.Parameter(torch.zeros(heads, width, 3))

    def forward(self, x):
        projected = F.linear(x, self.projection.weight.to(x.dtype))
        return split_norm(projected, self.heads, self.width)


class ServedBlock:
    """One decoder block of a served model (inference only):

        h, stream = norm(x + stream);  x = W_out attention(split(W_qkv h))
        h, stream = norm(x + stream);  x = experts(h)

    qkv: ``Weight4`` [3 * heads * width, heads * width]; out: ``Weight4`` [heads * width,
    heads * width]; norms: the two norms' weights [heads * width] bf16; experts:
    ``ExpertWeights``; fusion_a, fusion_b, alpha: the operator's parameters.  ``transform``
    (q, k) -> (q, k) is the caller's positional transform of the exact-local operands."""

    def __init__(self, heads, width, qkv, out, norms, experts, fusion_a, fusion_b, alpha, transform=None,
                 eps=RMS_EPS):
        channels = heads * width
        if qkv.shape != (3 * channels, channels) or out.shape != (channels, channels):
            raise ValueError("qkv is [3 * heads * width, heads * width] and out [heads * width, heads * width]")
        if experts.width != channels or len(norms) != 2:
            raise ValueError("the experts have heads * width channels, and there are two norms")
        self.heads, self.width, self.qkv, self.out, self.norms = heads, width, qkv, out, tuple(norms)
        self.experts, self.fusion_a, self.fusion_b, self.alpha = experts, fusion_a, fusion_b, alpha
        self.transform, self.eps = transform, eps

    def _operands(self, x, stream, lead):
        h, stream = add_rms_norm(x, self.norms[0], stream, eps=self.eps)
        q, k, v, raw_q, raw_k = split_norm(linear4(h, self.qkv).view(*lead, -1), self.heads, self.width)
        if self.transform is not None:
            q, k = self.transform(q, k)
        return stream, (q, k, v), {"raw_q": raw_q, "raw_k": raw_k, "fusion_a": self.fusion_a,
                                   "fusion_b": self.fusion_b, "alpha": self.alpha}

    def _close(self, attention, stream):
        x = linear4(attention.reshape(stream.shape), self.out)
        h, stream = add_rms_norm(x, self.norms[1], stream, eps=self.eps)
        return expert_layer(h, self.experts), stream

    @torch.no_grad()
    def step(self, x, stream, states):
        """One token of ``len(states)`` requests: x [R, heads * width] (the block before's
        output, or the embedding with ``stream`` None) -> (x, stream) for the next block."""
        stream, (q, k, v), rest = self._operands(x, stream, (x.shape[0], 1))
        attention, _ = tao_attention_decode_batch(q, k, v, states=states, **rest)
        return self._close(attention, stream)

    @torch.no_grad()
    def prefill(self, x, stream, state):
        """A prompt chunk of one request: x [T, heads * width] -> (x, stream)."""
        stream, (q, k, v), rest = self._operands(x, stream, (1, x.shape[0]))
        attention, _ = tao_attention_prefill(q, k, v, state=state, position=state.position, **rest)
        return self._close(attention, stream)


def sorted_experts(x, ids, weights, gate, up, down):
    """A mixture-of-experts layer for many tokens, differentiable: x [tokens, channels], a router's choices ids
    [tokens, top_k] (outside of the experts: none) and their weights; gate and up [experts, inner, channels], down
    [experts, channels, inner].  out = sum over a token's choices of weight * down_e(silu(gate_e x) * (up_e x)),
    with what goes into down and what comes out of it rounded to x's type."""
    order = sort_tokens(ids, gate.shape[0])
    mid = expert_linear(gather_tokens(x, order), gate, order.offsets, up=up, activation="silu")
    return return_tokens(expert_linear(mid, down, order.offsets), order, weights)


class TrainedBlock(nn.Module):
    """One decoder block in training, its weights in bf16 (the attention's type):

        h, stream = norm(x + stream);  x = W_out attention(split(W_qkv h))
        h, stream = norm(x + stream);  x = experts(h), or dense: W_2 gelu(W_1 h + b_1) + b_2 + stream, stream None

    ``experts`` 0: the dense form, whose sum with the stream is rounded once.  ``transform`` (q, k) -> (q, k) is the
    caller's positional transform; ``eps`` is the residual norms'.  ``prefill`` and ``step`` take prompts and decode with the same weights."""

    def __init__(self, heads, width, inner, experts=0, top_k=2, renormalize=True, alpha=0.5, transform=None, eps=RMS_EPS,
                 config=DEFAULT_CONFIG, device="cuda", dtype=_BF16):
        super().__init__()
        channels = heads * width
        if experts < 0 or (experts and not 1 <= top_k <= experts):
            raise ValueError("a token takes 1 to as many experts as there are")
        if dtype != _BF16:
            raise ValueError("the block's weights are bf16, as what the attention takes")
        self.heads, self.width, self.experts, self.top_k, self.renormalize = heads, width, experts, top_k, renormalize
        self.alpha, self.transform, self.eps, self.config = alpha, transform, eps, config

        def weight(*shape):
            return nn.Parameter((torch.randn(*shape, device=device) * shape[-1] ** -0.5).to(dtype))

        self.norms = nn.ParameterList([nn.Parameter(torch.ones(channels, device=device, dtype=dtype)) for _ in range(2)])
        self.qkv, self.out = weight(3 * channels, channels), weight(channels, channels)
        self.fusion_a = nn.Parameter(torch.zeros(heads, width, 3, device=device))
        self.fusion_b = nn.Parameter(torch.zeros(heads, width, 3, device=device))
        if experts:
            self.router = weight(experts, channels)
            self.gate, self.up = weight(experts, inner, channels), weight(experts, inner, channels)
            self.down = weight(experts, channels, inner)
        else:
            self.first, self.second = weight(inner, channels), weight(channels, inner)
            self.first_bias = nn.Parameter(torch.zeros(inner, device=device, dtype=dtype))
            self.second_bias = nn.Parameter(torch.zeros(channels, device=device, dtype=dtype))

    def route(self, h):
        """(ids, weights) [tokens, top_k] of h [tokens, channels]."""
        weights, ids = torch.softmax(linear(h, self.router).float(), -1).topk(self.top_k, -1)
        return ids, weights / weights.sum(-1, keepdim=True) if self.renormalize else weights

    def _operands(self, x, stream):
        h, stream = add_rms_norm(x, self.norms[0], stream, eps=self.eps)
        q, k, v, raw_q, raw_k = split_norm(linear(h, self.qkv), self.heads, self.width)
        if self.transform is not None:
            q, k = self.transform(q, k)
        return stream, (q, k, v), {"raw_q": raw_q, "raw_k": raw_k, "fusion_a": self.fusion_a,
                                   "fusion_b": self.fusion_b, "alpha": self.alpha}

    def _close(self, attention, stream):
        x = linear(attention.reshape(stream.shape), self.out)
        h, stream = add_rms_norm(x, self.norms[1], stream, eps=self.eps)
        if not self.experts:
            mid = linear(h, self.first, self.first_bias, activation="gelu")
            return linear(mid, self.second, self.second_bias, residual=stream), None
        rows = h.reshape(-1, h.shape[-1])
        return sorted_experts(rows, *self.route(rows), self.gate, self.up, self.down).view(h.shape), stream

    def forward(self, x, stream=None):
        """Whole sequences x [batch, tokens, heads * width] -> (x, stream) for the next block."""
        stream, (q, k, v), rest = self._operands(x, stream)
        return self._close(tao_attention(q, k, v, config=self.config, **rest), stream)

    @torch.no_grad()
    def prefill(self, x, stream, state):
        """A prompt chunk of one request: x [1, tokens, heads * width] -> (x, stream)."""
        stream, (q, k, v), rest = self._operands(x, stream)
        attention, _ = tao_attention_prefill(q, k, v, state=state, position=state.position, **rest)
        return self._close(attention, stream)

    @torch.no_grad()
    def step(self, x, stream, states):
        """One token of ``len(states)`` requests: x [requests, 1, heads * width] -> (x, stream)."""
        stream, (q, k, v), rest = self._operands(x, stream)
        attention, _ = tao_attention_decode_batch(q, k, v, states=states, **rest)
        return self._close(attention, stream)


class TrainedDecoder(nn.Module):
    """``TrainedBlock``s between an embedding (scaled by the root of its channels) and a head with the same table."""

    def __init__(self, vocab, blocks, device="cuda", dtype=_BF16):
        super().__init__()
        self.blocks = nn.ModuleList(blocks)
        if dtype != _BF16:
            raise ValueError("the decoder's weights are bf16, as its blocks'")
        channels = blocks[0].heads * blocks[0].width
        self.scale, self.eps = channels ** 0.5, blocks[0].eps
        self.table = nn.Parameter((torch.randn(vocab, channels, device=device) / self.scale).to(dtype))
        self.norm = nn.Parameter(torch.ones(channels, device=device, dtype=dtype))

    def _check(self, requests):
        if any(len(states) != len(self.blocks) for states in requests):
            raise ValueError(f"a request has a state for each of the {len(self.blocks)} blocks")

    def _head(self, x, stream):
        return linear(add_rms_norm(x, self.norm, stream, eps=self.eps)[0], self.table)

    def forward(self, ids):
        """ids [batch, tokens] -> logits [batch, tokens, vocab]; an id outside of the vocabulary is padding."""
        x, stream = embed(ids, self.table, self.scale), None
        for block in self.blocks:
            x, stream = block(x, stream)
        return self._head(x, stream)

    @torch.no_grad()
    def prefill(self, ids, states):
        """A prompt [tokens] of one request, a state for each block: the last token's logits [1, vocab]."""
        self._check([states])
        x, stream = embed(ids[None], self.table, self.scale), None
        for block, state in zip(self.blocks, states):
            x, stream = block.prefill(x, stream, state)
        return self._head(x[0, -1:], None if stream is None else stream[0, -1:])

    @torch.no_grad()
    def step(self, ids, requests):
        """One token of each request, ids [requests], a sequence of states each: logits [requests, vocab]."""
        self._check(requests)
        x, stream = embed(ids[:, None], self.table, self.scale), None
        for layer, block in enumerate(self.blocks):
            x, stream = block.step(x, stream, [states[layer] for states in requests])
        return self._head(x[:, 0], None if stream is None else stream[:, 0])


__all__ = ["ProjectedInputs", "ServedBlock", "TrainedBlock", "TrainedDecoder", "sorted_experts", "split_norm", "RMS_EPS"]
