"""Mixture-of-experts layer for the few tokens of a decode step: routing, the chosen experts'
gate, up and down products and their weighted sum in one kernel, whose time is the time to
read the chosen experts.  Weights in bf16 or 4 bits (``Weight4`` stacks).
"""

import ctypes

import torch

from . import _lib
from .linear4 import Weight4
from .norm import _rows, refuse_derivatives

_BF16 = torch.bfloat16
_TOKENS = 64  # of one launch
_HEADER = 256  # bytes of a workspace that have to be zero at first


class ExpertWeights:
    """One layer's router and experts: router [experts, width] bf16; gate, up [experts, inner,
    width] and down [experts, width, inner], all bf16 tensors (views of a fused tensor are taken
    as they are where their rows start on 16 bytes) or all ``Weight4`` stacks of one group and
    kind.  ``renormalize``: the chosen experts' softmax weights are divided by their sum.  May be
    copied, saved and loaded; its tensors cannot be exchanged."""

    def __init__(self, router, gate, up, down, top_k, renormalize=True):
        four = [isinstance(w, Weight4) for w in (gate, up, down)]
        if any(four) and not all(four):
            raise ValueError("gate, up and down are all bf16 tensors or all Weight4 stacks")
        if router.dim() != 2 or len(gate.shape) != 3:
            raise ValueError("the router is [experts, width] and experts are stacked [experts, ...]")
        experts, width = router.shape
        inner = gate.shape[1]
        if (tuple(gate.shape) != (experts, inner, width) or tuple(up.shape) != (experts, inner, width)
                or tuple(down.shape) != (experts, width, inner)):
            raise ValueError("gate and up are [experts, inner, width], down [experts, width, inner]")
        if any(t.dtype != _BF16 for t in (router, gate, up, down)):
            raise ValueError("the expert layer takes bf16 weights (4-bit: bf16 scales)")
        if not router.is_cuda or any(t.device != router.device for t in (gate, up, down)):
            raise ValueError("the expert layer's weights are on one CUDA device (no CPU fallback)")
        if all(four) and (len({w.group for w in (gate, up, down)}) > 1
                          or len({w.zeros is None for w in (gate, up, down)}) > 1):
            raise ValueError("4-bit experts share one group size, and have zero points all or none")
        if not 1 <= top_k <= experts:
            raise ValueError("top_k is 1 to 16 and at most the number of experts")
        self.width, self.inner, self.experts, self.top_k = width, inner, experts, top_k
        self.renormalize, self.device = bool(renormalize), router.device
        if not all(four):
            gate, up, down = (_aligned(w) for w in (gate, up, down))
        router = _aligned(router)
        if router.stride(0) != width:
            router = router.contiguous()
        self._weights = router, gate, up, down
        self._four, self._layer_at = all(four), None
        self._error = _error_word(self.device)
        lib = _lib.lib()
        self._workspace_bytes = lib.tao_expert_workspace_bytes(self.layer(), _TOKENS)
        if self._workspace_bytes == 0:
            _lib.check(_lib.TAO_ERR_ARG)

    router = property(lambda self: self._weights[0])
    gate = property(lambda self: self._weights[1])
    up = property(lambda self: self._weights[2])
    down = property(lambda self: self._weights[3])

    @property
    def floats(self):
        """The tensors that a derivative could be taken of."""
        router, *weights = self._weights
        return (router, *(w.scales if self._four else w for w in weights))

    def layer(self):
        """What tao_expert_layer takes of it, of the tensors as they are now."""
        router, *weights = self._weights
        if self._four:
            at = (router.data_ptr(), *(p for i in range(3) for p in (w.args[i] for w in weights)))
        else:
            at = (router.data_ptr(), *(w.data_ptr() for w in weights))
        if at != self._layer_at:
            strides = [0] * 6 if self._four else [s for w in weights for s in w.stride()[:2]]
            self._layer = _lib.TaoExperts(*at, *(None,) * (10 - len(at)), *strides, self.width, self.inner,
                                          self.experts, self.top_k, weights[0].group if self._four else 0,
                                          int(self.renormalize), self._error.data_ptr())
            self._layer_at = at
        return ctypes.byref(self._layer)

    def __getstate__(self):
        return (*self._weights, self.top_k, self.renormalize)

    def __setstate__(self, state):
        self.__init__(*state)


def _aligned(t):
    """``t`` with a contiguous last axis and rows that start on 16 bytes."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in t.stride()[:-1])
    return t if ok else t.clone(memory_format=torch.contiguous_format)


_ERRORS = {}


def _error_word(device):
    """The device's word of waits that ran out, which outlives workspaces and the graphs that hold one."""
    if device not in _ERRORS:
        _ERRORS[device] = torch.zeros(1, dtype=torch.int32, device=device)
    return _ERRORS[device]


class _Room:
    """Workspaces of the expert layer: zeroed once, one for a device and stream, so calls on
    two streams do not meet in one; a captured call gets one of its own, whose header its graph
    zeroes."""

    cache = {}

    @classmethod
    def get(cls, device, stream, nbytes):
        if torch.cuda.is_current_stream_capturing():
            buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
            buf[:_HEADER].zero_()
            return buf
        buf = cls.cache.get((device, stream))
        if buf is None or buf.numel() < nbytes:
            buf = cls.cache[(device, stream)] = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        return buf

    @classmethod
    def on_device(cls, device):
        return [b for (d, _), b in list(cls.cache.items()) if d == device]


def expert_layer(x, weights, out=None, return_routing=False):
    """sum over the ``top_k`` experts of a token of weight * down(silu(gate x) * (up x)): x
    [..., width] bf16 -> [..., width] bf16.  With ``return_routing`` also the chosen experts
    [..., top_k] int32 (most probable first, ties to the lowest) and their weights in fp32.

    One launch for 64 tokens; made for the few tokens of a decode step, it reads the chosen
    experts again for each 64 more.  ``out`` may be x itself; with more than 64 tokens it must not
    overlap x otherwise.  No gradient."""
    if not isinstance(weights, ExpertWeights):
        raise ValueError("expert_layer takes ExpertWeights")
    if x.dtype != _BF16 or not x.is_cuda or x.device != weights.device:
        raise ValueError("expert_layer takes bf16 CUDA activations on the weights' device (no CPU fallback)")
    if x.dim() == 0 or x.shape[-1] != weights.width:
        raise ValueError(f"activations have {weights.width} channels, as the layer")
    refuse_derivatives("expert_layer", x, *weights.floats)
    rows = _rows(x, weights.width)
    if rows.data_ptr() % 16 or rows.stride(0) % 8:
        rows = rows.clone(memory_format=torch.contiguous_format)
    result = out
    if out is None:
        out = result = x.new_empty(x.shape)
    elif out.shape != x.shape or out.dtype != _BF16 or out.device != x.device or not out.is_contiguous():
        raise ValueError("out is a contiguous tensor of x's shape, type and device")
    elif out.data_ptr() % 8:  # the kernel stores 8 bytes at a time
        result = x.new_empty(x.shape)
    ids = route = ids_at = route_at = None
    if return_routing:
        ids = x.new_empty((*x.shape[:-1], weights.top_k), dtype=torch.int32)
        route = x.new_empty(ids.shape, dtype=torch.float32)
        ids_at, route_at = ids.data_ptr(), route.data_ptr()
    device = x.device.index
    ws = _Room.get(x.device, torch._C._cuda_getCurrentRawStream(device), weights._workspace_bytes)
    _lib.on_device(device, _lib.lib().tao_expert_layer, weights.layer(), rows.data_ptr(), rows.stride(0), rows.shape[0],
                   result.data_ptr(), ids_at, route_at, ws.data_ptr(), ws.numel())
    if result is not out:
        out.copy_(result)
    return (out, ids, route) if return_routing else out


def check_workspaces(device):
    """Raise if an expert layer on ``device``, in a graph or not, reported an error since the last check
    (part of ``stream.check_device``; the device is synchronised)."""
    stream = torch.cuda.current_stream(device).cuda_stream
    failed = False
    for ws in _Room.on_device(device):
        rc = _lib.lib().tao_expert_check(ws.data_ptr(), ws.numel(), None, stream)
        if rc != _lib.TAO_ERR_DEVICE:
            _lib.check(rc)
        failed |= rc != _lib.TAO_OK
    if device in _ERRORS and int(_ERRORS[device]):
        _ERRORS[device].zero_()
        failed = True
    if failed:  # said once, with every word cleared
        raise _lib.TaoError("an expert layer's blocks did not meet in time")


__all__ = ["ExpertWeights", "expert_layer"]
