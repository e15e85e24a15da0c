"""B200-native (sm_100a) TaoMemory attention operator.

Drop-in for the reference package's public API (``tao_attention/__init__.py``):
``new_state``, ``tao_attention``, ``tao_attention_prefill``,
``tao_attention_decode``, ``StreamCache`` and ``TaoConfig``; plus
``tao_attention_decode_batch`` for many requests per launch, and
``copy_to_device`` / ``copy_to_host`` for a decode step's operands in page-locked
host memory, ``DecodeSession`` for a serving loop over a fixed batch whose
tokens arrive in and leave through page-locked host memory, and the serving caller
(``RequestStates``, ``DecodeScheduler``, ``save_snapshot`` / ``load_snapshot``);
``tao_memory_b200.model`` holds the model-side neighbours (``ProjectedInputs``, ``ServedBlock``).
Around the attention stand ``add_rms_norm`` / ``add_rms_norm_fp8``, ``linear4`` on 4-bit
``Weight4`` (``quantize4``) and ``expert_layer`` on ``ExpertWeights``; for training and prompts,
with gradients, ``embed``, ``linear`` and ``expert_linear`` over tokens sorted by expert
(``sort_tokens``, ``gather_tokens``, ``return_tokens``).  All compute runs in ``libtao_b200.so`` (hand-written CUDA for sm_100a) behind a C ABI.
"""

from .config import TaoConfig
from .embedding import embed
from .experts import ExpertWeights, expert_layer
from .host_io import copy_to_device, copy_to_host
from .linear import expert_linear, linear
from .linear4 import Weight4, linear4, quantize4
from .norm import add_rms_norm, add_rms_norm_fp8
from .operator import (new_state, tao_attention, tao_attention_decode,
                       tao_attention_decode_batch, tao_attention_prefill)
from .serving import DecodeScheduler, RequestStates, load_snapshot, save_snapshot
from .stream import DecodeSession, StreamCache
from .tokens import TokenOrder, gather_tokens, return_tokens, sort_tokens

__all__ = ["new_state", "tao_attention", "tao_attention_prefill",
           "tao_attention_decode", "tao_attention_decode_batch", "StreamCache",
           "TaoConfig", "copy_to_device", "copy_to_host", "DecodeSession", "RequestStates",
           "DecodeScheduler", "save_snapshot", "load_snapshot", "add_rms_norm", "add_rms_norm_fp8",
           "Weight4", "quantize4", "linear4", "ExpertWeights", "expert_layer",
           "linear", "expert_linear", "TokenOrder", "sort_tokens", "gather_tokens", "return_tokens", "embed"]
