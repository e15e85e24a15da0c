"""Expert layers in a graph: the error word that outlives the graph's workspace, and what of the workspace
has to be zero."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def _layer(width=128, inner=64, experts=6, top_k=2):
    from tao_memory_b200 import ExpertWeights
    g = torch.Generator(device="cuda").manual_seed(5)
    n = lambda *s: (torch.randn(*s, device="cuda", generator=g) * s[-1] ** -0.5).bfloat16()
    return ExpertWeights(n(experts, width), n(experts, inner, width), n(experts, inner, width),
                         n(experts, width, inner), top_k=top_k)


def _captured(layer, x, before=None):
    from tao_memory_b200 import expert_layer
    expert_layer(x, layer)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if before is not None:
            before()
        y = expert_layer(x, layer)
    return graph, y


def test_a_captured_launchs_error_is_reported():
    """The word that a captured launch sets is set here by hand: a wait cannot be made to run out."""
    from tao_memory_b200 import _lib, expert_layer, experts
    from tao_memory_b200.stream import check_device
    layer = _layer()
    x = torch.randn(3, 128, device="cuda").bfloat16()
    graph, y = _captured(layer, x)
    graph.replay()
    assert check_device() == 0
    # the address that every launch of the layer gets is the word that the check reads
    word = experts._error_word(x.device)
    struct = ctypes.cast(layer.layer(), ctypes.POINTER(_lib.TaoExperts)).contents
    assert struct.error == word.data_ptr()
    word.fill_(1)
    graph.replay()  # a later replay does not clear it
    with pytest.raises(_lib.TaoError, match="did not meet"):
        check_device()
    assert check_device() == 0 and int(word) == 0
    graph.replay()
    assert torch.equal(y, expert_layer(x, layer))


@pytest.mark.parametrize("tokens", [1, 9, 100])
def test_a_captured_launch_needs_no_more_than_its_header_zeroed(tokens):
    """The graph's workspace lies where the graph itself left other things before."""
    from tao_memory_b200 import expert_layer
    layer = _layer()
    x = torch.randn(tokens, 128, device="cuda").bfloat16()

    def junk():
        for size in (layer._workspace_bytes, 16 << 20):
            torch.full((size,), 255, device="cuda", dtype=torch.uint8)

    graph, y = _captured(layer, x, junk)
    for seed in range(3):
        x.copy_(torch.randn(tokens, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)))
        graph.replay()
        assert torch.equal(y, expert_layer(x, layer))


def test_an_error_survives_its_workspace():
    """A workspace that a larger one replaces takes its own word with it; the device's stays."""
    from tao_memory_b200 import _lib, expert_layer, experts
    from tao_memory_b200.stream import check_device
    small = _layer()
    x = torch.randn(2, 128, device="cuda").bfloat16()
    with torch.cuda.stream(torch.cuda.Stream()):
        expert_layer(x, small)
        experts._error_word(x.device).fill_(1)
        large = _layer(1024, 512, 8, 8)
        expert_layer(torch.randn(2, 1024, device="cuda").bfloat16(), large)
    with pytest.raises(_lib.TaoError, match="did not meet"):
        check_device()
    assert check_device() == 0


def test_a_workspace_is_reset_when_its_check_returns():
    """A launch on another stream may use it at once."""
    from tao_memory_b200 import _lib
    room = torch.full((1 << 30,), 7, device="cuda", dtype=torch.uint8)  # its reset takes 100 us and more
    room[:4] = torch.tensor([1, 0, 0, 0], dtype=torch.uint8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    flags = ctypes.c_int(0)
    rc = _lib.lib().tao_expert_check(room.data_ptr(), room.numel(), ctypes.byref(flags), side.cuda_stream)
    done = side.query()
    assert rc == _lib.TAO_ERR_DEVICE and flags.value == 1 and done
    assert not room.any()


@pytest.mark.parametrize("device", ["cuda", "cuda:0", 0, None])
def test_a_device_without_its_index_is_the_current_one(device):
    from tao_memory_b200 import _lib, experts
    from tao_memory_b200.stream import check_device
    _layer()
    assert check_device(device) == 0
    experts._error_word(torch.device("cuda", 0)).fill_(1)
    with pytest.raises(_lib.TaoError, match="did not meet"):
        check_device(device)
    assert check_device(device) == 0
