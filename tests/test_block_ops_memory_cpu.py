"""The block operators' memory, as far as no GPU is needed to see it: what the C entries refuse
before any CUDA call."""
import ctypes

from tao_memory_b200 import _lib


def _layer(**k):
    return _lib.TaoExperts(**{**dict(router=1 << 20, gate=1 << 20, up=1 << 20, down=1 << 20, gate_expert=64,
                                     gate_row=8, up_expert=64, up_row=8, down_expert=64, down_row=8, width=8, inner=8,
                                     experts=2, top_k=1, group=0, renormalize=1), **k})


def _experts(x, out, tokens=1, stride=8):
    # a workspace too small is refused last: no call here launches anything, whatever the machine
    return _lib.lib().tao_expert_layer(ctypes.byref(_layer()), x, stride, tokens, out, None, None, 1 << 21, 16, None)


def test_an_expert_layers_out_starts_on_8_bytes():
    # the sums' kernel stores 8 bytes at a time
    for offset in (1, 2, 4, 6, 10):
        assert _experts(16, (1 << 22) + offset) == _lib.TAO_ERR_ARG
        assert b"8 bytes" in _lib.lib().tao_last_error()


def _overlaps(x, y, rows=4, stride=128, x_type=0, x_scale=None, bias=None):
    """tao_linear4's refusal of a y [rows, 128] over its operands (only calls that it refuses are made here)."""
    rc = _lib.lib().tao_linear4(x, stride, x_type, x_scale, 1 << 20, 1 << 21, None, 128, 0, bias, rows, 128, 128, y,
                                None)
    return rc == _lib.TAO_ERR_ARG and b"overlap" in _lib.lib().tao_last_error()


def test_a_products_output_does_not_overlap_its_operands():
    # blocks write their part of y while others still read x: any overlap is a race
    x, size = 1 << 24, 4 * 128 * 2
    for y in (x, x + 2, x - 2, x + size - 2, x - size + 2):
        assert _overlaps(x, y), y - x
    # rows apart
    for off in (128 - 1, 2048 - 255, 2048, 2048 + 127):
        assert _overlaps(x, x + off * 2, rows=2, stride=2048), off
    assert _overlaps(x, x + 100, stride=0)  # one row for all
    # e4m3 rows, their scales, and the bias
    assert _overlaps(x, x + 4 * 128 - 2, x_type=3)
    assert _overlaps(x, x + 4096, x_type=3, x_scale=x + 4096 + size - 4)
    assert _overlaps(x, x + 4096, bias=x + 4096 + size - 2)


def test_an_expert_layers_output_does_not_overlap_a_later_launchs_tokens():
    # 64 tokens a launch: rows of a later one would be read after this one wrote them
    x, row = 1 << 24, 16

    def refused(out, tokens, stride=8):
        return _experts(x, out, tokens, stride) == _lib.TAO_ERR_ARG and b"overlap" in _lib.lib().tao_last_error()

    for out in (x + row, x - row, x + 199 * row, x - 199 * row):
        assert refused(out, 200), out - x
    assert refused(x, 200, stride=16) and refused(x, 200, stride=0)  # rows over others' rows
    # a launch writes after its last read of x; the same rows; rows next to each other
    for out, tokens in ((x, 64), (x + row, 64), (x, 200), (x + 200 * row, 200), (x - 200 * row, 200)):
        assert not refused(out, tokens), (out - x, tokens)


def test_operands_start_on_their_elements():
    """A misaligned address would be a fault of the GPU; each is refused (only such calls are made here)."""
    lib, arg, at = _lib.lib(), _lib.TAO_ERR_ARG, 1 << 20
    names = lambda rc: rc == arg and b"element" in lib.tao_last_error()

    def norm(type, fp8=False, **k):
        a = {**dict(x=at, r=at, w=at, s=at, y=at, scale=at), **k}
        head = (a["x"], 64, a["r"], 64, a["w"], 3, 64, type, 1e-6)
        if fp8:
            return lib.tao_add_rms_norm_fp8(*head, 0, a["s"], a["y"], a["scale"], None)
        return lib.tao_add_rms_norm(*head, a["s"], a["y"], None)

    for type, size in ((0, 2), (1, 2), (2, 4)):
        for name in ("x", "r", "w", "s"):
            assert names(norm(type, **{name: at + size // 2})) and names(norm(type, fp8=True, **{name: at + 1}))
        assert names(norm(type, y=at + 1)) and names(norm(type, fp8=True, scale=at + 2))
        room = 1 << 20
        back = dict(dy=at, ds=at, s=at, w=at, dx=at, dw=at, ws=at)
        for name in back:
            b = {**back, name: at + (2 if name == "ws" else size // 2)}
            assert names(lib.tao_add_rms_norm_backward(b["dy"], 64, b["ds"], 64, b["s"], 64, b["w"], 3, 64, type, 1e-6,
                                                       b["dx"], b["dw"], b["ws"], room, None)), (type, name)

    def product(x=at, x_type=0, x_scale=None, bias=None, y=1 << 22):
        return lib.tao_linear4(x, 128, x_type, x_scale, at, at, None, 128, 0, bias, 1, 16, 128, y, None)

    assert names(product(x=at + 1)) and names(product(y=at + 4097)) and names(product(bias=at + 9001))
    assert names(product(x_type=3, x_scale=at + 9002))

    def layer(ids=None, weights=None, error=None):
        return lib.tao_expert_layer(ctypes.byref(_layer(error=error)), at, 8, 1, 1 << 22, ids, weights, 1 << 21, 1 << 20,
                                    None)

    assert names(layer(at + 2, at)) and names(layer(at, at + 1)) and names(layer(error=at + 2))
