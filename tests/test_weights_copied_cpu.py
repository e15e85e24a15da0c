"""Laid-out weights that are copied, saved or loaded: the library gets the addresses
of the tensors they hold."""
import copy
import io
import pickle

import pytest
import torch

from tao_memory_b200 import Weight4, quantize4


def _addresses(w):
    return (w.codes.data_ptr(), w.scales.data_ptr(), None if w.zeros is None else w.zeros.data_ptr())


def _weight(zeros=True):
    return quantize4(torch.randn(20, 200, generator=torch.Generator().manual_seed(0)), group=64, zeros=zeros)


def _round_trips(w):
    buf = io.BytesIO()
    torch.save(w, buf)
    buf.seek(0)
    return copy.deepcopy(w), pickle.loads(pickle.dumps(w)), torch.load(buf, weights_only=False)


def test_a_copied_weight_names_its_own_tensors():
    for zeros in (False, True):
        w = _weight(zeros)
        for other in _round_trips(w):
            assert isinstance(other, Weight4) and other.codes.data_ptr() != w.codes.data_ptr()
            assert other.args == (*_addresses(other), 64, 0) and other.shape == w.shape
            assert torch.equal(other.dequantize(), w.dequantize())
            assert other.dtype == w.dtype and other.device == w.device


def test_a_weights_tensors_stay_its_own():
    w, other = _weight(), _weight()
    for name in ("codes", "scales", "zeros"):
        with pytest.raises(AttributeError):
            setattr(w, name, getattr(other, name))
    w.codes.data = other.codes.clone()  # the same tensor with other memory
    assert w.args == (*_addresses(w), 64, 0) and w.args[0] != other.args[0]
