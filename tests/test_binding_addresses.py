"""CPU tests of what the binding takes as an address: tensors, integers, numpy arrays, None - and
nothing whose memory is gone when the call runs."""
import ctypes as C

import numpy as np
import pytest
import torch

import paged_attn_b200 as pa


def test_addresses_of_what_a_call_passes():
    t = torch.zeros(8, 4)
    assert pa._ptr(t) == t.data_ptr() and pa._ptr(t[3:, 1:]) == t.data_ptr() + (3 * 4 + 1) * 4
    a = np.arange(24, dtype=np.int32).reshape(4, 6)
    for x in (a, a[1:, 2:], a[::2], a[:0], np.array(7), a.view(np.matrix)):
        assert pa._ptr(x) == x.ctypes.data
    assert pa._ptr(None) == 0 and pa._ptr(0) == 0 and pa._ptr(0x7f0012345678) == 0x7f0012345678


def test_an_object_with_an_address_of_its_own_kind():
    class Buffer:  # what numpy arrays are taken by, without being one
        def __init__(self):
            self.memory = (C.c_char * 16)()
            self.ctypes = type("Address", (), {"data": C.addressof(self.memory)})
    b = Buffer()
    assert pa._ptr(b) == C.addressof(b.memory)


@pytest.mark.parametrize("x", [np.int64(12345678), np.uint64(1 << 40), np.int32(7), np.float32(1.0), np.bool_(True)])
def test_numpy_scalars_are_refused(x):
    """They offer the address of a copy that is freed before a call could use it."""
    with pytest.raises(TypeError):
        pa._ptr(x)


@pytest.mark.parametrize("x", [1.5, "buffer", b"bytes", [1, 2], (3,), object()])
def test_everything_else_is_refused(x):
    with pytest.raises(TypeError):
        pa._ptr(x)


def test_a_temporary_array_interface_is_refused():
    class Temporary:  # an array made for the asking, as image objects do
        @property
        def __array_interface__(self):
            return np.arange(4).__array_interface__
    with pytest.raises(TypeError):
        pa._ptr(Temporary())
