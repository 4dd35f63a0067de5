"""Calls without rows or tokens still launch what writes their other outputs (gradients of weights
become zero, final states the initial ones).  What such a launch reads has to be there: NULL is
refused on the host, before anything is enqueued."""
import ctypes

import numpy as np
import pytest

from salt_b200 import _lib, sequence
from salt_b200 import device as D

F = np.float32
AT = 1 << 20


def fake(shape, dtype=F):
    return D.DeviceArray(AT, shape, dtype, None)


def refused(name, args, text):
    """Both entries of a call with a workspace, or the one of a call without, say which."""
    lib, n = _lib.lib(), ctypes.c_size_t(0)
    assert getattr(lib, name + "_workspace_size")(ctypes.byref(args), ctypes.byref(n)) == \
        _lib.SALT_BAD_ARG
    assert text in lib.salt_last_error()
    assert getattr(lib, name)(ctypes.byref(args), AT, 1 << 40, None) == _lib.SALT_BAD_ARG
    assert text in lib.salt_last_error()


def test_norm_backward_of_no_rows_needs_its_weight():
    a = _lib.RmsNormBackwardArgs(rows=0, dim=64, dweight=AT)
    refused("salt_rms_norm_backward", a, b"weight is NULL")
    with pytest.raises(ValueError, match="weight is NULL"):
        sequence.rms_norm_backward(fake((0, 64)), fake((0, 64)), None, fake((0,)),
                                   dx=fake((0, 64)), dweight=fake((64,)))


def test_conv_backward_of_no_tokens_needs_its_weight():
    a = _lib.CausalConvBackwardArgs(batch=2, len=0, dim=16, width=4, dweight=AT)
    refused("salt_causal_conv_backward", a, b"weight is NULL")


def test_scan_of_no_tokens_needs_its_decay():
    a = _lib.SelectiveScanArgs(batch=2, len=0, dim=16, state=8, groups=1)
    refused("salt_selective_scan", a, b"A is NULL")
    with pytest.raises(ValueError, match="A is NULL"):
        sequence.selective_scan(fake((2, 0, 16)), fake((2, 0, 16)), None, fake((2, 0, 1, 8)),
                                fake((2, 0, 1, 8)), out=fake((2, 0, 16)))


def test_scan_backward_of_no_tokens_needs_its_decay():
    a = _lib.SelectiveScanBackwardArgs(batch=2, len=0, dim=16, state=8, groups=1, dA=AT)
    refused("salt_selective_scan_backward", a, b"A is NULL")
