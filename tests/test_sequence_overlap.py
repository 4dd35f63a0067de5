"""Outputs whose strides let two rows share elements are refused: threads would race for them.  Any
strides that keep rows apart are taken.  The queries of workspaces make the same checks as the calls
and launch nothing."""
import ctypes
import itertools

import numpy as np
import pytest

from salt_b200 import _lib, sequence
from salt_b200 import device as D

AT = 1 << 20


class Views:
    """A device array that is never read, with strides of its own."""

    def __init__(self, shape, strides):
        self.shape, self._strides, self.dtype = shape, strides, np.dtype(np.float32)

    def data_ptr(self):
        return AT

    def stride(self):
        return self._strides


def taken(batch, n, dim, batch_stride, stride):
    lib, size = _lib.lib(), ctypes.c_size_t(0)
    a = _lib.CausalConvBackwardArgs(
        batch=batch, len=n, dim=dim, width=4, dx_batch_stride=batch_stride, dx_stride=stride,
        x_stride=dim, dy_stride=dim, dy=AT, x=AT, weight=AT, dx=AT, dweight=AT)
    got = lib.salt_causal_conv_backward_workspace_size(ctypes.byref(a), ctypes.byref(size))
    if got:
        assert got == _lib.SALT_BAD_ARG and b"dx's strides" in lib.salt_last_error()
    return got == _lib.SALT_OK


def test_strides_that_keep_rows_apart():
    """Against all pairs of rows, for every pair of strides up to a little over the largest reach."""
    for batch, n, dim in ((1, 4, 3), (4, 1, 3), (2, 2, 3), (2, 5, 2), (4, 3, 2), (3, 3, 1)):
        for bs, ts in itertools.product(range(0, 5 * dim * 3), repeat=2):
            seen = [b * bs + t * ts + c for b in range(batch) for t in range(n) for c in range(dim)]
            want = len(set(seen)) == len(seen)
            assert taken(batch, n, dim, bs, ts) == want, (batch, n, dim, bs, ts)


def test_large_strides():
    assert taken(4, 1 << 20, 64, 1 << 62, 1 << 41)      # nothing here may pass 64 bits
    assert not taken(1 << 10, 1 << 20, 64, 64, 64)
    assert taken(1 << 10, 1 << 20, 64, 64, 64 << 10)    # tokens first
    assert not taken(1 << 10, 1 << 20, 64, 64, (64 << 10) - 64)


def test_refused_from_python():
    f = lambda *s: D.DeviceArray(AT, s, np.float32, None)  # noqa: E731
    with pytest.raises(ValueError, match="out's strides"):
        sequence.causal_conv(f(2, 9, 16), f(16, 4), out=Views((2, 9, 16), (16, 16, 1)))
    with pytest.raises(ValueError, match="out's strides"):
        sequence.selective_scan(f(2, 9, 16), f(2, 9, 16), f(16, 8), f(2, 9, 1, 8), f(2, 9, 1, 8),
                                out=Views((2, 9, 16), (32, 16, 1)))
