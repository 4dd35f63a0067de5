"""Sizes past what a launch can count are refused on the host."""
import ctypes

from salt_b200 import _lib

AT = 1 << 20


def test_conv_rows_have_fewer_threads_than_32_bits_count():
    """A row of 2^38 elements, whose threads (32 tokens of a channel each) number 2^33."""
    lib, dim, n = _lib.lib(), 255, (1 << 30) - 64
    a = _lib.CausalConvArgs(batch=1, len=n, dim=dim, width=4, out_stride=dim, x=AT, weight=AT, out=AT)
    assert lib.salt_causal_conv(ctypes.byref(a), None) == _lib.SALT_BAD_ARG
    assert b"too large" in lib.salt_last_error()
