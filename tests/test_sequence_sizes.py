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


def test_scan_gradient_of_the_most_groups_and_states():
    """A token's dB and dC of 2^24 groups of 64 states would number 2^31."""
    lib, n = _lib.lib(), ctypes.c_size_t(0)
    for groups, want in ((1 << 24, _lib.SALT_BAD_ARG), (1 << 23, _lib.SALT_OK)):
        a = _lib.SelectiveScanBackwardArgs(
            batch=1, len=1, dim=1 << 24, state=64, groups=groups, dx_stride=1 << 24,
            **{k: AT for k in "x delta B C dy A checkpoints dx ddelta dB dC dA".split()})
        assert lib.salt_selective_scan_backward_workspace_size(ctypes.byref(a),
                                                               ctypes.byref(n)) == want
