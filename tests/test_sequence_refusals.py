"""What the sequence operators refuse before anything is enqueued, on the Python side and in the C
ABI, and the ABI's struct layouts.  No device is needed: the checks come first."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from salt_b200 import _lib, sequence
from salt_b200 import device as D

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F, I = np.float32, np.int32

STRUCTS = {"salt_rms_norm_args": _lib.RmsNormArgs,
           "salt_rms_norm_backward_args": _lib.RmsNormBackwardArgs,
           "salt_causal_conv_args": _lib.CausalConvArgs,
           "salt_causal_conv_step_args": _lib.CausalConvStepArgs,
           "salt_causal_conv_backward_args": _lib.CausalConvBackwardArgs,
           "salt_selective_scan_args": _lib.SelectiveScanArgs,
           "salt_selective_scan_step_args": _lib.SelectiveScanStepArgs,
           "salt_selective_scan_backward_args": _lib.SelectiveScanBackwardArgs}


def test_struct_layouts_match_the_header(tmp_path):
    lines = [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for c, p in STRUCTS.items()
             for f, _ in p._fields_]
    lines += [f'printf("{c} - %zu\\n", sizeof({c}));' for c in STRUCTS]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "salt_b200.h"\n'
                   "int main(void){\n" + "\n".join(lines) + "\nreturn 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        c, f, at = line.split()
        got = ctypes.sizeof(STRUCTS[c]) if f == "-" else getattr(STRUCTS[c], f).offset
        assert got == int(at), line
    assert sequence.CHECKPOINT == 16


def fake(shape, dtype=F):
    """An array that is never read: the checks look at its shape and type."""
    return D.DeviceArray(1 << 20, shape, dtype, None)


class Views:
    """A device array with strides of its own."""

    def __init__(self, shape, strides, dtype=F):
        self.shape, self._strides, self.dtype = shape, strides, np.dtype(dtype)

    def data_ptr(self):
        return 1 << 20

    def stride(self):
        return self._strides


def norm(**k):
    a = dict(x=fake((4, 64)), weight=fake((64,)))
    return sequence.rms_norm(**{**a, "out": fake((4, 64)), **k})


def norm_q8(**k):
    a = dict(x=fake((4, 64)), weight=fake((64,)), out=fake((4, 64), D.float8_e4m3),
             scale=fake((4, 2)), group=32)
    return sequence.rms_norm_q8(**{**a, **k})


def norm_backward(**k):
    a = dict(dy=fake((4, 64)), x=fake((4, 64)), weight=fake((64,)), rstd=fake((4,)),
             dx=fake((4, 64)), dweight=fake((64,)))
    return sequence.rms_norm_backward(**{**a, **k})


def conv(**k):
    a = dict(x=fake((2, 9, 16)), weight=fake((16, 4)), out=fake((2, 9, 16)))
    return sequence.causal_conv(**{**a, **k})


def conv_step(**k):
    a = dict(x=fake((2, 16)), state=fake((3, 16, 3)), weight=fake((16, 4)), out=fake((2, 16)))
    return sequence.causal_conv_step(**{**a, **k})


def conv_backward(**k):
    a = dict(dy=fake((2, 9, 16)), x=fake((2, 9, 16)), weight=fake((16, 4)), dx=fake((2, 9, 16)),
             dweight=fake((16, 4)))
    return sequence.causal_conv_backward(**{**a, **k})


def scan(**k):
    a = dict(x=fake((2, 9, 16)), delta=fake((2, 9, 16)), A=fake((16, 8)), B=fake((2, 9, 2, 8)),
             C=fake((2, 9, 2, 8)), out=fake((2, 9, 16)))
    return sequence.selective_scan(**{**a, **k})


def scan_step(**k):
    a = dict(pool=fake((3, 16, 8)), x=fake((2, 16)), delta=fake((2, 16)), A=fake((16, 8)),
             B=fake((2, 2, 8)), C=fake((2, 2, 8)), out=fake((2, 16)))
    return sequence.selective_scan_step(**{**a, **k})


def scan_backward(**k):
    a = dict(dy=fake((2, 9, 16)), x=fake((2, 9, 16)), delta=fake((2, 9, 16)), A=fake((16, 8)),
             B=fake((2, 9, 2, 8)), C=fake((2, 9, 2, 8)), checkpoints=fake((2, 1, 16, 8)),
             dx=fake((2, 9, 16)), ddelta=fake((2, 9, 16)), dA=fake((16, 8)),
             dB=fake((2, 9, 2, 8)), dC=fake((2, 9, 2, 8)))
    return sequence.selective_scan_backward(**{**a, **k})


REFUSED = [
    (norm, dict(x=np.zeros((4, 64), F)), TypeError, "device array"),
    (norm, dict(x=fake((4, 64), np.float64)), TypeError, "unsupported type"),
    (norm, dict(x=fake((4, 64), I)), TypeError, "activations"),
    (norm, dict(weight=fake((63,))), ValueError, "weight"),
    (norm, dict(weight=fake((64,), np.float16)), TypeError, "weight"),
    (norm, dict(residual=fake((4, 64), np.float16)), TypeError, "residual"),
    (norm, dict(residual=fake((3, 64))), ValueError, "residual"),
    (norm, dict(out=fake((4, 64), np.float16)), TypeError, "out"),
    (norm, dict(out=fake((4, 63))), ValueError, "out"),
    (norm, dict(rstd=fake((5,))), ValueError, "rstd"),
    (norm, dict(x=Views((4, 64), (64, 2))), ValueError, "contiguous"),
    (norm, dict(out=Views((4, 64), (32, 1))), ValueError, "out_stride"),
    (norm, dict(x=Views((2, 2, 64), (999, 64, 1)), out=fake((2, 2, 64))), ValueError, "fold"),
    (norm, dict(eps=-1.0), ValueError, "eps"),
    (norm, dict(x=fake((1, 20000)), weight=fake((20000,)), out=fake((1, 20000))), ValueError,
     "16384"),
    (norm_q8, dict(group=48), ValueError, "group"),
    (norm_q8, dict(scale=fake((4, 1))), ValueError, "scale"),
    (norm_q8, dict(out=fake((4, 64))), TypeError, "out"),
    (norm_backward, dict(x=fake((4, 64), np.float16)), TypeError, "x"),
    (norm_backward, dict(rstd=fake((4,), np.float16)), TypeError, "rstd"),
    (norm_backward, dict(dx=fake((4, 65))), ValueError, "dx"),
    (conv, dict(x=fake((9, 16))), ValueError, "3 axes"),
    (conv, dict(weight=fake((16, 9))), ValueError, "width"),
    (conv, dict(weight=fake((15, 4))), ValueError, "weight"),
    (conv, dict(bias=fake((15,))), ValueError, "bias"),
    (conv, dict(weight=fake((16, 4), np.float16)), TypeError, "weight"),
    (conv, dict(n_real=fake((2,), np.int64)), TypeError, "n_real"),
    (conv, dict(n_real=fake((3,), I)), ValueError, "n_real"),
    (conv, dict(initial_state=fake((2, 16, 4))), ValueError, "initial_state"),
    (conv, dict(out=Views((2, 9, 16), (144, 8, 1))), ValueError, "out"),
    (conv, dict(x=Views((2, 9, 16), (-144, 16, 1))), ValueError, "negative"),
    (conv_step, dict(state=fake((1, 16, 3))), ValueError, "n_slots"),
    (conv_step, dict(state=fake((3, 16, 3), np.float16)), TypeError, "state"),
    (conv_step, dict(slots=fake((3,), I)), ValueError, "slots"),
    (conv_backward, dict(dy=fake((2, 9, 16), np.float16)), TypeError, "dy"),
    (conv_backward, dict(dweight=fake((16, 3))), ValueError, "dweight"),
    (scan, dict(delta=fake((2, 9, 15))), ValueError, "delta"),
    (scan, dict(z=fake((2, 8, 16))), ValueError, "z"),
    (scan, dict(A=fake((16, 8), np.float16)), TypeError, "A"),
    (scan, dict(A=Views((16, 8), (1, 16))), ValueError, "contiguous"),
    (scan, dict(B=fake((2, 9, 3, 8)), C=fake((2, 9, 3, 8))), ValueError, "groups"),
    (scan, dict(A=fake((16, 65)), B=fake((2, 9, 1, 65)), C=fake((2, 9, 1, 65))), ValueError,
     "state"),
    (scan, dict(C=fake((2, 9, 1, 8))), ValueError, "C"),
    (scan, dict(B=Views((2, 9, 2, 8), (144, 16, 16, 1))), ValueError, "contiguous"),
    (scan, dict(initial_state=fake((2, 16, 8), np.float16)), TypeError, "initial_state"),
    (scan, dict(checkpoints=fake((2, 2, 16, 8))), ValueError, "checkpoints"),
    (scan_step, dict(pool=fake((1, 16, 8))), ValueError, "n_slots"),
    (scan_step, dict(pool=fake((3, 16, 8), np.float16)), TypeError, "pool"),
    (scan_step, dict(B=fake((2, 16))), ValueError, "3 axes"),
    (scan_backward, dict(checkpoints=fake((2, 2, 16, 8))), ValueError, "checkpoints"),
    (scan_backward, dict(dB=fake((2, 9, 2, 8), np.float16)), TypeError, "dB"),
    (scan_backward, dict(dx=Views((2, 9, 16), (0, 16, 1))), ValueError, "strides"),
]


@pytest.mark.parametrize("call, change, error, text", REFUSED,
                         ids=[f"{c[0].__name__}-{'-'.join(c[1])}-{i}"
                              for i, c in enumerate(REFUSED)])
def test_refusals(call, change, error, text):
    with pytest.raises(error, match=text):
        call(**change)


def test_c_entries_refuse_null_and_small_workspaces():
    lib = _lib.lib()
    for name in ("salt_rms_norm", "salt_causal_conv", "salt_causal_conv_step",
                 "salt_selective_scan_step"):
        assert getattr(lib, name)(None, None) == _lib.SALT_BAD_ARG
        assert b"NULL" in lib.salt_last_error()
    n = ctypes.c_size_t(0)
    a = _lib.RmsNormBackwardArgs(8, 64, 0, 0, 0, 0, 64, 64, 0, 64, 1 << 20, 1 << 20, 1 << 20,
                                 1 << 20, None, 1 << 20, 1 << 20)
    assert lib.salt_rms_norm_backward_workspace_size(ctypes.byref(a), ctypes.byref(n)) == 0
    assert n.value > 0
    assert lib.salt_rms_norm_backward(ctypes.byref(a), None, 0, None) == \
        _lib.SALT_WORKSPACE_TOO_SMALL
    assert str(n.value).encode() in lib.salt_last_error()
    assert lib.salt_rms_norm_backward(ctypes.byref(a), (1 << 20) + 4, n.value, None) == \
        _lib.SALT_BAD_ARG
    a.dx = None
    assert lib.salt_rms_norm_backward(ctypes.byref(a), 1 << 20, n.value, None) == \
        _lib.SALT_BAD_ARG
    for bad in (3, -1):
        a.type = bad
        assert lib.salt_rms_norm_backward_workspace_size(ctypes.byref(a), ctypes.byref(n)) == \
            _lib.SALT_BAD_ARG
    s = _lib.SelectiveScanArgs(1, 2 ** 30 + 1, 16, 16, 1, 0, 1, 0)
    assert lib.salt_selective_scan_workspace_size(ctypes.byref(s), ctypes.byref(n)) == \
        _lib.SALT_BAD_ARG
    s = _lib.SelectiveScanArgs(1 << 20, 1 << 20, 4096, 16, 1, 0, 1, 0)
    assert lib.salt_selective_scan_workspace_size(ctypes.byref(s), ctypes.byref(n)) == \
        _lib.SALT_BAD_ARG


def test_a_refused_call_takes_no_other_type_for_its_own():
    """numpy has no bfloat16: uint16 bits are not taken for it."""
    with pytest.raises(TypeError):
        norm(x=fake((4, 64), np.uint16))
