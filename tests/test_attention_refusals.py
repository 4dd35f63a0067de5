"""What linear attention and the products in 8 bits refuse before anything is enqueued, on the Python
side and in the C ABI, and the ABI's struct layouts.  No device is needed: the checks come first."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from salt_b200 import _lib, sequence
from salt_b200 import device as D
from test_sequence_devices import on
from test_sequence_refusals import Views, fake

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F, H, I, E = np.float32, np.float16, np.int32, D.float8_e4m3

STRUCTS = {"salt_linear_attention_args": _lib.LinearAttentionArgs,
           "salt_linear_attention_step_args": _lib.LinearAttentionStepArgs,
           "salt_linear_attention_backward_args": _lib.LinearAttentionBackwardArgs,
           "salt_quantize_q8_args": _lib.QuantizeQ8Args,
           "salt_matmul_q8_args": _lib.MatmulQ8Args}


def test_struct_layouts_match_the_header(tmp_path):
    lines = [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for c, p in STRUCTS.items()
             for f, _ in p._fields_]
    lines += [f'printf("{c} - %zu\\n", sizeof({c}));' for c in STRUCTS]
    lines.append('printf("group - %d\\n", SALT_Q8_GROUP);')
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "salt_b200.h"\n'
                   "int main(void){\n" + "\n".join(lines) + "\nreturn 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        c, f, at = line.split()
        if c == "group":
            assert sequence.Q8_GROUP == int(at)
            continue
        got = ctypes.sizeof(STRUCTS[c]) if f == "-" else getattr(STRUCTS[c], f).offset
        assert got == int(at), line


def attention(**k):
    a = dict(q=fake((2, 9, 4, 16)), k=fake((2, 9, 2, 16)), v=fake((2, 9, 2, 8)),
             log_decay=fake((4,)), out=fake((2, 9, 4, 8)))
    return sequence.linear_attention(**{**a, **k})


def step(**k):
    a = dict(pool=fake((3, 4, 16, 8)), q=fake((2, 4, 16)), k=fake((2, 2, 16)), v=fake((2, 2, 8)),
             log_decay=fake((4,)), out=fake((2, 4, 8)))
    return sequence.linear_attention_step(**{**a, **k})


def backward(**k):
    a = dict(dout=fake((2, 9, 4, 8)), q=fake((2, 9, 4, 16)), k=fake((2, 9, 2, 16)),
             v=fake((2, 9, 2, 8)), log_decay=fake((4,)), dq=fake((2, 9, 4, 16)),
             dk=fake((2, 9, 2, 16)), dv=fake((2, 9, 2, 8)))
    return sequence.linear_attention_backward(**{**a, **k})


def quantize(**k):
    a = dict(x=fake((4, 200)), out=fake((4, 200), E), scale=fake((4, 2)))
    return sequence.quantize_q8(**{**a, **k})


def matmul(**k):
    a = dict(x=fake((4, 200), E), x_scale=fake((4, 2)), weight=fake((300, 200), E),
             weight_scale=fake((3, 2)), out=fake((4, 300)))
    return sequence.matmul_q8(**{**a, **k})


REFUSED = [
    (attention, dict(q=np.zeros((2, 9, 4, 16), F)), TypeError, "device array"),
    (attention, dict(q=fake((2, 9, 4, 16), I)), TypeError, "activations"),
    (attention, dict(q=fake((9, 4, 16))), ValueError, "4 axes"),
    (attention, dict(k=fake((2, 9, 2, 16), H)), TypeError, "k"),
    (attention, dict(k=fake((2, 9, 2, 8))), ValueError, "k"),
    (attention, dict(v=fake((2, 9, 4, 8))), ValueError, "v"),
    (attention, dict(k=fake((2, 9, 3, 16)), v=fake((2, 9, 3, 8))), ValueError, "kv_heads"),
    (attention, dict(q=fake((2, 9, 4, 160)), k=fake((2, 9, 2, 160))), ValueError, "dim_k"),
    (attention, dict(log_decay=fake((2,))), ValueError, "log_decay"),
    (attention, dict(log_decay=fake((4,), H)), TypeError, "log_decay"),
    (attention, dict(out=fake((2, 9, 4, 8), H)), TypeError, "out"),
    (attention, dict(q=Views((2, 9, 4, 16), (999, 99, 20, 1))), ValueError, "contiguous"),
    (attention, dict(q=Views((2, 9, 4, 16), (-576, 64, 16, 1))), ValueError, "negative"),
    (attention, dict(out=Views((2, 9, 4, 8), (288, 16, 8, 1))), ValueError, "overlap"),
    (attention, dict(n_real=fake((3,), I)), ValueError, "n_real"),
    (attention, dict(initial_state=fake((2, 4, 8, 16))), ValueError, "initial_state"),
    (attention, dict(initial_state=fake((2, 4, 16, 8), H)), TypeError, "initial_state"),
    (attention, dict(final_state=fake((2, 2, 16, 8))), ValueError, "final_state"),
    (attention, dict(scale=float("nan")), ValueError, "scale"),
    (step, dict(pool=fake((1, 4, 16, 8))), ValueError, "n_slots"),
    (step, dict(pool=fake((3, 4, 16, 8), H)), TypeError, "pool"),
    (step, dict(pool=fake((3, 2, 16, 8))), ValueError, "pool"),
    (step, dict(slots=fake((2,), np.int64)), TypeError, "slots"),
    (step, dict(q=fake((2, 9, 4, 16))), ValueError, "3 axes"),
    (step, dict(out=Views((2, 4, 8), (16, 8, 1))), ValueError, "out_stride"),
    (backward, dict(dout=fake((2, 9, 4, 16))), ValueError, "dout"),
    (backward, dict(dout=fake((2, 9, 4, 8), H)), TypeError, "dout"),
    (backward, dict(dk=fake((2, 9, 4, 16))), ValueError, "dk"),
    (backward, dict(dv=Views((2, 9, 2, 8), (0, 16, 8, 1))), ValueError, "overlap"),
    (backward, dict(dfinal=fake((2, 4, 8, 16))), ValueError, "dfinal"),
    (backward, dict(dinitial=fake((2, 4, 16, 8), H)), TypeError, "dinitial"),
    (quantize, dict(x=fake((4, 200), E)), TypeError, "activations"),
    (quantize, dict(out=fake((4, 200))), TypeError, "out"),
    (quantize, dict(scale=fake((4, 1))), ValueError, "scale"),
    (quantize, dict(blocks=True), ValueError, "scale"),
    (quantize, dict(transposed=True), ValueError, "out"),
    (quantize, dict(x=fake((2, 2, 200)), blocks=True), ValueError, "2 axes"),
    (quantize, dict(out=Views((4, 200), (100, 1), E)), ValueError, "out_stride"),
    (matmul, dict(x=fake((4, 200))), TypeError, "x"),
    (matmul, dict(x=np.zeros((4, 200), np.uint8)), TypeError, "device array"),
    (matmul, dict(x_scale=fake((4, 1))), ValueError, "x_scale"),
    (matmul, dict(x_scale=fake((4, 2), H)), TypeError, "x_scale"),
    (matmul, dict(weight=fake((300, 199), E)), ValueError, "weight"),
    (matmul, dict(weight_scale=fake((2, 2))), ValueError, "weight_scale"),
    (matmul, dict(weight_scale=fake((300, 1))), ValueError, "weight_scale"),
    (matmul, dict(bias=fake((299,))), ValueError, "bias"),
    (matmul, dict(bias=fake((300,), H)), TypeError, "bias"),
    (matmul, dict(out=fake((4, 300), I)), TypeError, "out"),
    (matmul, dict(out=fake((4, 299))), ValueError, "out"),
    (matmul, dict(out=Views((4, 300), (150, 1))), ValueError, "out_stride"),
]


@pytest.mark.parametrize("call, change, error, text", REFUSED,
                         ids=[f"{c[0].__name__}-{'-'.join(c[1])}-{i}"
                              for i, c in enumerate(REFUSED)])
def test_refusals(call, change, error, text):
    with pytest.raises(error, match=text):
        call(**change)


@pytest.mark.parametrize("call, name", [(attention, "k"), (attention, "log_decay"),
                                        (step, "pool"), (backward, "dout"), (quantize, "scale"),
                                        (matmul, "weight"), (matmul, "x_scale")])
def test_arrays_of_another_device_are_refused(monkeypatch, call, name):
    shapes = {"k": (2, 9, 2, 16), "log_decay": (4,), "pool": (3, 4, 16, 8), "dout": (2, 9, 4, 8),
              "scale": (4, 2), "weight": (300, 200), "x_scale": (4, 2)}
    monkeypatch.setattr(sequence, "_here", lambda: 0)
    a = on(1, *shapes[name])
    if name == "weight":
        a = D.DeviceArray(a.ptr, a.shape, E, a._owner)
    with pytest.raises(ValueError, match=f"{name}: not on the current device"):
        call(**{name: a})


def test_c_entries_refuse_null_sizes_and_small_workspaces():
    lib, n = _lib.lib(), ctypes.c_size_t(0)
    for name in ("salt_linear_attention_step", "salt_quantize_q8"):
        assert getattr(lib, name)(None, None) == _lib.SALT_BAD_ARG
        assert b"NULL" in lib.salt_last_error()
    for name in ("salt_linear_attention", "salt_linear_attention_backward", "salt_matmul_q8"):
        assert getattr(lib, name)(None, None, 0, None) == _lib.SALT_BAD_ARG
        assert getattr(lib, name + "_workspace_size")(None, ctypes.byref(n)) == _lib.SALT_BAD_ARG
    at = 1 << 20
    # heads that share a key head: the gradients' parts need room
    a = _lib.LinearAttentionBackwardArgs(1, 9, 4, 2, 16, 8, 0, 1.0, *(0, 64, 0, 32, 0, 16, 0, 32),
                                         *(0, 64, 0, 32, 0, 16), at, at, at, at, at, None, None,
                                         None, at, at, at, None)
    size = lib.salt_linear_attention_backward_workspace_size
    assert size(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value > 0
    assert size(ctypes.byref(a), None) == _lib.SALT_BAD_ARG
    run = lib.salt_linear_attention_backward
    assert run(ctypes.byref(a), None, 0, None) == _lib.SALT_WORKSPACE_TOO_SMALL
    assert run(ctypes.byref(a), at, n.value - 1, None) == _lib.SALT_WORKSPACE_TOO_SMALL
    assert run(ctypes.byref(a), at + 4, n.value, None) == _lib.SALT_BAD_ARG
    for field, bad in (("type", 3), ("len", -1), ("len", 2 ** 30 + 1), ("batch", -1), ("heads", 0),
                       ("kv_heads", 0), ("kv_heads", 3), ("dim_k", 0), ("dim_v", 129),
                       ("batch", 2 ** 23), ("scale", float("inf")), ("q_stride", -1),
                       ("dk_stride", 31), ("q", None), ("dq", None), ("log_decay", None)):
        old = getattr(a, field)
        setattr(a, field, bad)
        assert size(ctypes.byref(a), ctypes.byref(n)) == _lib.SALT_BAD_ARG, field
        setattr(a, field, old)
    m = _lib.MatmulQ8Args(4, 300, 200, 0, 0, 0, 200, 200, 300, at, at, at, at, None, at)
    size = lib.salt_matmul_q8_workspace_size
    assert size(ctypes.byref(m), ctypes.byref(n)) == 0
    for field, bad in (("type", 4), ("bias_type", 1), ("rows", -1), ("rows", 2 ** 31 - 1), ("n", 0), ("k", 0),
                       ("k", 2 ** 24 + 1), ("x_stride", -1), ("out_stride", 299), ("x", None),
                       ("weight_scale", None), ("out", None)):
        old = getattr(m, field)
        setattr(m, field, bad)
        assert size(ctypes.byref(m), ctypes.byref(n)) == _lib.SALT_BAD_ARG, field
        setattr(m, field, old)
    q = _lib.QuantizeQ8Args(4, 200, 0, 0, 0, 0, 200, 200, at, at, at)
    for field, bad in (("type", 4), ("rows", -1), ("rows", 2 ** 31 - 1), ("dim", 0),
                       ("dim", 2 ** 24 + 1), ("x_stride", -1), ("out_stride", 199), ("x", None),
                       ("scale", None)):
        old = getattr(q, field)
        setattr(q, field, bad)
        assert lib.salt_quantize_q8(ctypes.byref(q), None) == _lib.SALT_BAD_ARG, field
        setattr(q, field, old)
    m.type, m.bias_type, m.rows = 2, 1, 0  # without rows, too, and with a bias of neither type
    assert size(ctypes.byref(m), ctypes.byref(n)) == _lib.SALT_BAD_ARG
