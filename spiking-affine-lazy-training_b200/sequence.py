"""Sequence operators: root-mean-square norm, short causal convolution, selective state space scan.

The dense, trained counterpart of the float layers' affine scan, for sequences of feature vectors
(binned spike counts, tokens): ``h = exp(s A) h + s x B`` with a step ``s``, an input map ``B`` and
a readout ``C`` that depend on the token.  Each operator runs over whole rows, for single tokens on
a pool of states, and backward, as one call of the C ABI (include/salt_b200.h, "sequence operators")
on the current stream; no CPU fallback.  No reference counterpart.

Arrays are `DeviceArray`s or any object of another library with ``data_ptr()``, ``shape``,
``dtype`` and ``stride()`` (in elements) that lives on the current device.  Activations are float32,
float16 or bfloat16 (`device.bfloat16`), (batch, len, dim) with contiguous channels and any token
and batch strides; weights of the norm and the convolution hold that type or float32; the scan's
``A``, ``D``, ``delta_bias`` and its states are float32.  Every output is written into the array
given for it, or into a new `DeviceArray` where none is; an optional output takes ``None`` (not
wanted), ``True`` (make one) or an array.  Calls work on the arrays' memory alone: another library's
automatic differentiation does not see them, and gradients come from the `*_backward` calls.

Streams: a call enqueues on `device.current_stream()` and orders nothing else.  Arrays that another
stream writes have to be waited for (`Stream.wait_event`, `Stream.external`), and must stay
allocated until the call's work is done.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import NamedTuple

import numpy as np

from . import _lib
from .device import DeviceArray, _tls, bfloat16, empty, float8_e4m3

CHECKPOINT = 16       # tokens between the scan's checkpoints (SALT_SCAN_CHECKPOINT)
GROUPS_8BIT = (0, 32, 64, 128, 256)
_F32, _F16, _BF16, _I32, _E4M3 = range(5)
_NUMPY = {_F32: np.dtype(np.float32), _F16: np.dtype(np.float16), _BF16: bfloat16,
          _I32: np.dtype(np.int32), _E4M3: float8_e4m3}
_NAMES = ("float32", "float16", "bfloat16", "int32", "float8_e4m3")
_TYPE_IDS = {v: k for k, v in _NUMPY.items()}
_ACTIVATIONS = (_F32, _F16, _BF16)


class NormOutput(NamedTuple):
    out: object
    residual: object = None
    rstd: object = None
    scale: object = None


class NormGradients(NamedTuple):
    dx: object
    dweight: object = None


class ConvOutput(NamedTuple):
    out: object
    final_state: object = None


class ConvGradients(NamedTuple):
    dx: object
    dweight: object
    dbias: object = None
    dinitial: object = None


class ScanOutput(NamedTuple):
    out: object
    final_state: object = None
    checkpoints: object = None


class ScanGradients(NamedTuple):
    dx: object
    ddelta: object
    dA: object
    dB: object
    dC: object
    dD: object = None
    dz: object = None
    ddelta_bias: object = None
    dinitial: object = None


# ---------------------------------------------------------------- arguments

def _type_of(a, name: str) -> int:
    t = a.dtype
    got = _TYPE_IDS.get(t)
    if got is None:
        text = str(t).rsplit(".", 1)[-1].replace("float8_e4m3fn", "float8_e4m3")
        if text not in _NAMES:
            raise TypeError(f"{name}: unsupported type {t}")
        got = _TYPE_IDS[t] = _NAMES.index(text)
    return got


# Types of other libraries' arrays that know their device and whether they are contiguous.
_TORCH_LIKE: set = set()

# The checks of an array come in two forms.  A call on small inputs costs the host more time than
# the GPU, so each array first goes through one chain of comparisons that ends in its pointer;
# whatever fails there (an unusual layout, or a mistake) goes through `_look`, which decides and
# words the error.

def _activation(a, name: str) -> int:
    if not hasattr(a, "data_ptr"):
        raise TypeError(f"{name}: needs a device array, got {type(a).__name__}")
    t = _type_of(a, name)
    if t not in _ACTIVATIONS:
        raise TypeError(f"{name}: activations are float32, float16 or bfloat16")
    return t


def _look(here: int, a, name: str, shape: tuple, type_id: int, inner: int) -> None:
    """Raises unless `a` is an array of that shape and type on device `here` whose last `inner`
    axes are contiguous (an axis of length 1 has any stride)."""
    if not hasattr(a, "data_ptr"):
        raise TypeError(f"{name}: needs a device array, got {type(a).__name__}")
    if tuple(a.shape) != shape:
        raise ValueError(f"{name}: shape {tuple(a.shape)}, expected {shape}")
    got = _type_of(a, name)
    if got != type_id:
        raise TypeError(f"{name}: {_NAMES[got]}, expected {_NAMES[type_id]}")
    at = 1
    for n, s in list(zip(reversed(shape), reversed(a.stride())))[:inner]:
        if n != 1 and s != at and 0 not in shape:
            raise ValueError(f"{name}: must be contiguous" if inner == len(shape) else
                             f"{name}: its last {inner} axes must be contiguous")
        at *= n
    if isinstance(a, DeviceArray):
        where = here if a.device is None else a.device
    else:
        where = a.get_device() if hasattr(a, "get_device") else here
    if where != here:
        raise ValueError(f"{name}: not on the current device ({here})")


def _stream():
    """The current stream's handle: `device.stream_handle` without an object for the default one."""
    stack = getattr(_tls, "streams", None)
    return stack[-1].handle if stack else None


def _here() -> int:
    """The current device, -1 where there is none (the library then says so)."""
    d = ctypes.c_int32(-1)
    return d.value if _lib.lib().salt_get_device(ctypes.byref(d)) == _lib.SALT_OK else -1


@functools.lru_cache(maxsize=4096)
def _dense(shape: tuple) -> tuple:
    return DeviceArray(0, shape, np.uint8, None).stride()


def _whole(here: int, a, name: str, shape: tuple, type_id: int) -> int:
    """Pointer of a contiguous array on device `here`; 0 for None."""
    if a is None:
        return 0
    if type(a) is DeviceArray:
        if a.shape == shape and _TYPE_IDS.get(a.dtype) == type_id \
                and (a.device == here or a.device is None):
            return a.ptr
    elif type(a) in _TORCH_LIKE:
        if a.shape == shape and _TYPE_IDS.get(a.dtype) == type_id and a.is_contiguous() \
                and a.get_device() == here:
            return a.data_ptr()
    elif hasattr(a, "is_contiguous") and hasattr(a, "get_device"):
        _TORCH_LIKE.add(type(a))
    _look(here, a, name, shape, type_id, len(shape))
    return a.data_ptr()


def _rows(here: int, a, name: str, shape: tuple, type_id: int, inner: int = 1):
    """(pointer, strides of the leading axes) of an array whose last `inner` axes are contiguous;
    (0, zeros) for None."""
    if a is None:
        return 0, (0,) * (len(shape) - inner)
    if type(a) is DeviceArray:
        if a.shape == shape and _TYPE_IDS.get(a.dtype) == type_id \
                and (a.device == here or a.device is None):
            return a.ptr, _dense(shape)[:-inner]
    elif type(a) in _TORCH_LIKE and a.shape == shape and _TYPE_IDS.get(a.dtype) == type_id:
        s = a.stride()
        if s[-1] == 1 and (inner == 1 or s[-2] == shape[-1]) and a.get_device() == here:
            return a.data_ptr(), s[:-inner]
    _look(here, a, name, shape, type_id, inner)
    return a.data_ptr(), tuple(a.stride())[:-inner]


def _weight(here: int, a, name: str, shape: tuple, type_id: int):
    """(pointer, type) of a contiguous weight of type_id or float32."""
    if a is None:
        return 0, type_id
    got = _F32 if hasattr(a, "data_ptr") and _type_of(a, name) == _F32 else type_id
    return _whole(here, a, name, shape, got), got


def _flat(here: int, a, name: str, shape: tuple, type_id: int):
    """(pointer, row stride) of an array whose leading axes fold into one axis of rows."""
    if a is None:
        return 0, 0
    p, strides = _rows(here, a, name, shape, type_id)
    if len(shape) == 2:
        return p, strides[0]
    stride, span = shape[-1], None
    for n, s in zip(reversed(shape[:-1]), reversed(strides)):
        if n == 1:
            continue
        if span is None:
            stride = s
        elif s != span and 0 not in shape:
            raise ValueError(f"{name}: its leading axes do not fold into rows of one stride")
        span = s * n
    return p, stride


def _wanted(a, shape, type_id):
    """The array for an optional output: None, a new one for True, or what was given."""
    if a is None or a is False:
        return None
    return empty(shape, _NUMPY[type_id]) if a is True else a


def _made(a, shape, type_id):
    return empty(shape, _NUMPY[type_id]) if a is None else a


def _axes(a, name: str, n: int) -> tuple:
    shape = tuple(getattr(a, "shape", ()))
    if len(shape) != n:
        raise ValueError(f"{name}: needs {n} axes, got shape {shape}")
    return shape


def _row_count(shape: tuple, name: str) -> int:
    if not shape:
        raise ValueError(f"{name}: needs at least one axis")
    return math.prod(shape[:-1])


def _packer(struct_type) -> struct.Struct:
    """Packs the fields of an argument struct, in order, into its bytes (integers, floats and
    pointers as integers): a third of the time of filling the ctypes structure."""
    codes = {ctypes.c_int32: "i", ctypes.c_int64: "q", ctypes.c_float: "f", ctypes.c_void_p: "P"}
    pack = struct.Struct("@" + "".join(codes[t] for _, t in struct_type._fields_))
    assert pack.size == ctypes.sizeof(struct_type)
    return pack.pack


_pack_norm = _packer(_lib.RmsNormArgs)
_pack_norm_backward = _packer(_lib.RmsNormBackwardArgs)
_pack_conv = _packer(_lib.CausalConvArgs)
_pack_conv_step = _packer(_lib.CausalConvStepArgs)
_pack_conv_backward = _packer(_lib.CausalConvBackwardArgs)
_pack_scan = _packer(_lib.SelectiveScanArgs)
_pack_scan_step = _packer(_lib.SelectiveScanStepArgs)
_pack_scan_backward = _packer(_lib.SelectiveScanBackwardArgs)


def _with_workspace(query, call, args: bytes) -> None:
    """call(args, workspace, bytes, stream) with the workspace that query asks for: stream-ordered
    memory, given back behind the call's work."""
    lib, stream, n = _lib.lib(), _stream(), ctypes.c_size_t(0)
    _lib.check(query(args, ctypes.byref(n)))
    ws = ctypes.c_void_p()
    if n.value:
        _lib.check(lib.salt_malloc(n.value, stream, ctypes.byref(ws)))
    try:
        _lib.check(call(args, ws, n.value, stream))
    finally:
        if ws:
            lib.salt_free(ws, stream)


# ---------------------------------------------------------------- root-mean-square norm

def _norm(x, weight, residual, eps, out, residual_out, rstd, scale, group):
    here = _here()
    t = _activation(x, "x")
    shape = tuple(x.shape)
    rows, dim = _row_count(shape, "x"), shape[-1]
    wide = t if residual is None else _type_of(residual, "residual")
    if residual is None and residual_out is not None and residual_out is not True \
            and residual_out is not False:
        wide = _type_of(residual_out, "residual_out")
    if wide not in (t, _F32):
        raise TypeError("residual: must hold x's type or float32")
    out = _made(out, shape, _E4M3 if group is not None else t)
    residual_out = _wanted(residual_out, shape, wide)
    rstd = _wanted(rstd, shape[:-1], _F32)
    ps = 0
    if group is not None:
        parts = (-(-dim // group) if group else 1,)
        scale = _made(scale, shape[:-1] + parts, _F32)
        ps = _whole(here, scale, "scale", shape[:-1] + parts, _F32)
    pw, wt = _weight(here, weight, "weight", (dim,), t)
    px, sx = _flat(here, x, "x", shape, t)
    pr, sr = _flat(here, residual, "residual", shape, wide)
    po, so = _flat(here, out, "out", shape, t if group is None else _E4M3)
    pro, sro = _flat(here, residual_out, "residual_out", shape, wide)
    args = _pack_norm(
        rows, dim, t, wide, wt, group or 0, eps, sx, sr, so, sro, px, pr, pw, po, pro,
        _whole(here, rstd, "rstd", shape[:-1], _F32), ps)
    _lib.check(_lib.lib().salt_rms_norm(args, _stream()))
    return NormOutput(out, residual_out, rstd, scale)


def rms_norm(x, weight, *, residual=None, eps: float = 1e-5, out=None, residual_out=None,
             rstd=None) -> NormOutput:
    """``r = x + residual; out = r / sqrt(mean(r^2) + eps) * weight`` over the last axis (at most
    16384 wide).  `residual` holds x's type or float32; `residual_out` takes r in that type (it may
    be `residual`, and `out` may be `x`), `rstd` the factors that the gradient needs."""
    return _norm(x, weight, residual, eps, out, residual_out, rstd, None, None)


def rms_norm_q8(x, weight, *, residual=None, eps: float = 1e-5, group: int = 128, out=None,
                scale=None, residual_out=None, rstd=None) -> NormOutput:
    """`rms_norm` with an output in 8 bits (`device.float8_e4m3`): every `group` neighbouring
    elements (32, 64, 128, 256, or 0 for the whole row) share a float32 scale, the largest
    magnitude / 448 (1 for a group of zeros), and ``out * scale`` is the normed value."""
    if group not in GROUPS_8BIT:
        raise ValueError(f"group must be one of {GROUPS_8BIT}")
    return _norm(x, weight, residual, eps, out, residual_out, rstd, scale, int(group))


def rms_norm_backward(dy, x, weight, rstd, *, dresidual=None, dx=None, dweight=None
                      ) -> NormGradients:
    """Gradients of `rms_norm`: x is what was normed (`residual_out`, or the input where there was
    no residual), rstd its factors, dresidual the gradient that reaches `residual_out` from
    elsewhere.  dx, the gradient of the input and of the residual alike, holds x's type (it may be
    `dresidual`); dweight (float32) is made unless given, and left out for False."""
    here = _here()
    t, wide = _activation(dy, "dy"), _activation(x, "x")
    if wide not in (t, _F32):
        raise TypeError("x: must hold dy's type or float32")
    shape = tuple(dy.shape)
    rows, dim = _row_count(shape, "dy"), shape[-1]
    dx = _made(dx, shape, wide)
    dweight = _wanted(True if dweight is None else dweight, (dim,), _F32)
    pdy, sdy = _flat(here, dy, "dy", shape, t)
    px, sx = _flat(here, x, "x", shape, wide)
    pr, sr = _flat(here, dresidual, "dresidual", shape, wide)
    pdx, sdx = _flat(here, dx, "dx", shape, wide)
    pw, wt = _weight(here, weight, "weight", (dim,), t)
    args = _pack_norm_backward(
        rows, dim, t, wide, wt, 0, sdy, sx, sr, sdx, pdy, px, pw,
        _whole(here, rstd, "rstd", shape[:-1], _F32), pr, pdx,
        _whole(here, dweight, "dweight", (dim,), _F32))
    lib = _lib.lib()
    _with_workspace(lib.salt_rms_norm_backward_workspace_size, lib.salt_rms_norm_backward, args)
    return NormGradients(dx, dweight)


# ---------------------------------------------------------------- causal convolution

def causal_conv(x, weight, bias=None, *, n_real=None, initial_state=None, silu: bool = True,
                out=None, final_state=None) -> ConvOutput:
    """``p[t] = bias + sum_k weight[:, k] x[t - width + 1 + k]``, put through ``p * sigmoid(p)``
    with silu, over rows x (batch, len, dim) with weight (dim, width), width 1 to 8.  n_real
    (batch, int32) ends each row early: what lies past it is not read and comes back as zero.
    initial_state (batch, dim, width - 1) holds the inputs in front of the row, oldest first;
    final_state takes the last ones (and may be initial_state)."""
    here = _here()
    t = _activation(x, "x")
    batch, n, dim = shape = _axes(x, "x", 3)
    width = _axes(weight, "weight", 2)[1]
    edge = (batch, dim, width - 1)
    out, final_state = _made(out, shape, t), _wanted(final_state, edge, t)
    pw, wt = _weight(here, weight, "weight", (dim, width), t)
    px, sx = _rows(here, x, "x", shape, t)
    po, so = _rows(here, out, "out", shape, t)
    args = _pack_conv(
        batch, n, dim, width, t, wt, bool(silu), 0, *sx, *so, px, pw,
        _whole(here, bias, "bias", (dim,), wt), _whole(here, n_real, "n_real", (batch,), _I32),
        _whole(here, initial_state, "initial_state", edge, t), po,
        _whole(here, final_state, "final_state", edge, t))
    _lib.check(_lib.lib().salt_causal_conv(args, _stream()))
    return ConvOutput(out, final_state)


def causal_conv_step(x, state, weight, bias=None, *, slots=None, silu: bool = True, out=None
                     ) -> ConvOutput:
    """One token x (batch, dim) for each row: row b shifts it into state[slots[b]] of a pool
    (n_slots, dim, width - 1), in place.  Without slots row b is slot b.  A slot outside the pool
    marks an empty row (its out is zero); no slot may appear twice."""
    here = _here()
    t = _activation(x, "x")
    batch, dim = shape = _axes(x, "x", 2)
    width = _axes(weight, "weight", 2)[1]
    n_slots = _axes(state, "state", 3)[0]
    out = _made(out, shape, t)
    pw, wt = _weight(here, weight, "weight", (dim, width), t)
    px, sx = _rows(here, x, "x", shape, t)
    po, so = _rows(here, out, "out", shape, t)
    args = _pack_conv_step(
        batch, dim, width, n_slots, t, wt, bool(silu), 0, *sx, *so, px, pw,
        _whole(here, bias, "bias", (dim,), wt), _whole(here, slots, "slots", (batch,), _I32),
        _whole(here, state, "state", (n_slots, dim, width - 1), t), po)
    _lib.check(_lib.lib().salt_causal_conv_step(args, _stream()))
    return ConvOutput(out, state)


def causal_conv_backward(dy, x, weight, bias=None, *, n_real=None, initial_state=None,
                         silu: bool = True, dx=None, dweight=None, dbias=None, dinitial=None
                         ) -> ConvGradients:
    """Gradients of `causal_conv` for dy, the gradient of its out.  dweight and dbias are float32
    (dbias is made where there is a bias); dinitial (batch, dim, width - 1) holds x's type and is
    optional.  A gradient of final_state is not taken: that state holds inputs as they are, so it is
    the caller's to add to dx of the row's last width - 1 tokens (and to dinitial, in shorter
    rows)."""
    here = _here()
    t = _activation(x, "x")
    batch, n, dim = shape = _axes(x, "x", 3)
    width = _axes(weight, "weight", 2)[1]
    edge = (batch, dim, width - 1)
    dx, dweight = _made(dx, shape, t), _made(dweight, (dim, width), _F32)
    dbias = _wanted(bias is not None if dbias is None else dbias, (dim,), _F32)
    dinitial = _wanted(dinitial, edge, t)
    pw, wt = _weight(here, weight, "weight", (dim, width), t)
    pdy, sdy = _rows(here, dy, "dy", shape, t)
    px, sx = _rows(here, x, "x", shape, t)
    pdx, sdx = _rows(here, dx, "dx", shape, t)
    args = _pack_conv_backward(
        batch, n, dim, width, t, wt, bool(silu), 0, *sdy, *sx, *sdx, pdy, px, pw,
        _whole(here, bias, "bias", (dim,), wt), _whole(here, n_real, "n_real", (batch,), _I32),
        _whole(here, initial_state, "initial_state", edge, t), pdx,
        _whole(here, dinitial, "dinitial", edge, t),
        _whole(here, dweight, "dweight", (dim, width), _F32),
        _whole(here, dbias, "dbias", (dim,), _F32))
    lib = _lib.lib()
    _with_workspace(lib.salt_causal_conv_backward_workspace_size, lib.salt_causal_conv_backward,
                    args)
    return ConvGradients(dx, dweight, dbias, dinitial)


# ---------------------------------------------------------------- selective scan

def _checkpoint_shape(batch, n, dim, state):
    return batch, -(-n // CHECKPOINT), dim, state


def selective_scan(x, delta, A, B, C, *, D=None, z=None, delta_bias=None, softplus: bool = True,
                   n_real=None, initial_state=None, out=None, final_state=None, checkpoints=None
                   ) -> ScanOutput:
    """With ``s[t] = softplus(delta[t] + delta_bias)`` (or the sum itself without softplus):

        h[t] = exp(s[t] A) h[t-1] + s[t] x[t] B[t];   y[t] = sum_n C[t] h[t] + D x[t]

    and ``out = y``, or ``y * z * sigmoid(z)`` where z is given.  x, delta, z: (batch, len, dim); A:
    (dim, state) float32, finite, state 1 to 64; B, C: (batch, len, groups, state), channel d reading group
    ``d // (dim / groups)``; D, delta_bias: (dim,) float32.  n_real (batch, int32) ends each row
    early.  initial_state and final_state: (batch, dim, state) float32, may be one array.
    checkpoints takes the states that `selective_scan_backward` starts from."""
    here = _here()
    t = _activation(x, "x")
    batch, n, dim = shape = _axes(x, "x", 3)
    groups, state = _axes(B, "B", 4)[2:]
    both, ends = (batch, n, groups, state), (batch, dim, state)
    marks = _checkpoint_shape(batch, n, dim, state)
    out, final_state = _made(out, shape, t), _wanted(final_state, ends, _F32)
    checkpoints = _wanted(checkpoints, marks, _F32)
    px, sx = _rows(here, x, "x", shape, t)
    pd, sd = _rows(here, delta, "delta", shape, t)
    pz, sz = _rows(here, z, "z", shape, t)
    pb, sb = _rows(here, B, "B", both, t, 2)
    pc, sc = _rows(here, C, "C", both, t, 2)
    po, so = _rows(here, out, "out", shape, t)
    args = _pack_scan(
        batch, n, dim, state, groups, t, bool(softplus), 0, *sx, *sd, *sz, *sb, *sc, *so, px, pd,
        pz, pb, pc, _whole(here, A, "A", (dim, state), _F32), _whole(here, D, "D", (dim,), _F32),
        _whole(here, delta_bias, "delta_bias", (dim,), _F32),
        _whole(here, n_real, "n_real", (batch,), _I32),
        _whole(here, initial_state, "initial_state", ends, _F32), po,
        _whole(here, final_state, "final_state", ends, _F32),
        _whole(here, checkpoints, "checkpoints", marks, _F32))
    lib = _lib.lib()
    _with_workspace(lib.salt_selective_scan_workspace_size, lib.salt_selective_scan, args)
    return ScanOutput(out, final_state, checkpoints)


def selective_scan_step(pool, x, delta, A, B, C, *, D=None, z=None, delta_bias=None,
                        softplus: bool = True, slots=None, out=None) -> ScanOutput:
    """One token of `selective_scan` for each row, x, delta, z (batch, dim) and B, C (batch,
    groups, state), on pool[slots[b]] of float32 states (n_slots, dim, state), in place; slots as in
    `causal_conv_step`."""
    here = _here()
    t = _activation(x, "x")
    batch, dim = shape = _axes(x, "x", 2)
    groups, state = _axes(B, "B", 3)[1:]
    n_slots = _axes(pool, "pool", 3)[0]
    both = (batch, groups, state)
    out = _made(out, shape, t)
    px, (sx,) = _rows(here, x, "x", shape, t)
    pd, (sd,) = _rows(here, delta, "delta", shape, t)
    pz, (sz,) = _rows(here, z, "z", shape, t)
    pb, (sb,) = _rows(here, B, "B", both, t, 2)
    pc, (sc,) = _rows(here, C, "C", both, t, 2)
    po, (so,) = _rows(here, out, "out", shape, t)
    args = _pack_scan_step(
        batch, dim, state, groups, n_slots, t, bool(softplus), 0, sx, sd, sz, sb, sc, so, px, pd,
        pz, pb, pc, _whole(here, A, "A", (dim, state), _F32), _whole(here, D, "D", (dim,), _F32),
        _whole(here, delta_bias, "delta_bias", (dim,), _F32),
        _whole(here, slots, "slots", (batch,), _I32),
        _whole(here, pool, "pool", (n_slots, dim, state), _F32), po)
    _lib.check(_lib.lib().salt_selective_scan_step(args, _stream()))
    return ScanOutput(out, pool)


def selective_scan_backward(dy, x, delta, A, B, C, *, checkpoints, D=None, z=None,
                            delta_bias=None, softplus: bool = True, n_real=None, dfinal=None,
                            dx=None, ddelta=None, dA=None, dB=None, dC=None, dD=None, dz=None,
                            ddelta_bias=None, dinitial=None) -> ScanGradients:
    """Gradients of `selective_scan` for dy, the gradient of its out, and dfinal, that of its final
    state, from the forward's arguments and checkpoints.  dA, dD, ddelta_bias and dinitial are
    float32, the others hold x's type; dD, dz and ddelta_bias are made where their input is given,
    dinitial is optional."""
    here = _here()
    t = _activation(x, "x")
    batch, n, dim = shape = _axes(x, "x", 3)
    groups, state = _axes(B, "B", 4)[2:]
    both, ends = (batch, n, groups, state), (batch, dim, state)
    dx, ddelta = _made(dx, shape, t), _made(ddelta, shape, t)
    dA, dB, dC = _made(dA, (dim, state), _F32), _made(dB, both, t), _made(dC, both, t)
    dD = None if D is None else _made(dD, (dim,), _F32)
    dz = None if z is None else _made(dz, shape, t)
    ddelta_bias = None if delta_bias is None else _made(ddelta_bias, (dim,), _F32)
    dinitial = _wanted(dinitial, ends, _F32)
    px, sx = _rows(here, x, "x", shape, t)
    pd, sd = _rows(here, delta, "delta", shape, t)
    pz, sz = _rows(here, z, "z", shape, t)
    pb, sb = _rows(here, B, "B", both, t, 2)
    pc, sc = _rows(here, C, "C", both, t, 2)
    pdy, sdy = _rows(here, dy, "dy", shape, t)
    pdx, sdx = _rows(here, dx, "dx", shape, t)
    pdd, sdd = _rows(here, ddelta, "ddelta", shape, t)
    pdz, sdz = _rows(here, dz, "dz", shape, t)
    marks = _checkpoint_shape(batch, n, dim, state)
    args = _pack_scan_backward(
        batch, n, dim, state, groups, t, bool(softplus), 0, *sx, *sd, *sz, *sb, *sc, *sdy, *sdx,
        *sdd, *sdz, px, pd, pz, pb, pc, pdy, _whole(here, A, "A", (dim, state), _F32),
        _whole(here, D, "D", (dim,), _F32), _whole(here, delta_bias, "delta_bias", (dim,), _F32),
        _whole(here, n_real, "n_real", (batch,), _I32),
        _whole(here, checkpoints, "checkpoints", marks, _F32),
        _whole(here, dfinal, "dfinal", ends, _F32), pdx, pdd, pdz, _whole(here, dB, "dB", both, t),
        _whole(here, dC, "dC", both, t), _whole(here, dA, "dA", (dim, state), _F32),
        _whole(here, dD, "dD", (dim,), _F32),
        _whole(here, ddelta_bias, "ddelta_bias", (dim,), _F32),
        _whole(here, dinitial, "dinitial", ends, _F32))
    lib = _lib.lib()
    _with_workspace(lib.salt_selective_scan_backward_workspace_size,
                    lib.salt_selective_scan_backward, args)
    return ScanGradients(dx, ddelta, dA, dB, dC, dD, dz, ddelta_bias, dinitial)
