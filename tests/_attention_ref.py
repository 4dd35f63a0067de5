"""Linear attention and products in 8 bits from their definitions in 64 bits, each value with a
magnitude: the same formula over absolute values."""
import numpy as np

from _sequence_ref import tokens
from salt_b200 import device as D

G = 128


def decays(log_decay):
    """The decays that the operators use: log_decay within [-200, 0]."""
    return np.exp(np.clip(np.asarray(log_decay, np.float64), -200.0, 0.0))


def attention(q, k, v, log_decay, scale, n_real=None, init=None):
    """(out, its magnitude, final state, its magnitude), token after token."""
    batch, n, heads, dk = q.shape
    share, dv = heads // k.shape[2], v.shape[3]
    k, v = np.repeat(k, share, 2), np.repeat(v, share, 2)
    out, mag = np.zeros((2, batch, n, heads, dv))
    final, fmag = np.zeros((2, batch, heads, dk, dv))
    lam = decays(log_decay)[:, None, None]
    for b, real in enumerate(tokens(n_real, batch, n)):
        s = np.zeros((heads, dk, dv)) if init is None else init[b].astype(np.float64)
        m = np.abs(s)
        for t in range(real):
            kv = k[b, t][:, :, None] * v[b, t][:, None, :]
            s, m = lam * s + kv, lam * m + np.abs(kv)
            out[b, t] = scale * np.einsum("hk,hkv->hv", q[b, t], s)
            mag[b, t] = abs(scale) * np.einsum("hk,hkv->hv", np.abs(q[b, t]), m)
        final[b], fmag[b] = s, m
    return out, mag, final, fmag


def attention_backward(dout, q, k, v, log_decay, scale, n_real=None, init=None, dfinal=None):
    """{dq, dk, dv, dinitial}, each with its magnitude: the recurrence's own derivative."""
    batch, n, heads, dk = q.shape
    kv, dv = k.shape[2], v.shape[3]
    share = heads // kv
    K, V = np.repeat(k, share, 2), np.repeat(v, share, 2)
    lam = decays(log_decay)[:, None, None]
    o = {"dq": np.zeros((2,) + q.shape), "dk": np.zeros((2,) + K.shape),
         "dv": np.zeros((2,) + V.shape), "dinitial": np.zeros((2, batch, heads, dk, dv))}
    for b, real in enumerate(tokens(n_real, batch, n)):
        s = np.zeros((heads, dk, dv)) if init is None else init[b].astype(np.float64)
        m = np.abs(s)
        for t in range(real):
            now = K[b, t][:, :, None] * V[b, t][:, None, :]
            s, m = lam * s + now, lam * m + np.abs(now)
            o["dq"][0, b, t] = scale * np.einsum("hkv,hv->hk", s, dout[b, t])
            o["dq"][1, b, t] = abs(scale) * np.einsum("hkv,hv->hk", m, np.abs(dout[b, t]))
        d = np.zeros((heads, dk, dv)) if dfinal is None else dfinal[b].astype(np.float64)
        m = np.abs(d)
        for t in reversed(range(real)):
            now = scale * q[b, t][:, :, None] * dout[b, t][:, None, :]
            d, m = d + now, m + np.abs(now)
            for i, (w, x, y) in enumerate(((d, V[b, t], K[b, t]),
                                           (m, np.abs(V[b, t]), np.abs(K[b, t])))):
                o["dk"][i, b, t] = np.einsum("hkv,hv->hk", w, x)
                o["dv"][i, b, t] = np.einsum("hkv,hk->hv", w, y)
            d, m = lam * d, lam * m
        o["dinitial"][:, b] = d, m
    for name, dim in (("dk", dk), ("dv", dv)):
        o[name] = o[name].reshape(2, batch, n, kv, share, dim).sum(4)
    return o


# ---------------------------------------------------------------- 8 bits

E4M3 = D.from_float8_e4m3(np.arange(127, dtype=np.uint8).view(D.float8_e4m3)).astype(np.float64)
HALFWAY = (E4M3[1:] + E4M3[:-1]) / 2


def to_e4m3(v):
    """The nearest e4m3 values of float32 ones, ties to the even code; NaN stays one."""
    a = np.abs(np.asarray(v, np.float64))
    at = np.searchsorted(HALFWAY, a, side="left")  # a tie goes to the lower code
    at = np.where((at < 126) & (a == HALFWAY[np.minimum(at, 125)]) & (at % 2 == 1), at + 1, at)
    return np.where(np.isnan(v), np.nan, np.copysign(E4M3[at], v))


def quantized(x, blocks=False):
    """(8-bit values, scales) of a float32 matrix by groups of its rows, or by blocks."""
    x = np.asarray(x, np.float32)
    rows, dim = x.shape
    up, over = -(-rows // G), -(-dim // G)
    pad = np.zeros((up * G, over * G), np.float32)
    pad[:rows, :dim] = np.abs(x)
    most = np.fmax.reduce(pad.reshape(up * G, over, G), axis=2)
    if blocks:
        most = np.fmax.reduce(most.reshape(up, G, over), axis=1)
    else:
        most = most[:rows]
    scale = np.where(most == 0, np.float32(1), np.fmax(most / np.float32(448), 2.0 ** -149))
    scale = scale.astype(np.float32)
    by = np.repeat(scale, G, 1)[:, :dim]
    if blocks:
        by = np.repeat(by, G, 0)[:rows]
    with np.errstate(invalid="ignore"):
        return to_e4m3(x / by), scale


def random_e4m3(rng, *shape):
    """(device array, its values): all finite codes, the middle ones more often."""
    codes = np.minimum(np.abs(rng.normal(0, 40, shape)).astype(np.int64), 126)
    codes = (codes + 128 * rng.integers(0, 2, shape)).astype(np.uint8).view(D.float8_e4m3)
    return D.DeviceArray.from_host(codes, D.float8_e4m3), D.from_float8_e4m3(codes).astype(
        np.float64)


def spread(scale, rows, dim):
    """A scale's (rows or blocks, groups) for each value of a matrix."""
    if scale.shape[0] != rows:
        scale = np.repeat(scale, G, 0)[:rows]
    return np.repeat(scale.astype(np.float64), G, 1)[:, :dim]


def product(x, x_scale, w, w_scale, bias=None):
    """(out, its magnitude)."""
    a, b = x * spread(x_scale, *x.shape), w * spread(w_scale, *w.shape)
    out, mag = a @ b.T, np.abs(a) @ np.abs(b).T
    return (out, mag) if bias is None else (out + bias, mag + np.abs(bias))
