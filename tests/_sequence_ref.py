"""The sequence operators from their definitions in 64 bits, one token after the other, each value
with a magnitude: the same formula over absolute values.  Every rounding of a 32-bit evaluation is
relative to such a magnitude, which is what the tests derive their tolerances from.  `Strided` lays
an array out with gaps on the device."""
import numpy as np

from salt_b200 import device as D

U32 = 2.0 ** -24
ROUNDING = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# below these an output is subnormal, and off by up to half their spacing
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -126}


def sigmoid(v):
    return 1.0 / (1.0 + np.exp(-v))


def silu(v):
    return v * sigmoid(v)


def silu_slope(v):
    p = sigmoid(v)
    return p * (1 + v * (1 - p))


def softplus(v):
    return np.logaddexp(v, 0.0)


def rounded(a, kind):
    """The values that `kind` holds, as float64."""
    a = np.asarray(a, dtype=np.float32)
    if kind == "float16":
        a = a.astype(np.float16)
    elif kind == "bfloat16":
        a = D.from_bfloat16(D.to_bfloat16(a))
    return a.astype(np.float64)


def host_of(a, kind):
    a = np.asarray(a, dtype=np.float32)
    if kind == "bfloat16":
        return D.to_bfloat16(a)
    return a.astype(np.float16) if kind == "float16" else a


def dtype_of(kind):
    return D.bfloat16 if kind == "bfloat16" else np.dtype(kind)


def to_device(a, kind="float32"):
    h = host_of(a, kind)
    return D.DeviceArray.from_host(h, h.dtype)


def values(d, kind=None):
    """A device array's values as float64."""
    h = d.numpy()
    if h.dtype == D.bfloat16:
        return D.from_bfloat16(h).astype(np.float64)
    if h.dtype == D.float8_e4m3:
        return D.from_float8_e4m3(h).astype(np.float64)
    return h.astype(np.float64)


class Strided:
    """`a` on the device with `gap` NaN elements behind each row of its last `inner` axes, and
    `offset` in front: a slice of a wider projection."""

    def __init__(self, a, kind="float32", gap=8, offset=0, inner=1):
        a = np.asarray(a)
        lead, tail = a.shape[:a.ndim - inner], a.shape[a.ndim - inner:]
        width = int(np.prod(tail, dtype=np.int64))
        wide = np.full(lead + (offset + width + gap,), np.nan, np.float32)
        wide[..., offset:offset + width] = a.reshape(lead + (width,))
        self.memory = to_device(wide, kind)
        self.shape, self.dtype = a.shape, self.memory.dtype
        self._at = self.memory.data_ptr() + offset * self.dtype.itemsize
        self._stride = self.memory.stride()[:-1] + D.DeviceArray(0, tail, self.dtype, None).stride()
        self._cut = (Ellipsis, slice(offset, offset + width))

    def data_ptr(self):
        return self._at

    def stride(self):
        return self._stride

    def values(self):
        return values(self.memory)[self._cut].reshape(self.shape)

    def untouched(self):
        """Whether the gaps still hold NaN."""
        m = values(self.memory).copy()
        m[self._cut] = np.nan
        return bool(np.all(np.isnan(m)))


def assert_close(got, ref, mag, steps, kind, what, more=0.0):
    """|got - ref| within the output's rounding and `steps` roundings of 2^-24 of the magnitude."""
    limit = (ROUNDING[kind] * np.abs(ref) * 1.01 + steps * U32 * mag + TINY[kind] + more)
    off = np.abs(got - ref)
    bad = ~(off <= limit)
    if np.any(bad):
        i = np.unravel_index(np.argmax(np.where(bad, off / limit, 0)), off.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off; at {i} got {got[i]}, "
                             f"expected {ref[i]} within {limit[i]}")


# ---------------------------------------------------------------- norm

def norm(x, w, res, eps):
    r = x + (0 if res is None else res)
    rstd = 1 / np.sqrt(np.mean(r * r, -1) + eps)
    return r, rstd, r * rstd[:, None] * w


def norm_backward(dy, x, w, rstd, dres):
    """(dx, its magnitude, dweight, its magnitude)."""
    h = x * rstd[:, None]
    g = dy * w
    dx = rstd[:, None] * (g - h * np.mean(g * h, -1, keepdims=True))
    mag = rstd[:, None] * (np.abs(g) + np.abs(h) * np.mean(np.abs(g * h), -1, keepdims=True))
    if dres is not None:
        dx, mag = dx + dres, mag + np.abs(dres)
    return dx, mag, np.sum(dy * h, 0), np.sum(np.abs(dy * h), 0)


# ---------------------------------------------------------------- convolution

def tokens(n_real, batch, n):
    if n_real is None:
        return [n] * batch
    return [int(min(max(v, 0), n)) for v in n_real]


def conv(x, w, bias, n_real=None, init=None, act=True):
    """(out, its magnitude, final state)."""
    batch, n, dim = x.shape
    width = w.shape[1]
    out, mag = np.zeros(x.shape), np.zeros(x.shape)
    final = np.zeros((batch, dim, width - 1))
    for b, real in enumerate(tokens(n_real, batch, n)):
        head = np.zeros((dim, width - 1)) if init is None else init[b]
        line = np.concatenate((head, x[b, :real].T), 1)
        final[b] = line[:, real:]
        for t in range(real):
            seen = line[:, t:t + width]
            p = (w * seen).sum(1) + (0 if bias is None else bias)
            out[b, t] = silu(p) if act else p
            mag[b, t] = np.abs(w * seen).sum(1) + (0 if bias is None else np.abs(bias))
    return out, mag, final


def conv_backward(dy, x, w, bias, n_real=None, init=None, act=True):
    """{name: (value, magnitude)}."""
    batch, n, dim = x.shape
    width = w.shape[1]
    zero = lambda *s: [np.zeros(s), np.zeros(s)]  # noqa: E731
    o = {"dx": zero(*x.shape), "dweight": zero(*w.shape), "dbias": zero(dim),
         "dinitial": zero(batch, dim, width - 1)}
    for b, real in enumerate(tokens(n_real, batch, n)):
        head = np.zeros((dim, width - 1)) if init is None else init[b]
        line = np.concatenate((head, x[b, :real].T), 1)
        dline, mline = np.zeros(line.shape), np.zeros(line.shape)
        for t in range(real):
            seen = line[:, t:t + width]
            p = (w * seen).sum(1) + (0 if bias is None else bias)
            size = 1 + np.abs(w * seen).sum(1) + (0 if bias is None else np.abs(bias))
            g = dy[b, t] * (silu_slope(p) if act else 1.0)
            m = np.abs(dy[b, t]) * (size if act else 1.0)  # |d slope / dp| <= 1/2
            dline[:, t:t + width] += g[:, None] * w
            mline[:, t:t + width] += m[:, None] * np.abs(w)
            for k, v, a in (("dweight", g[:, None] * seen, m[:, None] * np.abs(seen)),
                            ("dbias", g, m)):
                o[k][0] += v
                o[k][1] += a
        for at, part in ((0, dline), (1, mline)):
            o["dinitial"][at][b] = part[:, :width - 1]
            o["dx"][at][b, :real] = part[:, width - 1:].T
    return o


# ---------------------------------------------------------------- scan

def _spread(v, dim):
    """(batch, groups, state) to (batch, dim, state)."""
    return np.repeat(v, dim // v.shape[1], axis=1)


def scan(x, delta, A, B, C, Dskip=None, z=None, bias=None, plus=True, n_real=None, init=None):
    """{"out", "final": (value, magnitude)}, the kept tokens for the gradient, the largest |s A|."""
    batch, n, dim = x.shape
    state = A.shape[1]
    raw = delta + (0 if bias is None else bias)
    s = softplus(raw) if plus else raw
    h = np.zeros((batch, dim, state)) if init is None else init.copy()
    m = np.abs(h)
    out, mag = np.zeros(x.shape), np.zeros(x.shape)
    real = np.array(tokens(n_real, batch, n))
    kept, most = [], 1.0
    for t in range(n):
        live = (t < real)[:, None]
        b_t, c_t = _spread(B[:, t], dim), _spread(C[:, t], dim)
        with np.errstate(all="ignore"):
            a = np.exp(s[:, t, :, None] * A)
            new = a * h + (s[:, t] * x[:, t])[..., None] * b_t
            newm = a * m + np.abs(s[:, t] * x[:, t])[..., None] * np.abs(b_t)
            y = (new * c_t).sum(-1) + (0 if Dskip is None else Dskip * x[:, t])
            ym = (newm * np.abs(c_t)).sum(-1) + (0 if Dskip is None else np.abs(Dskip * x[:, t]))
            gate = 1.0 if z is None else silu(z[:, t])
            gm = 1.0 if z is None else np.abs(z[:, t])
            kept.append((a, h, new, m, newm, b_t, c_t, y, ym))
            h, m = np.where(live[..., None], new, h), np.where(live[..., None], newm, m)
            out[:, t], mag[:, t] = np.where(live, y * gate, 0), np.where(live, ym * gm, 0)
            if np.any(live):
                most = max(most, 1 + np.max(np.abs(np.where(live, s[:, t], 0)[..., None] * A)))
    return {"out": (out, mag), "final": (h, m)}, kept, most


def scan_backward(dy, x, delta, A, B, C, Dskip=None, z=None, bias=None, plus=True, n_real=None,
                  init=None, dfinal=None):
    """{name: (value, magnitude)} of every gradient, and the largest |s A|."""
    batch, n, dim = x.shape
    groups, state = B.shape[2:]
    _, kept, most = scan(x, delta, A, B, C, Dskip, z, bias, plus, n_real, init)
    raw = delta + (0 if bias is None else bias)
    s = softplus(raw) if plus else raw
    slope = sigmoid(raw) if plus else np.ones(raw.shape)
    real = np.array(tokens(n_real, batch, n))
    pair = lambda *shape: [np.zeros(shape), np.zeros(shape)]  # noqa: E731
    o = {"dx": pair(*x.shape), "ddelta": pair(*x.shape), "dz": pair(*x.shape),
         "dA": pair(*A.shape), "dB": pair(*B.shape), "dC": pair(*C.shape), "dD": pair(dim),
         "ddelta_bias": pair(dim)}
    carry = np.zeros((batch, dim, state)) if dfinal is None else dfinal.copy()
    carrym = np.abs(carry)
    ab = np.abs
    for t in reversed(range(n)):
        live = (t < real)[:, None]
        keep = lambda v, l=live: np.where(l.reshape(l.shape[:1] + (1,) * (v.ndim - 1)), v, 0)  # noqa
        a, hb, hn, hbm, hnm, b_t, c_t, y, ym = kept[t]
        xs, st, sl = keep(x[:, t]), keep(s[:, t]), keep(slope[:, t])
        d_y = keep(dy[:, t])
        gate = 1.0 if z is None else silu(keep(z[:, t]))
        g = d_y * gate
        gm = ab(d_y) * (1.0 if z is None else ab(keep(z[:, t])))
        b_t, c_t, a, hb, hbm, hn, hnm, y, ym = (keep(v) for v in (b_t, c_t, a, hb, hbm, hn, hnm, y,
                                                                 ym))
        dh = keep(carry) + g[..., None] * c_t
        dhm = keep(carrym) + gm[..., None] * ab(c_t)
        mv, mvm = dh * a * hb, dhm * a * hbm
        to, tom = (dh * b_t).sum(-1), (dhm * ab(b_t)).sum(-1)
        ds, dsm = (mv * A).sum(-1) + xs * to, (mvm * ab(A)).sum(-1) + ab(xs) * tom
        skip = 0 if Dskip is None else Dskip
        for k, v, w in (("dx", st * to + g * skip, st * tom + gm * ab(skip)),
                        ("ddelta", ds * sl, dsm * sl)):
            o[k][0][:, t], o[k][1][:, t] = v, w
        if z is not None:
            zt = keep(z[:, t])
            o["dz"][0][:, t] = d_y * y * silu_slope(zt)
            o["dz"][1][:, t] = ab(d_y) * ym * (1 + ab(zt))
        o["dA"][0] += (mv * st[..., None]).sum(0)
        o["dA"][1] += (mvm * ab(st[..., None])).sum(0)
        split = (batch, groups, dim // groups, state)
        for k, v, w in (("dB", dh * (st * xs)[..., None], dhm * ab(st * xs)[..., None]),
                        ("dC", hn * g[..., None], hnm * gm[..., None])):
            o[k][0][:, t], o[k][1][:, t] = v.reshape(split).sum(2), w.reshape(split).sum(2)
        o["dD"][0] += (g * xs).sum(0)
        o["dD"][1] += (gm * ab(xs)).sum(0)
        o["ddelta_bias"][0] += (ds * sl).sum(0)
        o["ddelta_bias"][1] += (dsm * sl).sum(0)
        alive = live[..., None]
        carry, carrym = np.where(alive, a * dh, carry), np.where(alive, a * dhm, carrym)
    o["dinitial"] = [carry, carrym]
    return o, most
