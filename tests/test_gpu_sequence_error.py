"""The scan and its gradient against a running bound of their rounding errors.

test_gpu_sequence counts every token's roundings into every output.  Here the bound runs along with
the recurrence and decays with the states, so that a mistake of a few hundred ulp in a state, a step
or a gradient shows.  e(v) is a bound of v's error in units of 2^-24, M(v) the magnitude (the same
formula over absolute values), both in 64 bits; each rounding adds a magnitude once, and the fast
exponential, reciprocal and constants (2 ulp each at most, 4 units) and their arguments' roundings
make up these:
  raw = delta + bias        1 |raw|
  s = softplus(raw)         S = 12 + 4 (|delta| + |bias|) of s: its exponential's argument is rounded
                            twice, and the sum itself once; two 4s and the polynomial's steps
  a = exp(s A)              K = 4 + (S + 4) |s A| of a
  z sigmoid(z)              G = 12 + 2 |z| of it
The rows are short enough to stay whole (a chunk's sum of steps has roundings of its own)."""
import numpy as np
import pytest

import _sequence_ref as R
import salt_b200 as S

pytestmark = pytest.mark.gpu


def bounds(v, f):
    """{name: (value, bound)} of the forward and of every gradient."""
    x, delta, B, C, z, dy = (v[k] for k in ("x", "delta", "B", "C", "z", "dy"))
    A, skip, bias = f["A"], f["Dskip"], f["bias"]
    batch, n, dim = x.shape
    groups, state = B.shape[2:]
    ins = dict(x=x, delta=delta, A=A, B=B, C=C, Dskip=skip, z=z, bias=bias, init=f["init"])
    ahead, kept, _ = R.scan(**ins)
    back, _ = R.scan_backward(dy, **ins, dfinal=f["dfinal"])
    ab = np.abs
    s = R.softplus(delta + bias)
    raw = ab(delta) + ab(bias)
    Sn, G, gate = 12 + 4 * raw, 12 + 2 * ab(z), ab(R.silu(z))
    K = 4 + (Sn + 4)[..., None] * ab(s[..., None] * A)
    sx = ab(s * x)
    o = {k: np.zeros(a.shape) for k, (a, _) in (ahead | back).items()}
    e, eh, ey = np.zeros(f["init"].shape), [], []
    for t in range(n):
        a, h, new, m, newm, b_t, c_t, y, ym = kept[t]
        eh.append(e)
        e = a * (e + K[:, t] * m) + (Sn[:, t] + 2)[..., None] * sx[:, t][..., None] * ab(b_t) + newm
        ey.append((e * ab(c_t)).sum(-1) + (state + 4) * ym)
        o["out"][:, t] = (ey[t] + G[:, t] * ym) * gate[:, t]
        eh[t] = (eh[t], e)
    o["final"] = e
    g = ab(dy) * gate
    cm, ec = ab(f["dfinal"]), np.zeros(f["dfinal"].shape)
    sums = 16 + n / 16 + 16 + batch       # within a tile, over the tiles, over threads and rows
    split = (batch, groups, dim // groups, state)
    for t in reversed(range(n)):
        a, h, new, m, newm, b_t, c_t, y, ym = kept[t]
        gC = g[:, t][..., None] * ab(c_t)
        dhm = cm + gC
        edh = ec + (G[:, t] + 1)[..., None] * gC + dhm
        cm, ec = a * dhm, a * (edh + (K[:, t] + 1) * dhm)
        tom = (dhm * ab(b_t)).sum(-1)
        eto = (edh * ab(b_t)).sum(-1) + (state + 4) * tom
        mm = cm * m
        em = ec * m + cm * eh[t][0] + mm
        Asm = (mm * ab(A)).sum(-1)
        eAs = (em * ab(A)).sum(-1) + (state + 6) * Asm
        dsm = ab(x[:, t]) * tom + Asm
        slope = R.sigmoid(delta[:, t] + bias)
        ed = slope * (ab(x[:, t]) * eto + eAs + 2 * dsm + (4 * raw[:, t] + 10) * dsm)
        o["ddelta"][:, t] = ed
        gD = g[:, t] * ab(skip)
        o["dx"][:, t] = s[:, t] * (eto + (Sn[:, t] + 2) * tom) + (G[:, t] + 3) * gD
        az = 1 + ab(z[:, t])
        o["dz"][:, t] = ab(dy[:, t]) * (ey[t] * az + ym * (16 + 2 * ab(z[:, t])) * az)
        st = s[:, t][..., None]
        o["dA"] += (em * st + (Sn[:, t] + 1 + sums)[..., None] * mm * st).sum(0)
        xs = sx[:, t][..., None]
        o["dB"][:, t] = (edh * xs + (Sn[:, t] + 42)[..., None] * dhm * xs).reshape(split).sum(2)
        gt = g[:, t][..., None]
        o["dC"][:, t] = (gt * eh[t][1] + (G[:, t] + 41)[..., None] * gt * newm).reshape(split).sum(2)
        o["dD"] += ((G[:, t] + 1 + sums) * g[:, t] * ab(x[:, t])).sum(0)
        o["ddelta_bias"] += (ed + sums * slope * dsm).sum(0)
    o["dinitial"] = ec
    return {k: (a, o[k]) for k, (a, _) in (ahead | back).items()}


@pytest.mark.parametrize("kind", ("float32", "float16", "bfloat16"))
@pytest.mark.parametrize("dim, state, groups", [(70, 4, 1), (48, 8, 2), (65, 16, 1), (64, 12, 4),
                                                (40, 32, 1), (34, 64, 2)])
def test_scan_within_its_running_bound(kind, dim, state, groups):
    rng = np.random.default_rng(dim + state)
    batch, n = 2, 250
    v = {k: rng.normal(size=(batch, n, dim)) for k in ("x", "delta", "z", "dy")}
    v |= {k: rng.normal(size=(batch, n, groups, state)) for k in ("B", "C")}
    v = {k: R.rounded(a, kind) for k, a in v.items()}
    f = {"A": -rng.uniform(0.1, 1.5, (dim, state)) * np.arange(1, state + 1) / 4,
         "Dskip": rng.normal(size=dim), "bias": rng.uniform(-4, 0, dim),
         "init": rng.normal(size=(batch, dim, state)), "dfinal": rng.normal(size=(batch, dim, state))}
    f = {k: R.rounded(a, "float32") for k, a in f.items()}
    a, w = {k: R.to_device(u, kind) for k, u in v.items()}, {k: R.to_device(u) for k, u in f.items()}
    args = (a["x"], a["delta"], w["A"], a["B"], a["C"])
    named = dict(D=w["Dskip"], z=a["z"], delta_bias=w["bias"])
    got = S.selective_scan(*args, **named, initial_state=w["init"], final_state=True,
                           checkpoints=True)
    grads = S.selective_scan_backward(a["dy"], *args, **named, checkpoints=got.checkpoints,
                                      dfinal=w["dfinal"], dinitial=True)._asdict()
    grads |= {"out": got.out, "final": got.final_state}
    for k, (value, bound) in bounds(v, f).items():
        own = "float32" if k in ("final", "dA", "dD", "ddelta_bias", "dinitial") else kind
        # 1 % for the products of errors and the bound's own roundings
        R.assert_close(R.values(grads[k]), value, bound, 1.01, own, k)


BANDS = [2.0 ** -k for k in (13, 11, 9, 8, 7, 6)]  # |s A| log2(e) from here to twice that


@pytest.mark.parametrize("form", ["rows", "steps", "gradient"])
def test_decays_have_no_common_error(form):
    """A state without inputs is the product of its decays.  Over many channels and 250 tokens of
    random steps their errors' mean shows: at most 0.16 units of 2^-24 for arguments under 2^-7 (by
    the exponential's measured error and the shift that takes it away), 0.35 over it."""
    rng = np.random.default_rng(0)
    n, dim, state = 250, 2048, len(BANDS)
    delta = (1 + rng.random((1, n, dim))).astype(np.float32) / 1.5
    A = (-np.array(BANDS) * rng.uniform(1, 1.5, (dim, state)) / np.log2(np.e)).astype(np.float32)
    one, none = R.to_device(np.ones((1, dim, state))), R.to_device(np.zeros((1, n, dim)))
    B = R.to_device(np.zeros((1, n, 1, state)))
    dd, dA = R.to_device(delta), R.to_device(A)
    if form == "steps":
        zero, B1 = R.to_device(np.zeros((1, dim))), R.to_device(np.zeros((1, 1, state)))
        for t in range(n):
            S.selective_scan_step(one, zero, R.to_device(delta[:, t]), dA, B1, B1, softplus=False)
        h = R.values(one)[0]
    else:
        got = S.selective_scan(none, dd, dA, B, B, softplus=False, initial_state=one,
                               final_state=True, checkpoints=True)
        h = R.values(got.final_state)[0]
    if form == "gradient":
        h = R.values(S.selective_scan_backward(none, none, dd, dA, B, B, softplus=False, dfinal=one,
                                               checkpoints=got.checkpoints, dinitial=True).dinitial)[0]
    want = np.exp(A.astype(np.float64) * delta[0].astype(np.float64).sum(0)[:, None])
    mean = ((h / want - 1) / n / R.U32).mean(0)
    # 2048 x 250 errors of under a unit each leave the mean 0.002 uncertain
    assert np.all(np.abs(mean) <= np.where(np.array(BANDS) < 2.0 ** -7, 0.16, 0.35) + 0.01), mean
