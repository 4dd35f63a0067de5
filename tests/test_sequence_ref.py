"""The 64-bit reference of the sequence operators: its gradients against central differences of
its forwards, and the host conversions of the types numpy lacks."""
import numpy as np
import pytest

import _sequence_ref as R
from salt_b200 import device as D

STEP = 1e-5
# central differences in 64 bits: a truncation of STEP^2 and a rounding of 2^-52 / STEP, each times
# the function's size (under 1e3 here): 1e-7 and 2e-8
CLOSE = 1e-6


def differences(f, arrays, grads, rng):
    """Each array's gradient along a random direction against the central difference of f."""
    for k, a in arrays.items():
        way = rng.normal(size=a.shape)
        ahead = f(**{**arrays, k: a + STEP * way})
        back = f(**{**arrays, k: a - STEP * way})
        slope = (ahead - back) / (2 * STEP)
        along = float(np.sum(grads[k] * way))
        scale = 1 + float(np.sqrt(np.sum(grads[k] ** 2)))
        assert abs(slope - along) <= CLOSE * scale, (k, slope, along)


def test_norm_gradient():
    rng = np.random.default_rng(0)
    x, w, dy = rng.normal(size=(5, 37)), rng.normal(size=37), rng.normal(size=(5, 37))
    _, rstd, _ = R.norm(x, w, None, 1e-5)
    dx, _, dw, _ = R.norm_backward(dy, x, w, rstd, None)
    differences(lambda x, w: float((R.norm(x, w, None, 1e-5)[2] * dy).sum()),
                {"x": x, "w": w}, {"x": dx, "w": dw}, rng)


@pytest.mark.parametrize("act", [True, False])
@pytest.mark.parametrize("n_real", [None, [0, 9, 4]])
def test_conv_gradient(act, n_real):
    rng = np.random.default_rng(1)
    a = {"x": rng.normal(size=(3, 9, 5)), "w": rng.normal(size=(5, 4)), "bias": rng.normal(size=5),
         "init": rng.normal(size=(3, 5, 3))}
    dy = rng.normal(size=a["x"].shape)
    o = R.conv_backward(dy, a["x"], a["w"], a["bias"], n_real, a["init"], act)
    differences(lambda x, w, bias, init: float((R.conv(x, w, bias, n_real, init, act)[0]
                                                * dy).sum()), a,
                {"x": o["dx"][0], "w": o["dweight"][0], "bias": o["dbias"][0],
                 "init": o["dinitial"][0]}, rng)


@pytest.mark.parametrize("gated, plus, n_real", [(True, True, None), (True, True, [3, 11, 0]),
                                                 (False, False, [11, 1, 7])])
def test_scan_gradient(gated, plus, n_real):
    rng = np.random.default_rng(2)
    batch, n, dim, state, groups = 3, 11, 6, 5, 2
    a = {"x": rng.normal(size=(batch, n, dim)), "delta": rng.normal(size=(batch, n, dim)),
         "A": -rng.uniform(0.2, 2, (dim, state)), "B": rng.normal(size=(batch, n, groups, state)),
         "C": rng.normal(size=(batch, n, groups, state)), "Dskip": rng.normal(size=dim),
         "bias": rng.normal(size=dim), "init": rng.normal(size=(batch, dim, state))}
    if not plus:
        a["delta"] = np.abs(a["delta"]) + 0.1
        a["bias"] = np.abs(a["bias"])
    if gated:
        a["z"] = rng.normal(size=(batch, n, dim))
    dy, df = rng.normal(size=(batch, n, dim)), rng.normal(size=(batch, dim, state))

    def f(**k):
        o = R.scan(**k, plus=plus, n_real=n_real)[0]
        return float((o["out"][0] * dy).sum() + (o["final"][0] * df).sum())

    o, _ = R.scan_backward(dy, **a, plus=plus, n_real=n_real, dfinal=df)
    names = {"x": "dx", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "Dskip": "dD",
             "bias": "ddelta_bias", "init": "dinitial", "z": "dz"}
    differences(f, a, {k: o[names[k]][0] for k in a}, rng)


def test_bfloat16_on_the_host():
    exact = np.array([0.0, -1.5, 3.140625, 2.0 ** -133, np.inf, -np.inf], np.float32)
    np.testing.assert_array_equal(D.from_bfloat16(D.to_bfloat16(exact)), exact)
    ties = np.array([1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1 + 2.0 ** -8 + 2.0 ** -20], np.float32)
    np.testing.assert_array_equal(D.from_bfloat16(D.to_bfloat16(ties)),
                                  np.array([1, 1 + 2.0 ** -6, 1 + 2.0 ** -7], np.float32))
    assert np.isnan(D.from_bfloat16(D.to_bfloat16(np.float32(np.nan))))


def test_float8_on_the_host():
    bits = np.array([0x00, 0x01, 0x08, 0x38, 0x7E, 0xFE, 0x7F], np.uint8).view(D.float8_e4m3)
    np.testing.assert_array_equal(
        D.from_float8_e4m3(bits),
        np.array([0, 2.0 ** -9, 2.0 ** -6, 1, 448, -448, np.nan], np.float32))
