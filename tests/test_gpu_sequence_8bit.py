"""The 8-bit norm bit by bit.  The factor of each row comes back from the call, so that the values in
front of the rounding are known to the last bit: r * rstd * weight, two products in 32 bits.  What
follows is defined exactly: scale is the float32 quotient of the group's largest magnitude and 448,
and out the e4m3 value nearest to the float32 quotient value / scale, ties to even, so nothing here
has a tolerance."""
import numpy as np
import pytest

import _sequence_ref as R
import salt_b200 as S

pytestmark = pytest.mark.gpu

F = np.float32


def e4m3(q):
    """The nearest e4m3 values of float32 quotients: 3 bits of mantissa, steps of 2^-9 under 2^-6,
    448 at most."""
    q = q.astype(np.float64)
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -6))) - 3)
    return np.clip(np.rint(q / step) * step, -448, 448)


def check(x, w, group, eps=1e-5, kind="float32", residual=None):
    """x (rows, dim), w (dim,) hold values of `kind`."""
    rows, dim = x.shape
    got = S.rms_norm_q8(R.to_device(x, kind), R.to_device(w, kind), eps=eps, group=group, rstd=True,
                        residual=None if residual is None else R.to_device(residual, kind))
    r = x.astype(F) if residual is None else x.astype(F) + residual.astype(F)
    y = r * got.rstd.numpy()[:, None] * w.astype(F)
    g = group or dim
    wide = np.zeros((rows, -(-dim // g) * g), F)
    wide[:, :dim] = y
    wide = wide.reshape(rows, -1, g)
    most = np.abs(wide).max(-1)
    with np.errstate(under="ignore"):
        scale = np.where(most == 0, F(1), np.maximum(most / F(448), F(2.0 ** -149)))
        want = e4m3(wide / scale[..., None]).reshape(rows, -1)[:, :dim]
    np.testing.assert_array_equal(got.scale.numpy(), scale)
    np.testing.assert_array_equal(R.values(got.out), want)


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
@pytest.mark.parametrize("rows, dim, group", [(300, 4096, 128), (300, 1000, 32), (1200, 1031, 0),
                                              (900, 2504, 256), (40, 16384, 0)])
def test_8_bits_are_the_nearest_to_the_quotient(kind, rows, dim, group):
    rng = np.random.default_rng(dim)
    x = R.rounded(rng.normal(size=(rows, dim)), kind)
    w = R.rounded(1 + 0.3 * rng.normal(size=dim), kind)
    check(x, w, group, kind=kind, residual=R.rounded(2 * rng.normal(size=(rows, dim)), kind))


def test_8_bits_at_the_middle_of_two_values():
    """Rows of one magnitude have the factor 1 / (that magnitude) or close to it; weights that are
    448 times a middle of two e4m3 values, and float32's neighbours of it, then bring quotients to
    both sides of that middle and onto it."""
    rng = np.random.default_rng(0)
    dim, rows = 4096, 200
    middle = (rng.integers(8, 16, dim) + 0.5) / 8 * 2.0 ** rng.integers(-8, 8, dim)
    w = F(middle)
    w = (w.view(np.int32) + rng.integers(-2, 3, dim).astype(np.int32)).view(F)
    w[::32] = 448
    x = np.repeat(rng.uniform(0.5, 2, (rows, 1)), dim, 1).astype(F) * rng.choice([-1, 1], (rows, dim))
    check(x.astype(F), w, 32, eps=0.0)


@pytest.mark.parametrize("group", [0, 32])
def test_8_bits_of_large_values(group):
    """Groups whose largest value lies close to float32's largest."""
    rng = np.random.default_rng(1)
    x = rng.normal(size=(5, 512)).astype(F)
    w = (rng.uniform(0.5, 1, 512) * 2.0 ** 126).astype(F)
    x[np.abs(x) > 2] = 2  # below 2^128 with the factor, which is about 1
    check(x, w, group)


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
@pytest.mark.parametrize("group", [0, 32])
def test_8_bits_of_tiny_values(kind, group):
    """Groups of tiny values and zeros, down to float32's smallest: zeros stay zeros, and values keep
    their places between them."""
    rng = np.random.default_rng(2)
    sizes = np.array([1e-30, 1e-35, 1.2e-36, 1e-37, 1e-38, 1e-40, 1e-42, 1e-43, 3e-45, 0])
    w = np.repeat(sizes, 32) * rng.uniform(0.01, 1, 320) * rng.choice([0, 1, 1, -1], 320)
    w = R.rounded(w, kind)
    x = R.rounded(rng.normal(size=(4, 320)), kind)
    check(x, w, group, kind=kind)
    for k in range(0, 320, 32):  # one size a row
        check(x[:, k:k + 32], w[k:k + 32], group, kind=kind)
