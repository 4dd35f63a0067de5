"""Products of 8-bit matrices whose two scales multiply to what float32 does not hold, or not whole: the
definition's (x scale) (weight scale) does not meet that product.

Tolerance: the output's rounding, units of 2^-24 of the magnitude as in test_gpu_products_8bit.py (24 and
one a group), and half of float32's smallest step for each rounding of a subnormal value, two a group and
two more."""
import numpy as np
import pytest

import _attention_ref as A
import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu

G = 128
# (rows, n, scales by rows): every form of the product, and every number of rows a tile has
FORMS = ((300, 520, False), (1100, 4100, False), (5, 200, False), (30, 260, False), (64, 129, False),
         (100, 130, False), (300, 400, True), (3, 520, True), (300, 9000, True))


def codes(rng, rows, k):
    """All finite codes, as integers."""
    c = np.minimum(np.abs(rng.normal(0, 40, (rows, k))).astype(np.int64), 126)
    return (c + 128 * rng.integers(0, 2, (rows, k))).astype(np.uint8)


def check(x, sx, w, sw):
    dx, dw = (D.DeviceArray.from_host(c.view(D.float8_e4m3), D.float8_e4m3) for c in (x, w))
    x, w = (D.from_float8_e4m3(c.view(D.float8_e4m3)).astype(np.float64) for c in (x, w))
    got = R.values(S.matmul_q8(dx, R.to_device(sx), dw, R.to_device(sw), dtype=np.float32))
    want, mag = A.product(x, sx, w, sw)
    groups = sx.shape[1]
    limit = (1.01 * R.U32 * np.abs(want) + (24 + groups) * R.U32 * mag
             + (2 * groups + 2) * 2.0 ** -150)
    assert np.all(np.abs(want) < 2.0 ** 127)
    off = np.abs(got - want)
    bad = ~(off <= limit)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{bad.sum()} of {bad.size}: at {i} {got[i]}, {want[i]} within "
                             f"{limit[i]}")


def scales(rng, rows, n, groups, by_rows):
    one = lambda m: rng.uniform(1, 2, (m, groups))  # noqa: E731
    return one(rows), one(n if by_rows else -(-n // G))


@pytest.mark.parametrize("rows, n, by_rows", FORMS)
@pytest.mark.parametrize("k", (128, 1100))
def test_subnormal_products_of_scales(rows, n, by_rows, k):
    """Rows that lose all but seven bits or none at all, beside ordinary ones."""
    rng = np.random.default_rng(rows + k)
    sx, sw = scales(rng, rows, n, -(-k // G), by_rows)
    sx *= 2.0 ** np.array([-70, -30, 40])[np.arange(rows) % 3][:, None]
    sw *= 2.0 ** -72
    check(codes(rng, rows, k), sx.astype(np.float32), codes(rng, n, k), sw.astype(np.float32))


@pytest.mark.parametrize("rows, n, by_rows", FORMS)
@pytest.mark.parametrize("k", (128, 1100))
def test_infinite_products_of_scales(rows, n, by_rows, k):
    """Groups of zeros, and of a product that is small enough, under scales whose product is infinite."""
    rng = np.random.default_rng(rows + k)
    sx, sw = scales(rng, rows, n, -(-k // G), by_rows)
    x, w = codes(rng, rows, k), codes(rng, n, k)
    kind = np.arange(rows) % 3  # zeros, one value of 2^-9, anything
    x[kind < 2, :G] = 0
    x[kind == 1, 7], w[:, 7] = 1, 1
    sx[:, 0] *= 2.0 ** np.array([90, 78, -60])[kind]
    sw[:, 0] *= 2.0 ** 60
    check(x, sx.astype(np.float32), w, sw.astype(np.float32))


@pytest.mark.parametrize("rows, n, by_rows", FORMS)
def test_scales_of_zero(rows, n, by_rows):
    """A scale of zero takes its group out, whatever the other one is."""
    rng = np.random.default_rng(rows)
    sx, sw = scales(rng, rows, n, 4, by_rows)
    sx[::2, 1] = 0
    sw[:, 2] = 0
    sw[:, 1] *= 2.0 ** 100
    sx[1::2, 1] *= 2.0 ** -100
    check(codes(rng, rows, 512), sx.astype(np.float32), codes(rng, n, 512), sw.astype(np.float32))
