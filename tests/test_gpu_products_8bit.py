"""Quantisation to 8 bits against its definition, bit by bit, and products of 8-bit matrices against
64 bits.

Tolerance of a product: its output's rounding, and units of 2^-24 of its magnitude (the sum over
absolute values): the sum of a group is 4 instructions of 32 terms, taken as 4 units each, its
scale's product and the addition to the other groups 3, the bias 1: 24 and one a group."""
import numpy as np
import pytest

import _attention_ref as A
import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu

KINDS = ("float32", "float16", "bfloat16")


def values8(a):
    return R.values(a)


class Strided8(R.Strided):
    """An 8-bit array's bytes with `gap` bytes of NaN behind each row and `offset` in front."""

    def __init__(self, codes, gap, offset):
        rows, width = codes.shape
        wide = np.full((rows, offset + width + gap), 0x7F, np.uint8)
        wide[:, offset:offset + width] = codes.view(np.uint8)
        self.memory = D.DeviceArray.from_host(wide.view(D.float8_e4m3), D.float8_e4m3)
        self.shape, self.dtype = (rows, width), D.float8_e4m3
        self._at = self.memory.data_ptr() + offset
        self._stride = (offset + width + gap, 1)
        self._cut = (Ellipsis, slice(offset, offset + width))


# ---------------------------------------------------------------- quantisation

SHAPES = ((1, 1), (1, 128), (3, 129), (128, 128), (127, 8), (129, 1), (130, 257), (300, 72),
          (5, 1000), (256, 384))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, dim", SHAPES)
def test_quantize(kind, rows, dim):
    rng = np.random.default_rng(rows + dim)
    x = rng.normal(size=(rows, dim)) * np.exp(rng.uniform(-9, 9, (rows, 1)))
    x[:, :min(dim, 128)] *= rng.integers(0, 2)  # groups of zeros
    x = R.rounded(x, kind)
    for gap, offset in ((0, 0), (8, 16), (3, 1)):
        dx = R.Strided(x, kind, gap=gap, offset=offset)
        for blocks in (False, True):
            for transposed in (False, True):
                want, scale = A.quantized(x.T if transposed else x, blocks)
                out = Strided8(np.zeros(want.shape, np.uint8), gap, offset)
                got = S.quantize_q8(dx, blocks=blocks, transposed=transposed, out=out)
                np.testing.assert_array_equal(got.scale.numpy(), scale)
                np.testing.assert_array_equal(out.values(), want)
                assert out.untouched()


def test_quantize_takes_leading_axes():
    x = np.random.default_rng(0).normal(size=(2, 3, 200)).astype(np.float32)
    got = S.quantize_q8(R.to_device(x))
    want, scale = A.quantized(x.reshape(6, 200))
    assert got.out.shape == (2, 3, 200) and got.scale.shape == (2, 3, 2)
    np.testing.assert_array_equal(values8(got.out).reshape(6, 200), want)
    np.testing.assert_array_equal(got.scale.numpy().reshape(6, 2), scale)
    assert S.quantize_q8(D.zeros((0, 200), np.float32)).out.shape == (0, 200)


@pytest.mark.parametrize("blocks", (False, True))
@pytest.mark.parametrize("transposed", (False, True))
def test_quantize_extremes(blocks, transposed):
    """Subnormal groups, the largest values, infinities and NaN beside finite ones."""
    x = np.ones((260, 260), np.float32)
    x[:128, :128] = 1e-44
    x[:128, 128:] = 3e38
    x[130, 5] = np.inf
    x[131, 200] = np.nan
    x[259, 259] = -np.nan
    want, scale = A.quantized(x.T if transposed else x, blocks)
    got = S.quantize_q8(R.to_device(x), blocks=blocks, transposed=transposed)
    np.testing.assert_array_equal(got.scale.numpy(), scale)
    q = values8(got.out)
    bad = np.isnan(want)  # a NaN, and an infinity over an infinite scale
    assert np.array_equal(np.isnan(q), bad)
    np.testing.assert_array_equal(q[~bad], want[~bad])


def test_quantize_agrees_with_the_norms_8_bits():
    """A norm, then quantised, is the norm's 8-bit form where nothing is rounded in between: in 32
    bits, of whole numbers, whose squares add up to the same sum in either call's order."""
    x = np.random.default_rng(1).integers(-50, 51, size=(7, 500)).astype(np.float32)
    w = R.to_device(np.ones(500))
    n = S.rms_norm(R.to_device(x), w)
    a, b = S.quantize_q8(n.out), S.rms_norm_q8(R.to_device(x), w, group=128)
    np.testing.assert_array_equal(a.scale.numpy(), b.scale.numpy())
    np.testing.assert_array_equal(values8(a.out), values8(b.out))


# ---------------------------------------------------------------- products

def check_product(rows, n, k, kind="bfloat16", by_rows=False, bias=None, seed=0, gaps=(0, 0, 0),
                  offsets=(0, 0, 0)):
    rng = np.random.default_rng(seed)
    (dx, x), (dw, w) = A.random_e4m3(rng, rows, k), A.random_e4m3(rng, n, k)
    groups = -(-k // 128)
    sx = np.exp(rng.uniform(-4, 1, (rows, groups))).astype(np.float32)
    sw = np.exp(rng.uniform(-4, 1, (n if by_rows else -(-n // 128), groups))).astype(np.float32)
    hb = None if bias is None else R.rounded(rng.normal(size=n), bias)
    if any(gaps) or any(offsets):
        dx = Strided8(dx.numpy(), gaps[0], offsets[0])
        dw = Strided8(dw.numpy(), gaps[1], offsets[1])
    out = R.Strided(np.zeros((rows, n)), kind, gap=gaps[2], offset=offsets[2])
    S.matmul_q8(dx, R.to_device(sx), dw, R.to_device(sw),
                bias=None if hb is None else R.to_device(hb, bias), out=out)
    want, mag = A.product(x, sx, w, sw, hb)
    got = out.values()
    if kind == "float16":  # from halfway behind its largest value, 65504, on, the nearest is infinity
        far = np.abs(want) > 65520 + (24 + groups) * R.U32 * mag
        assert np.all(got[far] == np.sign(want[far]) * np.inf)
        got[far] = want[far]
    R.assert_close(got, want, mag, 24 + groups, kind, f"{rows} x {n} x {k}")
    assert out.untouched()


ROWS = (1, 2, 8, 9, 16, 17, 33, 64, 65, 100, 128, 129, 260, 500)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("by_rows", (False, True))
def test_product_rows(rows, by_rows):
    check_product(rows, 256, 384, by_rows=by_rows, seed=rows)
    check_product(rows, 200, 272, "float32", by_rows=by_rows, bias="float32", seed=rows)


@pytest.mark.parametrize("n", (1, 2, 7, 8, 64, 100, 127, 128, 129, 255, 256, 257, 520))
@pytest.mark.parametrize("by_rows", (False, True))
def test_product_widths(n, by_rows):
    for rows in (3, 40, 140):
        check_product(rows, n, 256, by_rows=by_rows, seed=n)
        check_product(rows, n, 160, "float16", by_rows=by_rows, bias="float16", seed=n)


@pytest.mark.parametrize("k", (1, 5, 16, 31, 32, 33, 100, 127, 128, 129, 144, 255, 256, 640, 1001,
                               2048, 5000))
def test_product_depths(k):
    for rows, by_rows in ((4, False), (130, False), (130, True)):
        check_product(rows, 136, k, "float32", by_rows=by_rows, seed=k)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bias", (None, "float32", "same"))
def test_product_types(kind, bias):
    for rows in (5, 150):
        check_product(rows, 300, 300, kind, bias=kind if bias == "same" else bias, seed=1)


@pytest.mark.parametrize("gaps, offsets", (((16, 16, 8), (0, 0, 0)), ((16, 0, 8), (16, 0, 8)),
                                           ((1, 0, 1), (0, 0, 0)), ((0, 3, 0), (5, 0, 1)),
                                           ((7, 7, 7), (1, 2, 3)), ((0, 0, 5), (0, 8, 0))))
def test_product_strides(gaps, offsets):
    for rows in (3, 40, 150):
        for k in (256, 144, 131):
            check_product(rows, 140, k, seed=rows, gaps=gaps, offsets=offsets)


def test_product_of_many_tiles():
    """More tiles than blocks that fit at once, in both directions."""
    check_product(1300, 2700, 256, seed=3)
    check_product(16, 20000, 300, seed=4)
    check_product(1300, 2700, 128, "float32", by_rows=True, seed=5)


def test_product_takes_leading_axes_and_makes_its_output():
    rng = np.random.default_rng(0)
    (dx, x), (dw, w) = A.random_e4m3(rng, 2, 3, 200), A.random_e4m3(rng, 30, 200)
    sx, sw = np.ones((2, 3, 2), np.float32), np.ones((1, 2), np.float32)
    out = S.matmul_q8(dx, R.to_device(sx), dw, R.to_device(sw))
    assert out.shape == (2, 3, 30) and out.dtype == D.bfloat16
    assert S.matmul_q8(dx, R.to_device(sx), dw, R.to_device(sw), dtype=np.float32).dtype == \
        np.float32
    want, mag = A.product(x.reshape(6, 200), sx.reshape(6, 2), w, sw)
    R.assert_close(R.values(out).reshape(6, 30), want, mag, 26, "bfloat16", "out")
    none = S.matmul_q8(D.zeros((0, 200), D.float8_e4m3), D.zeros((0, 2), np.float32), dw,
                       R.to_device(sw))
    assert none.shape == (0, 30)


@pytest.mark.parametrize("rows", (5, 150))
def test_nan_and_infinity_stay_in_their_row(rows):
    rng = np.random.default_rng(2)
    (dx, x), (dw, w) = A.random_e4m3(rng, rows, 300), A.random_e4m3(rng, 200, 300)
    sx, sw = np.ones((rows, 3), np.float32), np.ones((200, 3), np.float32)
    codes = dx.numpy().view(np.uint8).copy()
    codes[1, 299] = 0x7F
    dx = D.DeviceArray.from_host(codes.view(D.float8_e4m3), D.float8_e4m3)
    sx[3, 1], sw[7, 0] = np.inf, np.nan
    got = R.values(S.matmul_q8(dx, R.to_device(sx), dw, R.to_device(sw), dtype=np.float32))
    bad = np.zeros(got.shape, bool)
    bad[1], bad[3], bad[:, 7] = True, True, True
    assert not np.isfinite(got[bad]).any() and np.isfinite(got[~bad]).all()


def test_a_training_steps_products():
    """Forward, dx and dweight of a projection against the products of the quantised values."""
    rng = np.random.default_rng(4)
    rows, k, n = 300, 272, 200
    x, w = R.rounded(rng.normal(size=(rows, k)), "bfloat16"), R.rounded(
        rng.normal(size=(n, k)), "bfloat16")
    dy = R.rounded(rng.normal(size=(rows, n)), "bfloat16")
    dx_, dw_, ddy = (R.to_device(a, "bfloat16") for a in (x, w, dy))
    wq, wt = S.quantize_q8(dw_, blocks=True), S.quantize_q8(dw_, blocks=True, transposed=True)
    xq, xt = S.quantize_q8(dx_), S.quantize_q8(dx_, transposed=True)
    gq, gt = S.quantize_q8(ddy), S.quantize_q8(ddy, transposed=True)
    y = S.matmul_q8(xq.out, xq.scale, wq.out, wq.scale, dtype=np.float32)
    dx = S.matmul_q8(gq.out, gq.scale, wt.out, wt.scale, dtype=np.float32)
    dw = S.matmul_q8(gt.out, gt.scale, xt.out, xt.scale, dtype=np.float32)
    X, W, GY = A.quantized(x), A.quantized(w, True), A.quantized(dy)
    WT, XT, GT = A.quantized(w.T, True), A.quantized(x.T), A.quantized(dy.T)
    for got, want in ((y, A.product(*X, *W)), (dx, A.product(*GY, *WT)), (dw, A.product(*GT, *XT))):
        R.assert_close(R.values(got), *want, 24 + 3, "float32", "product")
    # the same weight's values either way around
    np.testing.assert_array_equal(values8(wq.out), values8(wt.out).T)
    # and all three are near those of the values before the quantisation: each operand is off by
    # at most 2^-4 of the largest value that shares its scale's rounding, so by 2^-4 of itself or
    # of the smallest normal value, 2^-6 of the scale
    for got, a, b in ((y, x, w), (dx, dy, w.T), (dw, dy.T, x.T)):
        off = np.abs(R.values(got) - a @ b.T)
        bound = (2 * 2.0 ** -4 + 2.0 ** -8) * (np.abs(a) @ np.abs(b).T)
        small = 2.0 ** -10 * 6 / 448 * (np.abs(a).sum(1)[:, None] + np.abs(b).sum(1))
        assert np.all(off <= bound + small)
