"""The 64-bit definitions that the GPU tests of linear attention and of the 8-bit values compare with:
against the closed form, against differences, and against the type's own spacing."""
import numpy as np

import _attention_ref as A


def inputs(n=9, heads=4, kv=2, dk=3, dv=5, batch=2):
    rng = np.random.default_rng(0)
    f = lambda *s: rng.normal(size=s)  # noqa: E731
    return (f(batch, n, heads, dk), f(batch, n, kv, dk), f(batch, n, kv, dv),
            np.array([-0.1, -1.0, 0.0, -30.0]), f(batch, heads, dk, dv), f(batch, n, heads, dv),
            f(batch, heads, dk, dv))


def test_attention_is_the_sum_over_earlier_tokens():
    q, k, v, g, init, *_ = inputs()
    out, mag, final, fmag = A.attention(q, k, v, g, 0.7, [9, 4], init)
    for b, real in enumerate((9, 4)):
        for h in range(4):
            lam = np.exp(g[h])
            for t in range(9):
                want = sum(lam ** (t - s) * (q[b, t, h] @ k[b, s, h // 2]) * v[b, s, h // 2]
                           for s in range(t + 1)) + lam ** (t + 1) * q[b, t, h] @ init[b, h]
                np.testing.assert_allclose(out[b, t, h], 0.7 * want if t < real else 0, atol=1e-12)
            want = lam ** real * init[b, h] + sum(
                lam ** (real - 1 - s) * np.outer(k[b, s, h // 2], v[b, s, h // 2])
                for s in range(real))
            np.testing.assert_allclose(final[b, h], want, atol=1e-12)
    assert np.all(np.abs(out) <= mag + 1e-12) and np.all(np.abs(final) <= fmag + 1e-12)


def test_gradients_are_the_slopes():
    q, k, v, g, init, dout, dfinal = inputs()
    real = [9, 5]
    grads = A.attention_backward(dout, q, k, v, g, 0.7, real, init, dfinal)

    def loss(q, k, v, init):
        out, _, final, _ = A.attention(q, k, v, g, 0.7, real, init)
        return (out * dout).sum() + (final * dfinal).sum()

    rng, args = np.random.default_rng(1), (q, k, v, init)
    for i, name in enumerate(("dq", "dk", "dv", "dinitial")):
        move = rng.normal(size=args[i].shape)
        up, down = ([a + s * move if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / 2  # the loss is linear in each
        np.testing.assert_allclose((grads[name][0] * move).sum(), slope, rtol=1e-9)


def test_decays_are_held_to_their_range():
    np.testing.assert_array_equal(A.decays([0.5, 0.0, -np.inf, -1e4]),
                                  np.exp([0.0, 0.0, -200.0, -200.0]))


def test_nearest_8_bit_values():
    assert len(A.E4M3) == 127 and A.E4M3[-1] == 448 and np.all(np.diff(A.E4M3) > 0)
    np.testing.assert_array_equal(A.to_e4m3(A.E4M3), A.E4M3)
    even = A.E4M3[np.arange(126) + np.arange(126) % 2]  # a tie's neighbour of even code
    np.testing.assert_array_equal(A.to_e4m3(A.HALFWAY), even)
    np.testing.assert_array_equal(A.to_e4m3(-A.HALFWAY * (1 - 1e-9)), -A.E4M3[:-1])
    assert np.isnan(A.to_e4m3(np.float32(np.nan)))


def test_quantized_groups_and_blocks():
    x = np.random.default_rng(2).normal(size=(130, 200)).astype(np.float32)
    x[:, :128] = 0
    q, scale = A.quantized(x)
    assert scale.shape == (130, 2) and np.all(scale[:, 0] == 1) and np.all(q[:, :128] == 0)
    assert np.all(np.abs(q).max(1) == 448)
    qb, blocks = A.quantized(x, True)
    qt, turned = A.quantized(x.T, True)
    assert blocks.shape == (2, 2)
    np.testing.assert_array_equal(qb, qt.T)
    np.testing.assert_array_equal(blocks, turned.T)
