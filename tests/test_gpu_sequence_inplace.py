"""States that are updated in place: the convolution's and the scan's final state may be the array of
the initial one.  Rows are cut among threads of several warps and blocks, none of which may read a
state that another has replaced already."""
import numpy as np
import pytest

import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", range(2, 9))
@pytest.mark.parametrize("batch, n, dim", [(1, 9, 256), (2, 40, 1001), (1, 24, 8192), (3, 8, 4096)])
def test_conv_in_place(batch, n, dim, width):
    """Every run of tokens but the first keeps to the row's own tokens, whatever the first writes."""
    rng = np.random.default_rng(width)
    x, w = rng.normal(size=(batch, n, dim)), rng.normal(size=(dim, width))
    init = rng.normal(size=(batch, dim, width - 1))
    x, w, init = (R.rounded(a, "float32") for a in (x, w, init))
    n_real = [n, n - 2, 5][:batch]
    ref, mag, final = R.conv(x, w, None, n_real, init)
    dx, dw, real = R.to_device(x), R.to_device(w), D.to_device(np.array(n_real), np.int32)
    apart = S.causal_conv(dx, dw, n_real=real, initial_state=R.to_device(init), final_state=True)
    R.assert_close(R.values(apart.out), ref, mag, 2 * width + 20, "float32", "out")
    for _ in range(20):
        state = R.to_device(init)
        out = S.causal_conv(dx, dw, n_real=real, initial_state=state, final_state=state).out
        np.testing.assert_array_equal(out.numpy(), apart.out.numpy())
        np.testing.assert_array_equal(R.values(state), final)


@pytest.mark.parametrize("n", [40, 700])  # whole rows, and rows in chunks
def test_scan_in_place(n):
    rng = np.random.default_rng(n)
    batch, dim, state = 2, 100, 16
    f = lambda *s: R.to_device(rng.normal(size=s))  # noqa: E731
    x, delta, B, C = f(batch, n, dim), f(batch, n, dim), f(batch, n, 1, state), f(batch, n, 1, state)
    A, init = R.to_device(-rng.uniform(0.1, 1, (dim, state))), rng.normal(size=(batch, dim, state))
    apart = S.selective_scan(x, delta, A, B, C, initial_state=R.to_device(init), final_state=True)
    for _ in range(10):
        h = R.to_device(init)
        got = S.selective_scan(x, delta, A, B, C, initial_state=h, final_state=h)
        np.testing.assert_array_equal(got.out.numpy(), apart.out.numpy())
        np.testing.assert_array_equal(h.numpy(), apart.final_state.numpy())
