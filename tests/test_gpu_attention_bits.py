"""Linear attention where its sums cancel: outputs of 16 bits come from states and weights within a chunk
that hold 24 bits, as outputs of 32 bits do.

Everything here is a difference of two values of [1, 2) with random bits down to 2^-23 that lie within
2^-13 of one another, under no decay and a scale of 1, so the weights are exact.  What may be off, in
units of 2^-24 of the magnitude (the sum of both): the tensor cores' sums, each instruction's taken as 4
units; one instruction makes a score, and one for each pair of parts an output (3 for bfloat16, 5 for
float16, 6 for float32); the sum of an output's two sources, a unit, and its scale, another.  An output's
own rounding is relative to the difference."""
import numpy as np
import pytest

import _sequence_ref as R
import salt_b200 as S

pytestmark = pytest.mark.gpu

PRODUCTS = {"bfloat16": 3, "float16": 5, "float32": 6}
KINDS = tuple(PRODUCTS)
BATCH, HEADS = 4, 8


def pairs(rng, *shape):
    """Two arrays of 24-bit values of [1, 2), less than 2^-13 apart."""
    a = np.floor(rng.uniform(1.001, 1.998, shape) * 2.0 ** 23) / 2.0 ** 23
    b = a + np.floor(rng.uniform(-1, 1, shape) * 2.0 ** 10) / 2.0 ** 23
    return a, b


def three(a):
    """Values of bfloat16 (and float16) that add up to a, in a last axis of 3."""
    parts = []
    for at in (7, 15, 23):
        x = np.floor(a * 2.0 ** at) / 2.0 ** at
        parts.append(x)
        a = a - x
    return np.stack(parts, -1)


def call(name, arrays, kind, **states):
    """One output of a call on host arrays; absent ones are zero."""
    d = {k: R.to_device(v, kind) for k, v in arrays.items()}
    states = {k: R.to_device(v) for k, v in states.items()}
    decay = R.to_device(np.zeros(HEADS))
    if name == "out":
        return R.values(S.linear_attention(d["q"], d["k"], d["v"], decay, **states).out)
    got = S.linear_attention_backward(d["dout"], d["q"], d["k"], d["v"], decay, **states)
    return R.values(getattr(got, name))


# An output is a sum over tokens of (one of its arrays . `left`) times `right`, and of a state's rows
# or columns: (own, left, right, earlier tokens, the state's name, whether it is read across).
ROLES = {"out": ("q", "k", "v", True, "initial_state", False),
         "dq": ("dout", "v", "k", True, "initial_state", True),
         "dk": ("v", "dout", "q", False, "dfinal", True),
         "dv": ("k", "q", "dout", False, "dfinal", False)}


def zeros(n, dk, dv):
    return {"q": np.zeros((BATCH, n, HEADS, dk)), "k": np.zeros((BATCH, n, HEADS, dk)),
            "v": np.zeros((BATCH, n, HEADS, dv)), "dout": np.zeros((BATCH, n, HEADS, dv))}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", (48, 128))
@pytest.mark.parametrize("name", ROLES)
@pytest.mark.parametrize("n", (3, 128, 300))
def test_weights_within_a_chunk(kind, dim, name, n):
    """The difference of two tokens' scores, at every token that both reach: the tokens beside one
    another, and a block of 32 tokens apart."""
    own, left, right, forward, _, _ = ROLES[name]
    rng = np.random.default_rng(n + dim)
    for s0, s1 in ((0, 1), (n - 2, n - 1), (n // 2, min(n // 2 + 37, n - 1))):
        arrays = zeros(n, dim, dim)
        a, b = pairs(rng, BATCH, HEADS)
        arrays[own][..., :3] = 1
        arrays[left][:, s0, :, :3], arrays[left][:, s1, :, :3] = three(a), three(b)
        arrays[right][:, s0], arrays[right][:, s1] = 1, -1
        got = call(name, arrays, kind)
        reach = slice(s1, n) if forward else slice(0, s0 + 1)
        got = got[:, reach]
        want = np.broadcast_to((a - b)[:, None, :, None], got.shape)
        mag = np.broadcast_to((a + b)[:, None, :, None], got.shape)
        R.assert_close(got, want, mag, 4 * (1 + PRODUCTS[kind]) + 2, kind, f"{name} {s0} {s1}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", (48, 128))
@pytest.mark.parametrize("name", ROLES)
@pytest.mark.parametrize("n", (1, 128, 300))
def test_states(kind, dim, name, n):
    """The difference of two rows of the state that the call starts from."""
    own, _, _, _, state, across = ROLES[name]
    rng = np.random.default_rng(n + dim)
    arrays = zeros(n, dim, dim)
    a, b = pairs(rng, BATCH, HEADS, dim)
    arrays[own][..., 0], arrays[own][..., 1] = 1, -1
    s = np.zeros((BATCH, HEADS, dim, dim))
    s[:, :, 0], s[:, :, 1] = a, b
    got = call(name, arrays, kind, **{state: s.swapaxes(-1, -2) if across else s})
    want, mag = (np.broadcast_to(x[:, None], got.shape) for x in (a - b, a + b))
    R.assert_close(got, want, mag, 4 * PRODUCTS[kind] + 2, kind, name)
