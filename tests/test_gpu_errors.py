"""A call that the runtime refuses says so once: the next call, which is right, is not blamed for it."""
import numpy as np
import pytest

import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu


def product(rows=16):
    x = S.quantize_q8(R.to_device(np.ones((rows, 256)), "bfloat16"))
    w = S.quantize_q8(R.to_device(np.ones((128, 256)), "bfloat16"), blocks=True)
    return x, w


def spoilt_capture(call):
    """`call` on a stream whose recording has been spoilt by a wait."""
    stream = D.Stream()
    with pytest.raises(RuntimeError):
        with D.Graph.capture(stream):
            with pytest.raises(RuntimeError):
                stream.synchronize()
            with pytest.raises(RuntimeError):
                call()


def too_much_memory():
    with pytest.raises(RuntimeError):
        D.empty((1 << 46,), np.uint8)


def refused_product():
    x, w = product()
    out = D.empty((16, 128), D.bfloat16)
    D.current_stream().synchronize()
    spoilt_capture(lambda: S.matmul_q8(x.out, x.scale, w.out, w.scale, out=out))


def refused_attention():
    q = R.to_device(np.ones((1, 4, 2, 16)), "bfloat16")  # one launch, no workspace
    decay, out = R.to_device(np.zeros(2)), D.empty((1, 4, 2, 16), D.bfloat16)
    D.current_stream().synchronize()
    spoilt_capture(lambda: S.linear_attention(q, q, q, decay, out=out))


def quantize():
    a = S.quantize_q8(R.to_device(np.ones((4, 128)), "float32"))
    np.testing.assert_array_equal(R.values(a.scale), np.full((4, 1), np.float32(1 / 448)))


def norm():
    out = S.rms_norm(R.to_device(np.ones((4, 64))), R.to_device(np.ones(64)), eps=0.0).out
    np.testing.assert_allclose(R.values(out), 1.0, rtol=2.0 ** -20)


def token():
    one = R.to_device(np.ones((1, 1, 8)))
    out = S.linear_attention_step(D.zeros((1, 1, 8, 8), np.float32), one, one, one,
                                  R.to_device(np.zeros(1))).out
    np.testing.assert_array_equal(R.values(out), 8.0)


def attention():
    one = R.to_device(np.ones((1, 1, 1, 8)))
    out = S.linear_attention(one, one, one, R.to_device(np.zeros(1))).out
    np.testing.assert_array_equal(R.values(out), 8.0)


def multiply():
    x, w = product()
    out = S.matmul_q8(x.out, x.scale, w.out, w.scale, dtype=np.float32)
    np.testing.assert_allclose(R.values(out), 256.0, rtol=2.0 ** -20)


@pytest.mark.parametrize("after", (quantize, norm, token, attention, multiply))
@pytest.mark.parametrize("refused", (too_much_memory, refused_product, refused_attention))
def test_the_call_after_a_refused_one(refused, after):
    refused()
    after()
