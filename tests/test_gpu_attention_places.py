"""Linear attention whose outputs leave through the place of a chunk's values (bfloat16 heads over 64), over
many chunks of a block: by tensor copies, and value by value where no tensor copy takes the output."""
import numpy as np
import pytest

import _attention_ref as A
import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu

N, HEADS, KV = 900, 3, 1
REAL = [900, 641, 640, 0, 127, 899]


@pytest.mark.parametrize("dk, dv", ((128, 128), (100, 77), (72, 1), (65, 64), (77, 100)))
@pytest.mark.parametrize("gap, offset", ((0, 0), (8, 16), (3, 1)))
def test_many_chunks(dk, dv, gap, offset):
    """Enough rows and heads to keep each row in one block."""
    rng = np.random.default_rng(dk + gap)
    rows = [REAL[b % len(REAL)] for b in range(40)]
    few = range(len(REAL))  # the definition of these; the rows behind are the same ones again
    h = {x: R.rounded(rng.normal(size=(len(REAL), N) + s), "bfloat16")
         for x, s in (("q", (HEADS, dk)), ("k", (KV, dk)), ("v", (KV, dv)), ("dout", (HEADS, dv)))}
    dev = {x: R.Strided(a[[b % len(REAL) for b in range(40)]], "bfloat16", gap=gap, offset=offset,
                        inner=2) for x, a in h.items()}
    out = {x: R.Strided(np.zeros(dev[of].shape), "bfloat16", gap=gap, offset=offset, inner=2)
           for x, of in (("out", "dout"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    g = np.array([-0.001, -0.05, -0.7], np.float32)
    common = dict(scale=0.25, n_real=D.to_device(np.asarray(rows), np.int32))
    args = dev["q"], dev["k"], dev["v"], R.to_device(g)
    final = S.linear_attention(*args, out=out["out"], final_state=True, **common).final_state
    S.linear_attention_backward(dev["dout"], *args, dq=out["dq"], dk=out["dk"], dv=out["dv"], **common)
    a = A.attention(h["q"], h["k"], h["v"], g, 0.25, REAL)
    want = {"out": a[:2], **A.attention_backward(h["dout"], h["q"], h["k"], h["v"], g, 0.25, REAL)}
    for name, o in out.items():
        got = o.values()
        for b in range(len(REAL), 40):
            np.testing.assert_array_equal(got[b], got[b % len(REAL)])
        R.assert_close(got[few], *want[name], 200 + N / 8, "bfloat16", name)
        assert o.untouched()
    R.assert_close(R.values(final)[few], a[2], a[3], 200 + N / 8, "float32", "final state")
