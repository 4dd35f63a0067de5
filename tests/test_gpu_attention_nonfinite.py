"""Linear attention with one NaN or infinity in a live value of any input: exactly those outputs are not
finite that the recurrence makes so (an infinity may come out as NaN), and the others are as they are
without it.  Tolerances are those of test_gpu_linear_attention.py with 24-bit states and weights for every
type."""
import numpy as np
import pytest

import _attention_ref as A
import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu

KINDS = ("float32", "float16", "bfloat16")
N, HEADS, KV = 300, 4, 2
REAL = [300, 190]  # partial last chunks of 64 and of 128 tokens
FORWARD, BACKWARD = ("out", "final"), ("dq", "dk", "dv", "dinitial")


class Inputs:
    def __init__(self, dk, dv, kind):
        rng = np.random.default_rng(dk)
        shapes = {"q": (HEADS, dk), "k": (KV, dk), "v": (KV, dv), "dout": (HEADS, dv)}
        self.kind, self.scale = kind, 0.5
        self.host = {x: R.rounded(rng.normal(size=(len(REAL), N) + s), kind)
                     for x, s in shapes.items()}
        for x in ("initial_state", "dfinal"):
            self.host[x] = R.rounded(rng.normal(size=(len(REAL), HEADS, dk, dv)), "float32")
        self.log_decay = np.array([-0.01, -0.2, 0.0, -1.0], np.float32)

    def want(self):
        h = self.host
        with np.errstate(all="ignore"):
            a = A.attention(h["q"], h["k"], h["v"], self.log_decay, self.scale, REAL,
                            h["initial_state"])
            g = A.attention_backward(h["dout"], h["q"], h["k"], h["v"], self.log_decay,
                                     self.scale, REAL, h["initial_state"], h["dfinal"])
        return {"out": a[:2], "final": a[2:], **g}

    def got(self):
        d = {x: R.to_device(a, "float32" if x in ("initial_state", "dfinal") else self.kind)
             for x, a in self.host.items()}
        common = dict(scale=self.scale, n_real=D.to_device(np.asarray(REAL), np.int32),
                      initial_state=d["initial_state"])
        decay = R.to_device(self.log_decay)
        a = S.linear_attention(d["q"], d["k"], d["v"], decay, final_state=True, **common)
        g = S.linear_attention_backward(d["dout"], d["q"], d["k"], d["v"], decay,
                                        dfinal=d["dfinal"], dinitial=True, **common)
        return {"out": a.out, "final": a.final_state, "dq": g.dq, "dk": g.dk, "dv": g.dv,
                "dinitial": g.dinitial}


def check(inputs, where):
    want, got = inputs.want(), inputs.got()
    for name in FORWARD + BACKWARD:
        ref, mag = want[name]
        values, fine = R.values(got[name]), np.isfinite(ref)
        assert not np.isfinite(values[~fine]).any(), f"{where}: {name} lost a value that is not finite"
        kind = "float32" if name in ("final", "dinitial") else inputs.kind
        R.assert_close(values[fine], ref[fine], mag[fine], 200 + N / 8, kind, f"{where}: {name}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dk, dv", ((64, 40), (128, 72)))
@pytest.mark.parametrize("name", ("q", "k", "v", "dout", "initial_state", "dfinal"))
@pytest.mark.parametrize("bad", (np.nan, np.inf, -np.inf))
def test_one_value(kind, dk, dv, name, bad):
    places = {"q": [(0, 40, 1, 3), (1, 150, 2, dk - 1)], "k": [(0, 200, 0, 0), (1, 189, 1, 33)],
              "v": [(0, 127, 1, 5), (1, 64, 0, dv - 1)], "dout": [(0, 299, 3, 7), (1, 100, 0, 0)],
              "initial_state": [(0, 1, 3, 5), (1, 2, dk - 1, 0)],
              "dfinal": [(0, 0, 0, dv - 1), (1, 3, 40, 20)]}
    for at in places[name]:
        inputs = Inputs(dk, dv, kind)
        inputs.host[name][at] = bad
        check(inputs, f"{name}{at}")


@pytest.mark.parametrize("kind", KINDS)
def test_steps(kind):
    """The same of single tokens: each slot's state and output by themselves."""
    rng = np.random.default_rng(0)
    dk, dv, batch = 24, 36, 5
    h = {x: R.rounded(rng.normal(size=(batch, 1) + s), kind)
         for x, s in (("q", (HEADS, dk)), ("k", (KV, dk)), ("v", (KV, dv)))}
    pool = R.rounded(rng.normal(size=(batch, HEADS, dk, dv)), "float32")
    h["q"][0, 0, 1, 3], h["k"][1, 0, 1, 0] = np.nan, np.inf
    h["v"][2, 0, 0, 5], pool[3, 2, 1, 1] = -np.inf, np.inf
    g = np.array([-0.01, -0.2, 0.0, -1.0], np.float32)
    with np.errstate(all="ignore"):
        out, mag, state, smag = A.attention(h["q"], h["k"], h["v"], g, 0.5, None, pool)
    dev = R.to_device(pool)
    got = S.linear_attention_step(dev, *(R.to_device(h[x][:, 0], kind) for x in "qkv"),
                                  R.to_device(g), scale=0.5).out
    for values, ref, size, kind_, units in ((R.values(got), out[:, 0], mag[:, 0], kind, dk + 20),
                                            (R.values(dev), state, smag, "float32", 12)):
        fine = np.isfinite(ref)
        assert not np.isfinite(values[~fine]).any()
        R.assert_close(values[fine], ref[fine], size[fine], units, kind_, "step")
