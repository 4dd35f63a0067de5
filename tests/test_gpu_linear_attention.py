"""Linear attention on the GPU against its 64-bit definition, at the sizes and masks where it can go
wrong.

Tolerances: an output may be off by its own type's rounding, and by units of 2^-24 of its magnitude
(the same formula over absolute values), which count
  - the tensor cores' sums: up to 12 partial products of 16 to 128 terms, each instruction's sum
    taken as 4 units: 200 in all, and a rounding for each chunk that a state is carried through and
    for its decay, an eighth of the tokens;
  - operands in parts of bfloat16 (2^-8 each).  Three parts leave 2^-24 of a value, which the 200
    hold; outputs of 16 bits take the weights within a chunk, and the states, in two parts, which
    leave 2^-16, 256 units, each."""
import numpy as np
import pytest

import _attention_ref as A
import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu

KINDS = ("float32", "float16", "bfloat16")


def steps(n, kind="float32"):
    return 200 + n / 8 + (0 if kind == "float32" else 512)


def i32(a):
    return None if a is None else D.to_device(np.asarray(a), np.int32)


class Case:
    """Inputs of one call, on the host (as the type holds them) and on the device."""

    def __init__(self, kind, batch, n, heads, kv, dk, dv, seed=0, n_real=None, init=False, gap=0,
                 offset=0, log_decay=None):
        rng = np.random.default_rng(seed)
        self.kind, self.n, self.n_real = kind, n, n_real
        self.host, self.dev = {}, {}
        shapes = {"q": (heads, dk), "k": (kv, dk), "v": (kv, dv), "dout": (heads, dv)}
        for name, tail in shapes.items():
            a = R.rounded(rng.normal(size=(batch, n) + tail), kind)
            self.host[name] = a
            self.dev[name] = R.Strided(a, kind, gap=gap, offset=offset, inner=2)
        if log_decay is None:
            log_decay = np.log1p(-(2.0 ** -rng.uniform(1, 9, heads)))
        self.log_decay = np.asarray(log_decay, np.float32)
        self.decay = R.to_device(self.log_decay)
        self.scale = float(np.float32(dk ** -0.5))
        ends = (batch, heads, dk, dv)
        self.init = R.rounded(rng.normal(size=ends), "float32") if init else None
        self.dfinal = R.rounded(rng.normal(size=ends), "float32") if init else None
        self.empty = {name: lambda tail=tail: R.Strided(
            np.zeros((batch, n) + tail), kind, gap=gap, offset=offset, inner=2)
            for name, tail in (("out", shapes["dout"]), ("dq", shapes["q"]), ("dk", shapes["k"]),
                               ("dv", shapes["v"]))}

    def device(self, a):
        return None if a is None else R.to_device(a)

    def forward(self):
        out = self.empty["out"]()
        state = self.device(self.init)
        got = S.linear_attention(self.dev["q"], self.dev["k"], self.dev["v"], self.decay,
                                 scale=self.scale, n_real=i32(self.n_real), initial_state=state,
                                 out=out, final_state=True if state is None else state)
        return out, got.final_state

    def check_forward(self):
        h = self.host
        want = A.attention(h["q"], h["k"], h["v"], self.log_decay, self.scale, self.n_real,
                           self.init)
        out, final = self.forward()
        R.assert_close(out.values(), want[0], want[1], steps(self.n, self.kind), self.kind, "out")
        R.assert_close(R.values(final), want[2], want[3], steps(self.n), "float32", "final state")
        for b, real in enumerate(R.tokens(self.n_real, len(h["q"]), self.n)):
            assert np.all(out.values()[b, real:] == 0)
        assert out.untouched()

    def check_backward(self):
        h, e = self.host, {name: make() for name, make in self.empty.items()}
        want = A.attention_backward(h["dout"], h["q"], h["k"], h["v"], self.log_decay, self.scale,
                                    self.n_real, self.init, self.dfinal)
        got = S.linear_attention_backward(
            self.dev["dout"], self.dev["q"], self.dev["k"], self.dev["v"], self.decay,
            scale=self.scale, n_real=i32(self.n_real), initial_state=self.device(self.init),
            dfinal=self.device(self.dfinal), dq=e["dq"], dk=e["dk"], dv=e["dv"], dinitial=True)
        for name in ("dq", "dk", "dv"):
            R.assert_close(e[name].values(), *want[name], steps(self.n, self.kind), self.kind,
                           name)
            assert e[name].untouched()
        R.assert_close(R.values(got.dinitial), *want["dinitial"], steps(self.n), "float32",
                       "dinitial")


LENGTHS = (1, 2, 17, 63, 64, 65, 128, 129, 200, 321)
DIMS = ((64, 64), (128, 128), (16, 32), (1, 1), (75, 50), (33, 128), (128, 7), (40, 72))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", LENGTHS)
def test_lengths(kind, n):
    Case(kind, 2, n, 2, 1, 64, 48, n).check_forward()
    Case(kind, 1, n, 1, 1, 32, 80, n, init=True).check_forward()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dk, dv", DIMS)
def test_dims(kind, dk, dv):
    for gap, offset in ((0, 0), (8, 8), (3, 1)):
        Case(kind, 2, 150, 4, 2, dk, dv, dk + dv, init=True, gap=gap, offset=offset
             ).check_forward()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dk, dv", DIMS)
def test_backward_dims(kind, dk, dv):
    for gap, offset in ((0, 0), (8, 8), (3, 1)):
        Case(kind, 2, 150, 4, 2, dk, dv, dk + dv, init=True, gap=gap, offset=offset
             ).check_backward()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", LENGTHS)
def test_backward_lengths(kind, n):
    Case(kind, 2, n, 2, 2, 64, 48, n).check_backward()
    Case(kind, 1, n, 3, 1, 32, 80, n, init=True).check_backward()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("init", (False, True))
def test_ragged_rows(kind, init):
    """Rows without tokens, of one, up to a chunk's border and past it; lengths out of range."""
    real = [0, 1, 63, 64, 65, 128, 190, 500, -3]
    for dk, dv in ((128, 64), (64, 128), (24, 50)):
        c = Case(kind, len(real), 190, 2, 1, dk, dv, 7, n_real=real, init=init)
        for b, n in enumerate(R.tokens(real, len(real), 190)):  # never read
            for name in ("q", "k", "v", "dout"):
                c.host[name][b, n:] = np.nan
        c.dev = {name: R.Strided(a, kind, inner=2) for name, a in c.host.items()}
        c.check_forward()
        c.check_backward()


@pytest.mark.parametrize("kind", KINDS)
def test_decays(kind):
    """No decay, decays that forget within a token, that underflow, and out of range."""
    g = [0.0, -0.0, -1e-6, -0.7, -3.0, -50.0, -87.5, -120.0, -300.0, -np.inf, 0.5, np.inf]
    c = Case(kind, 1, 200, len(g), len(g), 32, 24, 3, init=True, log_decay=g)
    c.check_forward()
    c.check_backward()


def test_a_nan_decay_stays_in_its_head():
    c = Case("bfloat16", 1, 130, 3, 3, 64, 64, 5, log_decay=[-0.1, np.nan, -0.2])
    out, final = c.forward()
    assert np.isnan(out.values()[:, :, 1]).all() and np.isnan(R.values(final)[:, 1]).all()
    assert np.isfinite(out.values()[:, :, ::2]).all()
    assert np.isfinite(R.values(final)[:, ::2]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_a_nan_or_infinity_reaches_later_tokens_of_its_head_alone(kind):
    for bad in (np.nan, np.inf):
        c = Case(kind, 2, 200, 2, 2, 64, 64, 6)
        c.host["v"][1, 70, 1, 5] = bad
        c.dev["v"] = R.Strided(c.host["v"], kind, inner=2)
        out, final = c.forward()
        got = out.values()
        touched = np.zeros(got.shape, bool)
        touched[1, 70:, 1, 5] = True
        assert not np.isfinite(got[touched]).any()
        # within the chunk of the token the value's column alone, and no earlier token
        assert np.isfinite(got[~touched]).all()
        f = R.values(final)
        assert not np.isfinite(f[1, 1, :, 5]).any()
        f[1, 1, :, 5] = 0
        assert np.isfinite(f).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n, dk, dv", ((2500, 128, 128), (4100, 64, 64), (1000, 128, 40)))
def test_long_rows_of_few_heads(kind, n, dk, dv):
    """Rows that are split along their tokens."""
    for batch, real in ((1, None), (2, [n, n // 3])):
        c = Case(kind, batch, n, 2, 1, dk, dv, n, n_real=real, init=True,
                 log_decay=[-1e-4, -0.01])
        c.check_forward()
        c.check_backward()


@pytest.mark.parametrize("kind, dk", (("bfloat16", 128), ("bfloat16", 32), ("float16", 128),
                                      ("float16", 64), ("float32", 64)))
def test_segments_of_many_chunks(kind, dk):
    """More heads than a few, so that each segment of a row has tens of chunks: both passes go around
    all their buffers again and again.  The definition in chunks here: 64 bits, 50 tokens at a time."""
    heads, n, dv = 16, 9000, 64
    c = Case(kind, 1, n, heads, heads, dk, dv, 11, log_decay=np.log1p(-(2.0 ** -np.linspace(3, 11, heads))))
    q, k, v = (c.host[x][0].transpose(1, 0, 2) for x in "qkv")
    lam = A.decays(c.log_decay)[:, None, None]
    at = np.arange(50)
    inner = np.where(at[:, None] >= at, lam ** np.maximum(at[:, None] - at, 0), 0)
    s, m = np.zeros((2, heads, dk, dv))
    want, mag = np.zeros((2, heads, n, dv))
    for t in range(0, n, 50):
        cut = slice(t, t + 50)
        for w, size, f in ((want, s, lambda a: a), (mag, m, np.abs)):
            qc, kc, vc = (f(a[:, cut]) for a in (q, k, v))
            w[:, cut] = (qc * lam ** (at[:, None] + 1)) @ size + ((qc @ kc.swapaxes(1, 2)) * inner) @ vc
            size *= lam ** 50
            size += (kc * lam ** (49 - at[:, None])).swapaxes(1, 2) @ vc
    out, final = c.forward()
    R.assert_close(out.values()[0].transpose(1, 0, 2), c.scale * want, c.scale * mag,
                   steps(n, kind), kind, "out")
    R.assert_close(R.values(final)[0], s, m, steps(n), "float32", "state")


def test_many_rows_and_heads():
    """More heads than blocks that fit at once."""
    c = Case("bfloat16", 40, 70, 16, 4, 32, 32, 1, n_real=list(range(0, 80, 2)))
    c.check_forward()
    c.check_backward()


def test_large_values():
    """float16 values whose products and states lie far past float16's range."""
    for kind in KINDS:
        c = Case(kind, 1, 300, 1, 1, 64, 64, 2, log_decay=[0.0])
        for name in ("q", "k", "v"):
            c.host[name] = R.rounded(c.host[name] * 3000, kind)
            c.dev[name] = R.Strided(c.host[name], kind, inner=2)
        c.scale = 2.0 ** -32
        c.check_forward()


@pytest.mark.parametrize("kind", KINDS)
def test_empty_rows_and_batches(kind):
    c = Case(kind, 2, 0, 2, 1, 16, 24, 0, init=True)
    out, final = c.forward()
    np.testing.assert_array_equal(R.values(final), c.init)
    g = S.linear_attention_backward(c.dev["dout"], c.dev["q"], c.dev["k"], c.dev["v"], c.decay,
                                    dfinal=R.to_device(c.dfinal), dinitial=True)
    np.testing.assert_array_equal(R.values(g.dinitial), c.dfinal)
    c = Case(kind, 0, 5, 2, 1, 16, 24, 0)
    assert c.forward()[1].shape == (0, 2, 16, 24)


def test_a_row_without_tokens_keeps_its_state():
    c = Case("bfloat16", 2, 5, 2, 1, 16, 24, 0, init=True, n_real=[0, 0])
    out, final = c.forward()
    np.testing.assert_array_equal(R.values(final), c.init)
    assert np.all(out.values() == 0)
    c = Case("bfloat16", 2, 5, 2, 1, 16, 24, 0, n_real=[0, 0])
    assert np.all(R.values(c.forward()[1]) == 0)


def test_gradients_against_differences():
    """Every input moved by a little either way, in 32 bits: the loss is linear in each of them, so
    the difference has no error of its own but the outputs' roundings."""
    c = Case("float32", 1, 75, 2, 1, 12, 9, 4, init=True)
    rng = np.random.default_rng(1)
    grads = S.linear_attention_backward(
        c.dev["dout"], c.dev["q"], c.dev["k"], c.dev["v"], c.decay, scale=c.scale,
        initial_state=R.to_device(c.init), dfinal=R.to_device(c.dfinal), dinitial=True)

    def loss(**moved):
        a = {**{k: c.host[k] for k in "qkv"}, "init": c.init, **moved}
        got = S.linear_attention(*(R.to_device(a[k]) for k in "qkv"), c.decay, scale=c.scale,
                                 initial_state=R.to_device(a["init"]), final_state=True)
        return ((R.values(got.out) * c.host["dout"]).sum()
                + (R.values(got.final_state) * c.dfinal).sum())

    for name, grad in (("q", grads.dq), ("k", grads.dk), ("v", grads.dv),
                       ("init", grads.dinitial)):
        base = c.init if name == "init" else c.host[name]
        move = R.rounded(np.sign(rng.normal(size=base.shape)), "float32")
        slope = (loss(**{name: base + move}) - loss(**{name: base - move})) / 2
        want = (R.values(grad) * move).sum()
        size = np.abs(R.values(grad)).sum()
        assert abs(slope - want) < 1e-4 * size, name


def test_the_same_call_gives_the_same_bits():
    c = Case("bfloat16", 1, 2000, 2, 1, 128, 128, 9, init=True)
    a, b = c.forward(), c.forward()
    np.testing.assert_array_equal(a[0].values(), b[0].values())
    np.testing.assert_array_equal(R.values(a[1]), R.values(b[1]))


# ---------------------------------------------------------------- single tokens

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dk, dv", DIMS)
def test_step(kind, dk, dv):
    rng = np.random.default_rng(dk)
    heads, kv, slots = 4, 2, [3, -1, 0, 7, 5]
    pool = R.rounded(rng.normal(size=(6, heads, dk, dv)), "float32")
    for gap, offset in ((0, 0), (8, 8), (3, 1)):
        for at in (slots, None):
            batch = 5
            c = Case(kind, batch, 1, heads, kv, dk, dv, dk + gap, gap=gap, offset=offset)
            q, k, v = (R.Strided(c.host[x][:, 0], kind, gap=gap, offset=offset, inner=2)
                       for x in "qkv")
            out = R.Strided(np.zeros((batch, heads, dv)), kind, gap=gap, offset=offset, inner=2)
            state = R.to_device(pool)
            S.linear_attention_step(state, q, k, v, c.decay, scale=c.scale, slots=i32(at),
                                    out=out)
            got, after = out.values(), R.values(state)
            want = pool.copy()
            for b, slot in enumerate(range(batch) if at is None else at):
                if not 0 <= slot < 6:
                    assert np.all(got[b] == 0)
                    continue
                y, m, s, sm = A.attention(*(c.host[x][b:b + 1] for x in "qkv"), c.log_decay,
                                          c.scale, init=pool[slot:slot + 1])
                R.assert_close(got[b], y[0, 0], m[0, 0], dk + 20, kind, "out")
                R.assert_close(after[slot], s[0], sm[0], 12, "float32", "state")
                want[slot] = after[slot]
            np.testing.assert_array_equal(after, want)  # the other slots as they were
            assert out.untouched()


def test_steps_follow_rows():
    """A prompt and single tokens behind it against one prompt of all."""
    c = Case("float32", 2, 40, 4, 2, 32, 16, 8)
    h = c.host
    want, mag, final, fmag = A.attention(h["q"], h["k"], h["v"], c.log_decay, c.scale)
    f = S.linear_attention(*(R.to_device(h[x][:, :30]) for x in "qkv"), c.decay, scale=c.scale,
                           final_state=True)
    for t in range(30, 40):
        o = S.linear_attention_step(f.final_state, *(R.to_device(h[x][:, t]) for x in "qkv"),
                                    c.decay, scale=c.scale)
        R.assert_close(R.values(o.out), want[:, t], mag[:, t], steps(40), "float32", f"token {t}")
    R.assert_close(R.values(f.final_state), final, fmag, steps(40), "float32", "state")


def test_step_of_many_rows():
    c = Case("bfloat16", 300, 1, 8, 2, 64, 64, 8, init=True)
    state = R.to_device(c.init)
    out = S.linear_attention_step(state, *(R.to_device(c.host[x][:, 0], "bfloat16") for x in "qkv"),
                                  c.decay, scale=c.scale).out
    y, m, s, sm = A.attention(*(c.host[x] for x in "qkv"), c.log_decay, c.scale, init=c.init)
    R.assert_close(R.values(out), y[:, 0], m[:, 0], 84, "bfloat16", "out")
    R.assert_close(R.values(state), s, sm, 12, "float32", "state")


@pytest.mark.parametrize("dk, dv", ((64, 64), (75, 52), (128, 100)))
@pytest.mark.parametrize("n", (1, 100, 700))
def test_a_state_at_any_address(n, dk, dv):
    """States whose memory starts a float behind a multiple of 16 bytes: the same bits, and nothing
    beside them is written."""
    c = Case("bfloat16", 2, n, 2, 1, dk, dv, 4, init=True)
    out, final = c.forward()
    size = c.init.size
    around = R.to_device(np.concatenate([[7.0], c.init.ravel(), [7.0]]))
    state = D.DeviceArray(around.ptr + 4, c.init.shape, np.float32, around)
    moved = S.linear_attention(c.dev["q"], c.dev["k"], c.dev["v"], c.decay, scale=c.scale,
                               initial_state=state, final_state=state)
    np.testing.assert_array_equal(R.values(moved.out), out.values())
    got = R.values(around)
    np.testing.assert_array_equal(got[1:-1], R.values(final).ravel())
    assert got[0] == 7.0 and got[size + 1] == 7.0
