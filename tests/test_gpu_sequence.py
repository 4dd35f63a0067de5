"""The sequence operators on the GPU against their 64-bit definitions, at the sizes and masks where
they can go wrong.

Tolerances: an output may be off by its own type's rounding, and by the roundings of the 32-bit
evaluation, each at most 2^-24 of the magnitude that it happens at (the same formula over absolute
values, from _sequence_ref).  Their numbers are counts of operations, doubled for the fast
exponential and division (2 ulp each):
  norm            dim + 20: the sum of squares, then a handful
  conv            2 * width + 20, times 2 for the slope backward; a sum over tokens adds their number
  scan            a state of age k has k roundings of its own and of exp(s A), which is off by
                  12 + 12 |s A| ulp (the argument's own rounding, and that of s, times |s A|):
                  len * (12 + 12 |s A|), twice that backward, plus the terms of the sums."""
import numpy as np
import pytest

import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu

KINDS = ("float32", "float16", "bfloat16")


def i32(a):
    return None if a is None else D.to_device(np.asarray(a), np.int32)


# ---------------------------------------------------------------- norm

NORM_DIMS = (1, 7, 8, 64, 250, 257, 1024, 1025, 2500, 4096, 4104, 8200, 16384)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", NORM_DIMS)
def test_norm(kind, dim):
    rng = np.random.default_rng(dim)
    rows, eps = 5, 1e-5
    for wide, w_kind, gap in (((kind, kind, 0)), ("float32", "float32", 8), (kind, "float32", 3)):
        x = R.rounded(rng.normal(size=(rows, dim)), kind)
        res = R.rounded(2 * rng.normal(size=(rows, dim)), wide)
        x[3] = res[3] = 0  # eps alone
        w = R.rounded(1 + 0.3 * rng.normal(size=dim), w_kind)
        r, rstd, y = R.norm(x, w, res, eps)
        dx = R.Strided(x, kind, gap=gap, offset=gap)
        dres = R.Strided(res, wide, gap=gap, offset=2 * gap)
        out = R.Strided(np.zeros_like(x), kind, gap=gap)
        # the residual is updated in place
        got = S.rms_norm(dx, R.to_device(w, w_kind), residual=dres, eps=eps, out=out,
                         residual_out=dres, rstd=True)
        R.assert_close(dres.values(), r, np.abs(x) + np.abs(res), 1, wide, "residual")
        R.assert_close(R.values(got.rstd), rstd, rstd, dim + 20, "float32", "rstd")
        mag = (np.abs(x) + np.abs(res)) * rstd[:, None] * np.abs(w)
        R.assert_close(out.values(), y, mag, dim + 20, kind, "out")
        if gap:
            assert out.untouched() and dres.untouched() and dx.untouched()
        # without a residual, over x itself
        y0 = R.norm(x, w, None, eps)[2]
        S.rms_norm(dx, R.to_device(w, w_kind), eps=eps, out=dx)
        R.assert_close(dx.values(), y0, np.abs(y0), dim + 20, kind, "in place")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", (1, 31, 128, 200, 1000, 1024, 1031, 2048, 5000, 9000))
@pytest.mark.parametrize("group", (0, 32, 64, 128, 256))
def test_norm_in_8_bits(kind, dim, group):
    rng = np.random.default_rng(dim + group)
    rows = 3
    x = R.rounded(rng.normal(size=(rows, dim)), kind)
    w = R.rounded(1 + 0.3 * rng.normal(size=dim), kind)
    w[:min(dim, 128)] = 0  # whole groups of zeros
    y = R.norm(x, w, None, 1e-5)[2]
    got = S.rms_norm_q8(R.to_device(x, kind), R.to_device(w, kind), group=group)
    assert got.out.dtype == D.float8_e4m3
    g = group or dim
    q, scale = R.values(got.out), R.values(got.scale)
    assert scale.shape == (rows, -(-dim // g))
    for p in range(scale.shape[1]):
        part, qp = y[:, p * g:(p + 1) * g], q[:, p * g:(p + 1) * g]
        most = np.abs(part).max(1)
        want = np.where(most > 0, most / 448, 1)
        R.assert_close(scale[:, p], want, want, dim + 22, "float32", "scale")
        # the nearest of values 1/16 apart (relative), or 2^-9 under 2^-6
        limit = np.maximum(np.abs(part / want[:, None]) / 16, 2.0 ** -10) * (1 + 1e-3)
        assert np.all(np.abs(qp - part / want[:, None]) <= limit)


def test_norm_8_bits_rounds_to_the_nearest():
    """With a weight that undoes the norm, the values in front of the rounding are known."""
    row = np.array([448.0] + [1.0, 1.0625, 1.1, 1.1875, 2.125, -17.0, 300.0, 0.001, 0.0009]
                   + [0.0] * 22)
    w = np.ones(32)
    x = np.tile(row, (1, 1))
    rms = np.sqrt(np.mean(x * x))
    q = R.values(S.rms_norm_q8(R.to_device(x), R.to_device(w * rms), eps=0.0, group=32).out)[0]
    # 1.0625, 1.1875, 2.125 and -17 lie halfway between neighbours: within one rounding of the
    # scaled value either is right, so they are only held to the distance
    for v, got in zip(row, q):
        step = max(2.0 ** (np.floor(np.log2(max(abs(v), 2.0 ** -6))) - 3), 2.0 ** -9)
        assert abs(got - v) <= step / 2 * (1 + 1e-4), (v, got)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", NORM_DIMS)
def test_norm_backward(kind, dim):
    rng = np.random.default_rng(dim + 1)
    for rows, wide, gap, with_res in ((1, kind, 0, False), (7, "float32", 4, True),
                                      (700, kind, 8, True)):
        if rows * dim > 2_000_000:
            rows = 40
        x = R.rounded(rng.normal(size=(rows, dim)), wide)
        dy = R.rounded(rng.normal(size=(rows, dim)), kind)
        dres = R.rounded(rng.normal(size=(rows, dim)), wide) if with_res else None
        w = R.rounded(1 + 0.3 * rng.normal(size=dim), kind)
        rstd = R.rounded(1 / np.sqrt(np.mean(x * x, -1) + 1e-5), "float32")
        dx, mag, dw, dwmag = R.norm_backward(dy, x, w, rstd, dres)
        ddy, dxx = R.Strided(dy, kind, gap=gap), R.Strided(x, wide, gap=gap, offset=gap)
        dd = None if dres is None else R.Strided(dres, wide, gap=gap)
        got = S.rms_norm_backward(ddy, dxx, R.to_device(w, kind), R.to_device(rstd),
                                  dresidual=dd, dx=dd)
        r = dd.values() if dd is not None else R.values(got.dx)
        R.assert_close(r, dx, mag, dim + 20, wide, "dx")
        R.assert_close(R.values(got.dweight), dw, dwmag, rows + 20, "float32", "dweight")
    again = S.rms_norm_backward(ddy, dxx, R.to_device(w, kind), R.to_device(rstd))
    more = S.rms_norm_backward(ddy, dxx, R.to_device(w, kind), R.to_device(rstd))
    assert np.array_equal(again.dweight.numpy(), more.dweight.numpy())  # the same bits


def test_norm_of_no_rows_and_of_nonfinite_rows():
    w = R.to_device(np.ones(64))
    assert S.rms_norm(D.empty((0, 64), np.float32), w).out.shape == (0, 64)
    g = S.rms_norm_backward(D.empty((0, 64), np.float32), D.empty((0, 64), np.float32), w,
                            D.empty((0,), np.float32))
    assert not np.any(g.dweight.numpy())
    x = np.ones((3, 64))
    x[1, 5], x[2, 7] = np.nan, np.inf
    y = R.values(S.rms_norm(R.to_device(x), w).out)
    assert np.all(np.isfinite(y[0])) and np.all(np.isnan(y[1])) and np.isnan(y[2, 7])
    x3 = np.random.default_rng(0).normal(size=(2, 3, 64))  # leading axes fold
    y3 = R.values(S.rms_norm(R.Strided(x3, gap=8), w).out)
    R.assert_close(y3.reshape(6, 64), R.norm(x3.reshape(6, 64), np.ones(64), None, 1e-5)[2],
                   np.abs(y3.reshape(6, 64)), 84, "float32", "folded")


# ---------------------------------------------------------------- convolution

CONV = [  # batch, len, dim, width, n_real, state?
    (1, 1, 1, 1, None, False), (2, 1, 8, 4, None, True), (2, 3, 7, 4, None, True),
    (3, 40, 64, 4, [40, 0, 17], True), (2, 65, 130, 3, [64, 2], True),
    (2, 33, 24, 2, [-5, 99], False), (1, 70, 9, 8, None, True), (2, 530, 136, 4, [513, 530], True),
    (4, 5, 16, 6, [1, 2, 3, 4], True), (2, 0, 8, 4, None, True), (1, 2100, 8, 4, None, False)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", CONV, ids=str)
@pytest.mark.parametrize("act", [True, False])
def test_conv(kind, case, act):
    batch, n, dim, width, n_real, with_state = case
    rng = np.random.default_rng(n + dim)
    for w_kind, gap, with_bias in ((kind, 8, True), ("float32", 3, False)):
        x = R.rounded(rng.normal(size=(batch, n, dim)), kind)
        for b, real in enumerate(R.tokens(n_real, batch, n)):
            x[b, real:] = np.nan  # not to be read
        w = R.rounded(rng.normal(size=(dim, width)), w_kind)
        bias = R.rounded(rng.normal(size=dim), w_kind) if with_bias else None
        init = R.rounded(rng.normal(size=(batch, dim, width - 1)), kind) if with_state else None
        ref, mag, final = R.conv(x, w, bias, n_real, init, act)
        dx, out = R.Strided(x, kind, gap=gap, offset=gap), R.Strided(x * 0 + 7, kind, gap=gap)
        state = R.to_device(init, kind) if with_state else D.empty((batch, dim, width - 1),
                                                                   R.dtype_of(kind))
        S.causal_conv(dx, R.to_device(w, w_kind), None if bias is None else
                      R.to_device(bias, w_kind), n_real=i32(n_real),
                      initial_state=state if with_state else None, silu=act, out=out,
                      final_state=state)
        R.assert_close(out.values(), ref, mag, 2 * width + 20, kind, "out")
        np.testing.assert_array_equal(R.values(state), final)
        assert out.untouched()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", CONV, ids=str)
@pytest.mark.parametrize("act", [True, False])
def test_conv_backward(kind, case, act):
    batch, n, dim, width, n_real, with_state = case
    rng = np.random.default_rng(n + dim + 1)
    for w_kind, gap, with_bias in ((kind, 8, True), ("float32", 3, False)):
        x = R.rounded(rng.normal(size=(batch, n, dim)), kind)
        dy = R.rounded(rng.normal(size=(batch, n, dim)), kind)
        for b, real in enumerate(R.tokens(n_real, batch, n)):
            x[b, real:] = dy[b, real:] = np.nan
        w = R.rounded(rng.normal(size=(dim, width)), w_kind)
        bias = R.rounded(rng.normal(size=dim), w_kind) if with_bias else None
        init = R.rounded(rng.normal(size=(batch, dim, width - 1)), kind) if with_state else None
        ref = R.conv_backward(dy, x, w, bias, n_real, init, act)
        dx = R.Strided(x * 0 + 7, kind, gap=gap)
        args = (R.Strided(dy, kind, gap=gap), R.Strided(x, kind, gap=gap, offset=gap),
                R.to_device(w, w_kind), None if bias is None else R.to_device(bias, w_kind))
        more = dict(n_real=i32(n_real), silu=act,
                    initial_state=R.to_device(init, kind) if with_state else None)
        got = S.causal_conv_backward(*args, **more, dx=dx, dinitial=True)
        assert (got.dbias is None) == (bias is None)
        steps, tokens = 2 * (4 * width + 40), batch * n
        R.assert_close(dx.values(), *ref["dx"], steps, kind, "dx")
        R.assert_close(R.values(got.dinitial), *ref["dinitial"], steps, kind, "dinitial")
        R.assert_close(R.values(got.dweight), *ref["dweight"], steps + tokens, "float32",
                       "dweight")
        if bias is not None:
            R.assert_close(R.values(got.dbias), *ref["dbias"], steps + tokens, "float32", "dbias")
        assert dx.untouched()
        again = S.causal_conv_backward(*args, **more)
        assert np.array_equal(again.dweight.numpy(), got.dweight.numpy())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width, dim", [(1, 5), (2, 64), (3, 33), (4, 1), (4, 8), (4, 260), (8, 16)])
def test_conv_step(kind, width, dim):
    """Steps from a state continue the row: as causal_conv over the same tokens, slot by slot, with
    empty rows and slots that nobody names left alone."""
    rng = np.random.default_rng(width * dim)
    batch, pool = 4, 6
    slots = [5, -1, 0, 2]
    w = R.rounded(rng.normal(size=(dim, width)), kind)
    bias = R.rounded(rng.normal(size=dim), kind)
    state = R.rounded(rng.normal(size=(pool, dim, width - 1)), kind)
    x = R.rounded(rng.normal(size=(batch, 3, dim)), kind)
    live = [0, 2, 3]
    ref, mag, final = R.conv(x[live], w, bias, None, state[[slots[b] for b in live]])
    dstate, dw, db = R.to_device(state, kind), R.to_device(w, kind), R.to_device(bias, kind)
    for t in range(3):
        out = S.causal_conv_step(R.Strided(x[:, t], kind, gap=5), dstate, dw, db,
                                 slots=i32(slots)).out
        y = R.values(out)
        R.assert_close(y[live], ref[:, t], mag[:, t], 2 * width + 20, kind, f"out {t}")
        assert not np.any(y[1])
    after = state.copy()
    after[[slots[b] for b in live]] = final
    np.testing.assert_array_equal(R.values(dstate), after)
    # a slot past the pool is empty too; without slots row b is slot b
    S.causal_conv_step(R.to_device(x[:, 0], kind), dstate, dw, db, slots=i32([pool, -7, 99, -1]))
    np.testing.assert_array_equal(R.values(dstate), after)
    y = R.values(S.causal_conv_step(R.to_device(x[:, 0], kind), dstate, dw, db).out)
    ref, mag, _ = R.conv(x[:, :1], w, bias, None, after[:batch])
    R.assert_close(y, ref[:, 0], mag[:, 0], 2 * width + 20, kind, "without slots")


# ---------------------------------------------------------------- scan

SCAN = [  # batch, len, dim, state, groups, n_real, initial state?
    (1, 1, 1, 1, 1, None, False), (2, 5, 64, 16, 1, None, True), (1, 16, 65, 16, 1, None, False),
    (3, 17, 48, 16, 2, [17, 0, 9], True), (2, 33, 130, 12, 1, [33, 32], True),
    (2, 31, 24, 4, 3, None, True), (1, 47, 72, 3, 1, None, True), (2, 40, 20, 8, 1, [1, 40], False),
    (1, 35, 66, 7, 2, None, True), (1, 50, 40, 32, 1, None, True), (1, 18, 34, 20, 2, [99], True),
    (2, 33, 18, 64, 1, [33, -3], True), (1, 20, 17, 50, 1, None, False),
    (2, 300, 16, 16, 1, [300, 140], True), (1, 700, 8, 4, 1, None, True),
    (2, 290, 8, 64, 1, [0, 257], True), (1, 0, 8, 16, 1, None, True)]


def scan_inputs(case, kind, gated, plus, seed):
    batch, n, dim, state, groups, n_real, with_init = case
    rng = np.random.default_rng(seed)
    v = {"x": rng.normal(size=(batch, n, dim)), "delta": 0.7 * rng.normal(size=(batch, n, dim)),
         "B": rng.normal(size=(batch, n, groups, state)),
         "C": rng.normal(size=(batch, n, groups, state))}
    if not plus:
        v["delta"] = 0.05 + 0.1 * np.abs(v["delta"])
    if gated:
        v["z"] = rng.normal(size=(batch, n, dim))
    v = {k: R.rounded(a, kind) for k, a in v.items()}
    for b, real in enumerate(R.tokens(n_real, batch, n)):
        for a in v.values():
            a[b, real:] = np.nan
    f = {"A": -rng.uniform(0.5, 1.5, (dim, state)) * np.arange(1, state + 1)}
    if gated:  # the optional parts come and go together
        f["Dskip"] = rng.normal(size=dim)
        f["bias"] = rng.uniform(-4, -1, dim) if plus else rng.uniform(0.0, 0.1, dim)
    if with_init:
        f["init"] = rng.normal(size=(batch, dim, state))
    return v | {k: R.rounded(a, "float32") for k, a in f.items()}, rng


def scan_call(v, kind, n_real, gap):
    """Device arguments of the forward, positional and by name."""
    wide = {k: R.Strided(v[k], kind, gap=gap, offset=gap) for k in ("x", "delta", "z") if k in v}
    wide |= {k: R.Strided(v[k], kind, gap=gap, inner=2) for k in ("B", "C")}
    flat = {k: R.to_device(v[k]) for k in ("A", "Dskip", "bias", "init") if k in v}
    args = (wide["x"], wide["delta"], flat["A"], wide["B"], wide["C"])
    named = dict(D=flat.get("Dskip"), z=wide.get("z"), delta_bias=flat.get("bias"),
                 n_real=i32(n_real))
    return args, named, flat.get("init")


FORMS = [(True, True, 8), (False, False, 3), (False, True, 0)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", SCAN, ids=str)
@pytest.mark.parametrize("gated, plus, gap", FORMS)
def test_scan(kind, case, gated, plus, gap):
    batch, n, dim, state, groups, n_real, with_init = case
    v, rng = scan_inputs(case, kind, gated, plus, n + dim + state)
    ref, _, most = R.scan(**v, plus=plus, n_real=n_real)
    args, named, init = scan_call(v, kind, n_real, gap)
    out = R.Strided(np.zeros((batch, n, dim)) + 7, kind, gap=gap)
    final = init if with_init else D.empty((batch, dim, state), np.float32)
    S.selective_scan(*args, **named, softplus=plus, initial_state=init, out=out, final_state=final)
    steps = n * (12 + 12 * most) + state + 40
    R.assert_close(out.values(), *ref["out"], steps, kind, "out")
    R.assert_close(R.values(final), *ref["final"], steps, "float32", "final")
    assert out.untouched()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", SCAN, ids=str)
@pytest.mark.parametrize("gated, plus, gap", FORMS)
def test_scan_backward(kind, case, gated, plus, gap):
    batch, n, dim, state, groups, n_real, with_init = case
    v, rng = scan_inputs(case, kind, gated, plus, n + dim + state + 1)
    dy = R.rounded(rng.normal(size=(batch, n, dim)), kind)
    for b, real in enumerate(R.tokens(n_real, batch, n)):
        dy[b, real:] = np.nan
    df = R.rounded(rng.normal(size=(batch, dim, state)), "float32") if with_init else None
    ref, most = R.scan_backward(dy, **v, plus=plus, n_real=n_real, dfinal=df)
    args, named, init = scan_call(v, kind, n_real, gap)
    marks = S.selective_scan(*args, **named, softplus=plus, initial_state=init,
                             checkpoints=True).checkpoints
    outs = {k: R.Strided(np.zeros((batch, n, dim)) + 7, kind, gap=gap)
            for k in ("dx", "ddelta") + (("dz",) if gated else ())}
    ddy = R.Strided(dy, kind, gap=gap)
    call = dict(named, softplus=plus, checkpoints=marks,
                dfinal=None if df is None else R.to_device(df))
    got = S.selective_scan_backward(ddy, *args, **call, **outs, dinitial=True)
    steps = 2 * n * (12 + 12 * most) + state + 80
    for k, o in outs.items():
        R.assert_close(o.values(), *ref[k], steps, kind, k)
        assert o.untouched()
    for k in ("dB", "dC"):
        R.assert_close(R.values(getattr(got, k)), *ref[k], steps + dim, kind, k)
    for k in ("dA", "dD", "ddelta_bias", "dinitial"):
        if getattr(got, k) is None:
            assert not gated and k in ("dD", "ddelta_bias")
            continue
        R.assert_close(R.values(getattr(got, k)), *ref[k], steps + batch * n, "float32", k)
    again = S.selective_scan_backward(ddy, *args, **call)
    for k in ("dA", "dB", "dC"):
        assert getattr(again, k).numpy().tobytes() == getattr(got, k).numpy().tobytes(), k


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim, state, groups", [(1, 1, 1), (64, 16, 1), (70, 12, 2), (9, 3, 1),
                                                (40, 8, 4), (66, 32, 1), (33, 64, 1), (20, 17, 2)])
@pytest.mark.parametrize("gated, plus", [(True, True), (False, False)])
def test_scan_step(kind, dim, state, groups, gated, plus):
    """Steps continue a row slot by slot; empty rows and unnamed slots keep out of it."""
    batch, pool, n = 4, 6, 3
    v, rng = scan_inputs((batch, n, dim, state, groups, None, False), kind, gated, plus, dim)
    states = R.rounded(rng.normal(size=(pool, dim, state)), "float32")
    slots, live = [3, 5, 6, 0], [0, 1, 3]
    some = {k: a[live] if k in ("x", "delta", "B", "C", "z") else a for k, a in v.items()}
    ref, _, most = R.scan(**some, plus=plus, init=states[[slots[b] for b in live]])
    dev = R.to_device(states)
    flat = {k: R.to_device(v[k]) for k in ("A", "Dskip", "bias") if k in v}
    for t in range(n):
        at = {k: R.Strided(v[k][:, t], kind, gap=5, inner=2 if k in "BC" else 1)
              for k in ("x", "delta", "B", "C", "z") if k in v}
        out = S.selective_scan_step(dev, at["x"], at["delta"], flat["A"], at["B"], at["C"],
                                    D=flat.get("Dskip"), z=at.get("z"),
                                    delta_bias=flat.get("bias"), softplus=plus, slots=i32(slots))
        y = R.values(out.out)
        R.assert_close(y[live], ref["out"][0][:, t], ref["out"][1][:, t],
                       (t + 1) * (12 + 12 * most) + state + 40, kind, f"out {t}")
        assert not np.any(y[2])
    after = R.values(dev)
    keep = [s for s in range(pool) if s not in slots]
    np.testing.assert_array_equal(after[keep], states[keep])
    R.assert_close(after[[slots[b] for b in live]], *ref["final"], n * (12 + 12 * most) + 40,
                   "float32", "states")


def test_scan_in_pieces_is_the_scan():
    """A row cut into prompts that hand their state on, then single tokens: all one row."""
    case = (2, 61, 48, 16, 1, None, False)
    v, _ = scan_inputs(case, "float32", True, True, 5)
    ref, _, most = R.scan(**v)
    state = D.zeros((2, 48, 16), np.float32)
    flat = {k: R.to_device(v[k]) for k in ("A", "Dskip", "bias")}
    got = []
    for a, b in ((0, 1), (1, 38), (38, 57)):
        p = {k: R.to_device(v[k][:, a:b]) for k in ("x", "delta", "B", "C", "z")}
        got.append(R.values(S.selective_scan(
            p["x"], p["delta"], flat["A"], p["B"], p["C"], D=flat["Dskip"], z=p["z"],
            delta_bias=flat["bias"], initial_state=state, final_state=state).out))
    for t in range(57, 61):
        p = {k: R.to_device(v[k][:, t]) for k in ("x", "delta", "B", "C", "z")}
        got.append(R.values(S.selective_scan_step(
            state, p["x"], p["delta"], flat["A"], p["B"], p["C"], D=flat["Dskip"], z=p["z"],
            delta_bias=flat["bias"]).out)[:, None])
    steps = 61 * (12 + 12 * most) + 56
    R.assert_close(np.concatenate(got, 1), *ref["out"], steps, "float32", "out")
    R.assert_close(R.values(state), *ref["final"], steps, "float32", "state")


def test_scan_of_extreme_steps():
    """Steps so large that the state is forgotten, so small that it stays, and inputs outside a
    real row that are infinite."""
    batch, n, dim, state = 1, 40, 8, 16
    case = (batch, n, dim, state, 1, [33], True)
    v, _ = scan_inputs(case, "float32", True, True, 9)
    v["delta"][0, :8] = 90.0
    v["delta"][0, 8:20] = -60.0
    v["x"][0, 33:] = np.inf
    ref, _, most = R.scan(**v, n_real=[33])
    args, named, init = scan_call(v, "float32", [33], 8)
    got = S.selective_scan(*args, **named, initial_state=init, final_state=True)
    # exp(s A) with |s A| over 87 is 0 here and under 1e-38 there
    R.assert_close(R.values(got.out), *ref["out"], n * 600 + 60, "float32", "out", more=1e-30)
    R.assert_close(R.values(got.final_state), *ref["final"], n * 600 + 60, "float32", "final",
                   more=1e-30)


def test_streams():
    """Calls enqueue on the current stream: the same results on a stream of its own."""
    v, _ = scan_inputs((2, 200, 64, 16, 1, None, True), "bfloat16", True, True, 3)
    args, named, init = scan_call(v, "bfloat16", None, 8)
    want = S.selective_scan(*args, **named, initial_state=init).out.numpy()
    D.synchronize()
    side = D.Stream()
    with D.use_stream(side):
        got = S.selective_scan(*args, **named, initial_state=init).out
    side.synchronize()
    assert got.numpy().tobytes() == want.tobytes()
    with D.use_stream(D.Stream.external(side.handle)):
        got = S.selective_scan(*args, **named, initial_state=init).out.numpy()
    assert got.tobytes() == want.tobytes()
