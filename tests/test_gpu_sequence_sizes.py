"""The sequence operators where one block or thread has several rounds of work: rows past the first of
a block, runs of 8 to 32 tokens, several rows' states on their way, chunks of rows at every shape of
states, more blocks than the GPU holds, and calls with a workspace replayed from a graph.  Tolerances
as in test_gpu_sequence; where the definition would take long it is compared on a sample, and the
rest with calls small enough for one round."""
import numpy as np
import pytest

import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu


def i32(a):
    return D.to_device(np.asarray(a), np.int32)


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
@pytest.mark.parametrize("rows, dim", [(6001, 64), (5003, 250), (1501, 1100), (901, 2500), (701, 5120),
                                       (331, 16383)])
def test_norm_of_many_rows(kind, rows, dim):
    """Blocks go on to further rows, with the next one on its way; the residual in place."""
    rng = np.random.default_rng(rows)
    x, res = (R.rounded(s * rng.normal(size=(rows, dim)), kind) for s in (1, 2))
    w = R.rounded(1 + 0.3 * rng.normal(size=dim), kind)
    r, rstd, y = R.norm(x, w, res, 1e-5)
    dres, dx, dw = R.to_device(res, kind), R.to_device(x, kind), R.to_device(w, kind)
    got = S.rms_norm(dx, dw, residual=dres, residual_out=dres, rstd=True, out=dx)
    R.assert_close(R.values(dres), r, np.abs(x) + np.abs(res), 1, kind, "residual")
    R.assert_close(R.values(got.rstd), rstd, rstd, dim + 20, "float32", "rstd")
    mag = (np.abs(x) + np.abs(res)) * rstd[:, None] * np.abs(w)
    R.assert_close(R.values(dx), y, mag, dim + 20, kind, "out")


@pytest.mark.parametrize("rows, dim, group", [(6001, 72, 32), (1501, 1100, 128), (901, 4104, 0)])
def test_norm_in_8_bits_of_many_rows(rows, dim, group):
    """The same bits as row by row in calls of their own."""
    rng = np.random.default_rng(rows)
    x, w = rng.normal(size=(rows, dim)).astype(np.float32), R.to_device(rng.normal(size=dim))
    res = rng.normal(size=(rows, dim)).astype(np.float32)
    dres = R.to_device(res)
    all_ = S.rms_norm_q8(R.to_device(x), w, residual=dres, residual_out=dres, group=group)
    np.testing.assert_array_equal(dres.numpy(), x + res)
    for at in range(0, rows, 300):  # few enough for a block, or a warp, each
        cut = slice(at, at + 300)
        some = S.rms_norm_q8(R.to_device(x[cut]), w, residual=R.to_device(res[cut]), group=group)
        np.testing.assert_array_equal(R.values(all_.out)[cut], R.values(some.out))
        np.testing.assert_array_equal(all_.scale.numpy()[cut], some.scale.numpy())


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
@pytest.mark.parametrize("batch, n, dim, width", [
    (4, 300, 4096, 4), (2, 640, 8192, 3), (4, 640, 8192, 4), (1, 100, 8190, 8), (3, 200, 4099, 2),
    (2, 500, 8193, 6)])
def test_conv_of_long_runs(kind, batch, n, dim, width):
    """Threads of 8, 16 and 32 tokens, whose window goes on from token to token; ragged rows.  64
    channels are compared with the definition, the others with calls on 64 channels each (4 tokens a
    thread)."""
    rng = np.random.default_rng(n)
    x = R.rounded(rng.normal(size=(batch, n, dim)), kind)
    w, bias = R.rounded(rng.normal(size=(dim, width)), kind), R.rounded(rng.normal(size=dim), kind)
    init = R.rounded(rng.normal(size=(batch, dim, width - 1)), kind)
    n_real = [n, n - 3, 1, 0][:batch]
    got = S.causal_conv(R.to_device(x, kind), R.to_device(w, kind), R.to_device(bias, kind),
                        n_real=i32(n_real), initial_state=R.to_device(init, kind),
                        final_state=True)
    out, final = R.values(got.out), R.values(got.final_state)
    some = np.sort(rng.choice(dim, 64, replace=False))
    ref, mag, end = R.conv(x[..., some], w[some], bias[some], n_real, init[:, some])
    R.assert_close(out[..., some], ref, mag, 2 * width + 20, kind, "out")
    np.testing.assert_array_equal(final[:, some], end)
    for at in range(0, dim, 64 * 9):
        cut = slice(at, at + 64)
        few = S.causal_conv(R.to_device(x[..., cut], kind), R.to_device(w[cut], kind),
                            R.to_device(bias[cut], kind), n_real=i32(n_real),
                            initial_state=R.to_device(init[:, cut], kind), final_state=True)
        np.testing.assert_array_equal(out[..., cut], R.values(few.out))
        np.testing.assert_array_equal(final[:, cut], R.values(few.final_state))


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
@pytest.mark.parametrize("batch, dim, state, groups", [
    (250, 4096, 16, 1), (251, 4095, 12, 3), (255, 8192, 4, 2), (130, 4100, 7, 1), (249, 2048, 64, 1)])
def test_scan_step_of_many_rows(kind, batch, dim, state, groups):
    """Blocks walk over several rows with the states of the next ones on their way; rows without a
    slot lie between the others, and the last block has fewer rows."""
    rng = np.random.default_rng(batch)
    pool = batch + 5
    slots = rng.permutation(pool)[:batch].astype(np.int32)
    empty = rng.random(batch) < 0.2
    empty[[1, batch - 1]] = True, False
    slots[empty] = rng.choice([-1, pool, pool + 7], empty.sum())
    x, delta, z = (R.rounded(rng.normal(size=(batch, dim)), kind) for _ in range(3))
    B, C = (R.rounded(rng.normal(size=(batch, groups, state)), kind) for _ in range(2))
    A = R.rounded(-rng.uniform(0.5, 1.5, (dim, state)), "float32")
    skip, bias = (R.rounded(rng.normal(size=dim), "float32") for _ in range(2))
    states = rng.normal(size=(pool, dim, state)).astype(np.float32)
    dev = R.to_device(states)
    out = S.selective_scan_step(
        dev, *(R.to_device(v, kind) for v in (x, delta)), R.to_device(A),
        *(R.to_device(v, kind) for v in (B, C)), D=R.to_device(skip), z=R.to_device(z, kind),
        delta_bias=R.to_device(bias), slots=i32(slots)).out
    y, after = R.values(out), dev.numpy()
    live = np.flatnonzero(~empty)
    assert not np.any(y[empty])
    others = np.setdiff1d(np.arange(pool), slots[live])
    np.testing.assert_array_equal(after[others], states[others])
    one = lambda v: v[live][:, None]  # noqa: E731
    ref, _, most = R.scan(one(x), one(delta), A, one(B), one(C), skip, one(z), bias,
                          init=states[slots[live]].astype(np.float64))
    steps = 12 + 12 * most + state + 40
    R.assert_close(y[live], ref["out"][0][:, 0], ref["out"][1][:, 0], steps, kind, "out")
    R.assert_close(after[slots[live]].astype(np.float64), *ref["final"], steps, "float32", "states")


def scan_inputs(rng, batch, n, dim, state, groups, kind):
    v = {"x": rng.normal(size=(batch, n, dim)), "delta": 0.7 * rng.normal(size=(batch, n, dim)),
         "B": rng.normal(size=(batch, n, groups, state)),
         "C": rng.normal(size=(batch, n, groups, state)), "z": rng.normal(size=(batch, n, dim)),
         "dy": rng.normal(size=(batch, n, dim))}
    v = {k: R.rounded(a, kind) for k, a in v.items()}
    f = {"A": -rng.uniform(0.5, 1.5, (dim, state)), "Dskip": rng.normal(size=dim),
         "bias": rng.uniform(-4, -1, dim), "init": rng.normal(size=(batch, dim, state)),
         "dfinal": rng.normal(size=(batch, dim, state))}
    return v, {k: R.rounded(a, "float32") for k, a in f.items()}


def run_scan(v, f, kind, n_real, groups=slice(None), channels=slice(None)):
    """Forward and backward over a choice of groups and their channels: {name: values}."""
    a = {k: R.to_device(v[k][:, :, groups] if k in "BC" else v[k][..., channels], kind) for k in v}
    w = {k: R.to_device(f[k][:, channels] if f[k].ndim == 3 else f[k][channels]) for k in f}
    named = dict(D=w["Dskip"], z=a["z"], delta_bias=w["bias"], n_real=i32(n_real))
    args = (a["x"], a["delta"], w["A"], a["B"], a["C"])
    o = S.selective_scan(*args, **named, initial_state=w["init"], final_state=True,
                         checkpoints=True)
    g = S.selective_scan_backward(a["dy"], *args, **named, checkpoints=o.checkpoints,
                                  dfinal=w["dfinal"], dinitial=True)
    return {"out": R.values(o.out), "final": R.values(o.final_state)} | {
        k: R.values(t) for k, t in g._asdict().items()}


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
@pytest.mark.parametrize("batch, n, dim, state, n_real", [
    (2, 700, 16, 8, [700, 333]), (2, 523, 40, 24, [260, 523]), (1, 600, 12, 32, [600]),
    (2, 500, 70, 12, [0, 499]), (1, 450, 36, 40, [257])])
def test_scan_in_chunks(kind, batch, n, dim, state, n_real):
    """Rows cut into chunks at the shapes of states that test_gpu_sequence leaves whole."""
    rng = np.random.default_rng(n + state)
    v, f = scan_inputs(rng, batch, n, dim, state, 1, kind)
    got = run_scan(v, f, kind, n_real)
    ins = {k: v[k] for k in ("x", "delta", "B", "C", "z")} | {k: f[k] for k in
                                                              ("A", "Dskip", "bias", "init")}
    ref, _, most = R.scan(**ins, n_real=n_real)
    back, _ = R.scan_backward(v["dy"], **ins, n_real=n_real, dfinal=f["dfinal"])
    steps = n * (12 + 12 * most) + state + 40
    R.assert_close(got["out"], *ref["out"], steps, kind, "out")
    R.assert_close(got["final"], *ref["final"], steps, "float32", "final")
    for k, (value, mag) in back.items():
        kept = "float32" if k in ("dA", "dD", "ddelta_bias", "dinitial") else kind
        R.assert_close(got[k], value, mag, 2 * steps + dim + batch * n, kept, k)


@pytest.mark.parametrize("state, dim", [(4, 32768), (8, 16384), (16, 8192), (32, 8192), (64, 4096)])
def test_scan_of_more_blocks_than_the_gpu_holds(state, dim):
    """Several rounds of blocks, groups of 1024 channels: the same bits as the same rows with one group
    alone (none of them is cut into chunks), and dB and dC in the group's place."""
    rng = np.random.default_rng(state)
    batch, n, groups = 6, 70, dim // 1024
    n_real = [70, 1, 0, 33, 64, 70]
    v, f = scan_inputs(rng, batch, n, dim, state, groups, "float32")
    got = run_scan(v, f, "float32", n_real)
    for g in (0, groups - 1):
        cut = slice(g * 1024, (g + 1) * 1024)
        some = run_scan(v, f, "float32", n_real, slice(g, g + 1), cut)
        for k, value in some.items():
            if k in ("dB", "dC"):
                part = got[k][:, :, g:g + 1]
            elif k in ("dA", "dD", "ddelta_bias"):
                part = got[k][cut]
            else:
                part = got[k][:, cut] if k in ("final", "dinitial") else got[k][..., cut]
            np.testing.assert_array_equal(part, value, err_msg=k)


def test_calls_with_a_workspace_replay_as_a_graph():
    """A training step's operators on new inputs: replayed as called."""
    rng = np.random.default_rng(4)
    batch, n, dim, state, width = 2, 400, 48, 16, 4
    f = lambda *s: rng.normal(size=s).astype(np.float32)  # noqa: E731
    A, w, conv_w = (R.to_device(a) for a in (-np.abs(f(dim, state)) - 0.1, f(dim), f(dim, width)))
    tokens = [[f(batch, n, dim), f(batch, n, dim), f(batch, n, 1, state), f(batch, n, 1, state)]
              for _ in range(3)]

    def run(recorded):
        e = lambda *s: D.zeros(s, np.float32)  # noqa: E731
        x, delta, B, C = e(batch, n, dim), e(batch, n, dim), e(batch, n, 1, state), e(batch, n, 1, state)
        out, marks = e(batch, n, dim), e(batch, n // 16, dim, state)
        o = {k: e(batch, n, dim) for k in ("dx", "ddelta")}
        o |= {"dA": e(dim, state), "dB": e(batch, n, 1, state), "dC": e(batch, n, 1, state)}
        c = {"dx": e(batch, n, dim), "dweight": e(dim, width)}
        m = {"dx": e(batch, n, dim), "dweight": e(dim)}
        rstd = R.to_device(np.ones((batch, n)))

        def step():
            S.selective_scan(x, delta, A, B, C, out=out, checkpoints=marks)
            S.selective_scan_backward(out, x, delta, A, B, C, checkpoints=marks, **o)
            S.causal_conv_backward(o["dx"], x, conv_w, **c)
            S.rms_norm_backward(c["dx"], x, w, rstd, **m)

        stream = D.Stream()
        D.synchronize()
        got = []
        with D.use_stream(stream):
            if recorded:
                with D.Graph.capture(stream) as graph:
                    step()
            for token in tokens:
                for to, a in zip((x, delta, B, C), token):
                    to.copy_from(a, sync=True)
                graph.replay(stream) if recorded else step()
                got.append([a.numpy() for a in (out, *o.values(), *c.values(), *m.values())])
        return got

    for a, b in zip(run(False), run(True)):
        for p, q in zip(a, b):
            np.testing.assert_array_equal(p, q)
