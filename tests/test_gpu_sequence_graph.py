"""Single-token operators recorded as one CUDA graph and replayed: the same states and outputs as
the calls themselves, token after token."""
import numpy as np
import pytest

import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu


def test_steps_replay_as_a_graph():
    rng = np.random.default_rng(0)
    batch, dim, state, width = 3, 40, 16, 4
    f = lambda *shape: rng.normal(size=shape).astype(np.float32)  # noqa: E731
    norm_w, conv_w, conv_b = (R.to_device(v) for v in (f(dim), f(dim, width), f(dim)))
    A, Dskip, bias = (R.to_device(v) for v in (-np.abs(f(dim, state)) - 0.1, f(dim), f(dim)))
    tokens = [(f(batch, dim), f(batch, dim), f(batch, 1, state), f(batch, 1, state))
              for _ in range(4)]

    def run(recorded):
        x, delta = D.zeros((batch, dim), np.float32), D.zeros((batch, dim), np.float32)
        B, C = (D.zeros((batch, 1, state), np.float32) for _ in range(2))
        normed, mixed, out = (D.zeros((batch, dim), np.float32) for _ in range(3))
        conv, pool = D.zeros((batch, dim, width - 1), np.float32), D.zeros((batch, dim, state),
                                                                           np.float32)

        def step():
            S.rms_norm(x, norm_w, out=normed)
            S.causal_conv_step(normed, conv, conv_w, conv_b, out=mixed)
            S.selective_scan_step(pool, mixed, delta, A, B, C, D=Dskip, delta_bias=bias, out=out)

        stream = D.Stream()
        D.synchronize()
        with D.use_stream(stream):
            if recorded:
                with D.Graph.capture(stream) as graph:
                    step()
            outs = []
            for token in tokens:
                for to, v in zip((x, delta, B, C), token):
                    to.copy_from(v, sync=True)
                graph.replay(stream) if recorded else step()
                outs.append(out.numpy())
            return outs + [conv.numpy(), pool.numpy()]

    for a, b in zip(run(False), run(True)):
        np.testing.assert_array_equal(a, b)
