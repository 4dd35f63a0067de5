"""A trained sequence head on a spiking front end.

Events of two classes (a pattern that moves left or right) run through one quantised spiking conv
layer; its output spikes are counted in time bins, and a head of the sequence operators reads the
rows of counts: root-mean-square norm, short causal convolution, selective scan, and a readout of
the last bin.  The head is trained with the operators' gradients, then run again as a server would:
a prompt of the first bins, the other bins one at a time on pools of states.  The small matrix
products between the operators are numpy's; everything else is one call of the library each.

    python examples/sequence_head.py
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import salt_b200 as S  # noqa: E402
from salt_b200 import device as D  # noqa: E402
from salt_b200 import sequence as Q  # noqa: E402

SIDE, BINS, MS = 12, 24, 10       # the input's plane, bins of a row, milliseconds of a bin
DIM, STATE, TAPS = 32, 16, 4      # the head's channels, states of a channel, taps
F = np.float32


def events(rng, n):
    """A bar that moves right (class 1) or left (class 0) in 2 to BINS bins, with noise."""
    rows, label, length = [], rng.integers(0, 2, n), rng.integers(2, BINS + 1, n)
    for k in range(n):
        t, s = [], []
        for b in range(length[k]):
            at = b * SIDE // BINS
            at = at if label[k] else SIDE - 1 - at
            for y in rng.integers(0, SIDE, 12):
                t.append(b * MS + rng.integers(0, MS))
                s.append(y * SIDE + (at if rng.random() < 0.8 else rng.integers(0, SIDE)))
        order = np.argsort(t, kind="stable")
        rows.append((np.array(t)[order], np.array(s)[order]))
    most = max(len(t) for t, _ in rows)
    times, src = np.zeros((n, most), F), np.zeros((n, most), np.int32)
    for k, (t, s) in enumerate(rows):
        times[k, :len(t)], src[k, :len(t)] = t, s
    return S.InputEvents(times, src, np.array([len(t) for t, _ in rows], np.int32)), label, length


def front_end(rng):
    net = S.Network.build((1, SIDE, SIDE), [S.conv(4, k=3, s=2, p=1, init_k=1.0, tau=20.0,
                                                   max_queue_len=600, max_out_spikes=4000)])
    layer = net.layers[0]
    q = rng.integers(10, 60, layer.weight_shape).astype(np.int32)
    params = [S.QuantizedLayerParams(q=q, decay_table_int=S.build_decay_table_int(10, 20.0),
                                     v_th_int=np.full(layer.n_neurons, 80, np.int32), scale=1.0,
                                     f_a=10, f_V=0, i_V=24, overflow_mode="wrap")]
    return net, params


def binned(net, params, raw, length):
    """(n, BINS, neurons) counts of the front end's spikes; rows end at `length` bins."""
    stream = net.apply_batched(params, raw, keep_streams=True).streams[0]
    n, neurons = len(length), net.layers[0].n_neurons
    counts = np.zeros((n, BINS, neurons), F)
    for k in range(n):
        real = min(int(stream.n_real_events[k]), stream.event_times.shape[1])
        b = np.minimum(stream.event_times[k, :real].astype(int) // MS, BINS - 1)
        np.add.at(counts[k], (b, stream.event_source_idx[k, :real]), 1)
    return counts


class Head:
    """Weights on the host (they take the steps), the operators' arrays on the device."""

    def __init__(self, rng, neurons):
        g = lambda *shape, s: rng.normal(0, s, shape).astype(F)  # noqa: E731
        self.w = {
            "norm": np.ones(neurons, F), "into": g(neurons, 2 * DIM, s=neurons ** -0.5),
            "conv": g(DIM, TAPS, s=0.5), "conv_bias": np.zeros(DIM, F),
            "steps": g(DIM, DIM, s=0.1), "maps": g(DIM, 2 * STATE, s=DIM ** -0.5),
            "A": -np.tile(np.arange(1, STATE + 1, dtype=F), (DIM, 1)), "D": np.ones(DIM, F),
            "step_bias": np.full(DIM, -3.0, F), "out": g(DIM, 2, s=DIM ** -0.5)}

    def _d(self, *names):
        return [D.to_device(self.w[k], F) for k in names]

    def _inputs(self, u):
        """delta, B and C of convolved rows u (..., DIM)."""
        both = (u @ self.w["maps"])[..., None, :]
        return u @ self.w["steps"], both[..., :STATE], both[..., STATE:]

    def forward(self, counts, length, train=False):
        """Logits of each row's last bin; with train, what the backward pass needs."""
        dev = lambda a: D.to_device(a, F)  # noqa: E731
        n_real = D.to_device(length, np.int32)
        norm = Q.rms_norm(dev(counts), *self._d("norm"), rstd=True)
        xz = norm.out.numpy() @ self.w["into"]
        x, z = dev(xz[..., :DIM]), dev(xz[..., DIM:])
        u = Q.causal_conv(x, *self._d("conv", "conv_bias"), n_real=n_real).out
        delta, B, C = (dev(v) for v in self._inputs(u.numpy()))
        A, Dskip, bias = self._d("A", "D", "step_bias")
        scan = Q.selective_scan(u, delta, A, B, C, D=Dskip, z=z, delta_bias=bias, n_real=n_real,
                                final_state=True, checkpoints=train)
        last = scan.out.numpy()[np.arange(len(length)), length - 1]
        logits = last @ self.w["out"]
        return (logits, (norm, x, z, u, delta, A, B, C, Dskip, bias, n_real, scan, last)) \
            if train else logits

    def step(self, counts, length, label, rate):
        """One step of gradient descent on the cross entropy; the loss before it."""
        logits, (norm, x, z, u, delta, A, B, C, Dskip, bias, n_real, scan, last) = self.forward(
            counts, length, train=True)
        p = np.exp(logits - logits.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        rows = np.arange(len(label))
        loss = -np.mean(np.log(p[rows, label]))
        p[rows, label] -= 1
        p /= len(label)
        grad = {"out": last.T @ p}
        dy = np.zeros(scan.out.shape, F)
        dy[rows, length - 1] = p @ self.w["out"].T
        g = Q.selective_scan_backward(D.to_device(dy, F), u, delta, A, B, C, D=Dskip, z=z,
                                      delta_bias=bias, n_real=n_real, checkpoints=scan.checkpoints)
        grad |= {"A": g.dA.numpy(), "D": g.dD.numpy(), "step_bias": g.ddelta_bias.numpy()}
        # through the products that made delta, B and C from u
        un, ddelta = u.numpy(), g.ddelta.numpy()
        dmaps = np.concatenate((g.dB.numpy(), g.dC.numpy()), -1)[..., 0, :]
        flat = lambda v: v.reshape(-1, v.shape[-1])  # noqa: E731
        grad |= {"steps": flat(un).T @ flat(ddelta), "maps": flat(un).T @ flat(dmaps)}
        du = g.dx.numpy() + ddelta @ self.w["steps"].T + dmaps @ self.w["maps"].T
        c = Q.causal_conv_backward(D.to_device(du, F), x, *self._d("conv", "conv_bias"),
                                   n_real=n_real)
        grad |= {"conv": c.dweight.numpy(), "conv_bias": c.dbias.numpy()}
        dxz = np.concatenate((c.dx.numpy(), g.dz.numpy()), -1)
        grad["into"] = flat(norm.out.numpy()).T @ flat(dxz)
        dn = Q.rms_norm_backward(D.to_device(dxz @ self.w["into"].T, F), D.to_device(counts, F),
                                 *self._d("norm"), norm.rstd)
        grad["norm"] = dn.dweight.numpy()
        for k, v in grad.items():
            self.w[k] = (self.w[k] - rate * np.clip(v, -1, 1)).astype(F)
        self.w["A"] = np.minimum(self.w["A"], -1e-2)
        return float(loss)

    def serve(self, counts, prompt):
        """The scan's outputs of whole rows: `prompt` bins at once, then one bin after the other.
        The states lie in pools, request k in slot n - 1 - k, as a server hands them out."""
        n = counts.shape[0]
        order = np.arange(n - 1, -1, -1).astype(np.int32)
        dev = lambda a: D.to_device(np.ascontiguousarray(a), F)  # noqa: E731
        slots = D.to_device(order, np.int32)
        conv_w, conv_b, A, Dskip, bias, norm_w = self._d("conv", "conv_bias", "A", "D",
                                                         "step_bias", "norm")
        outs = []
        xz = Q.rms_norm(dev(counts[:, :prompt]), norm_w).out.numpy() @ self.w["into"]
        conv = Q.causal_conv(dev(xz[..., :DIM]), conv_w, conv_b, final_state=True)
        delta, B, C = (dev(v) for v in self._inputs(conv.out.numpy()))
        scan = Q.selective_scan(conv.out, delta, A, B, C, D=Dskip, z=dev(xz[..., DIM:]),
                                delta_bias=bias, final_state=True)
        outs.append(scan.out.numpy())
        conv_pool, scan_pool = dev(conv.final_state.numpy()[order]), dev(
            scan.final_state.numpy()[order])
        for t in range(prompt, counts.shape[1]):
            xz = Q.rms_norm(dev(counts[:, t]), norm_w).out.numpy() @ self.w["into"]
            u = Q.causal_conv_step(dev(xz[:, :DIM]), conv_pool, conv_w, conv_b, slots=slots).out
            delta, B, C = (dev(v) for v in self._inputs(u.numpy()))
            y = Q.selective_scan_step(scan_pool, u, delta, A, B, C, D=Dskip, z=dev(xz[:, DIM:]),
                                      delta_bias=bias, slots=slots).out
            outs.append(y.numpy()[:, None])
        return np.concatenate(outs, 1)


def main(rows=96, steps=60, rate=0.5, seed=0):
    rng = np.random.default_rng(seed)
    net, params = front_end(rng)
    raw, label, length = events(rng, rows)
    counts = binned(net, params, raw, length)
    head = Head(rng, counts.shape[2])
    losses = [head.step(counts, length, label, rate) for _ in range(steps)]
    hit = np.mean(head.forward(counts, length).argmax(1) == label)
    full = np.full(rows, BINS, np.int32)
    whole = head.forward(counts, full, train=True)[1][11].out.numpy()
    served = head.serve(counts, BINS // 2)
    q8 = Q.rms_norm_q8(D.to_device(whole, F), D.to_device(np.ones(DIM), F), group=32)
    normed = Q.rms_norm(D.to_device(whole, F), D.to_device(np.ones(DIM), F)).out.numpy()
    scaled = D.from_float8_e4m3(q8.out.numpy()) * q8.scale.numpy()
    result = {"losses": losses, "hit": float(hit),
              "served": float(np.max(np.abs(served - whole))), "largest": float(np.abs(whole).max()),
              "in_8_bits": float(np.max(np.abs(scaled - normed) / np.abs(normed).max()))}
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {steps} steps, {hit:.0%} of the rows right; "
          f"served bin by bin within {result['served']:.1e} of {result['largest']:.1f}; "
          f"the readout's norm in 8 bits within {result['in_8_bits']:.1e}")
    return result


if __name__ == "__main__":
    main()
