"""Linear attention and the products in 8 bits as a block uses them together: norm to 8 bits, projection,
attention over prompts and then token by token, norm to 8 bits, projection; recorded as graphs, on other
streams, and from another library's arrays.  Each stage is held to its definition on the values that the
stage before left on the device, with that stage's own tolerance (test_gpu_linear_attention.py,
test_gpu_products_8bit.py)."""
import numpy as np
import pytest

import _attention_ref as A
import _sequence_ref as R
import salt_b200 as S
from salt_b200 import device as D

pytestmark = pytest.mark.gpu

KIND, DIM, HEADS, KV, HEAD = "bfloat16", 384, 4, 2, 64
CUT = (HEADS * HEAD, KV * HEAD, KV * HEAD)


class Part:
    """Columns of an array's last axis as (heads, dim)."""

    def __init__(self, a, at, heads, dim):
        self.array, self.dtype = a, a.dtype
        self.shape = a.shape[:-1] + (heads, dim)
        self._at = a.data_ptr() + at * a.dtype.itemsize

    def data_ptr(self):
        return self._at

    def stride(self):
        return self.array.stride()[:-1] + (self.shape[-1], 1)


class Block:
    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        self.norm = [R.to_device(1 + 0.1 * rng.normal(size=DIM if i == 0 else HEADS * HEAD), KIND)
                     for i in range(2)]
        shapes = (sum(CUT), DIM), (DIM, HEADS * HEAD)
        self.weights = [S.quantize_q8(R.to_device(rng.normal(size=s) * s[1] ** -0.5, KIND),
                                      blocks=True) for s in shapes]
        self.log_decay = np.log1p(-(2.0 ** -np.arange(1, HEADS + 1))).astype(np.float32)
        self.decay = R.to_device(self.log_decay)

    def project(self, x, i, out):
        n = S.rms_norm_q8(x, self.norm[i])
        w = self.weights[i]
        S.matmul_q8(n.out, n.scale, w.out, w.scale, out=out)
        return n

    def __call__(self, x, keep, attend):
        lead = x.shape[:-1]
        keep["qkv"] = D.empty(lead + (sum(CUT),), D.bfloat16)
        keep["n0"] = self.project(x, 0, keep["qkv"])
        parts, at = [], 0
        for width, heads in zip(CUT, (HEADS, KV, KV)):
            parts.append(Part(keep["qkv"], at, heads, HEAD))
            at += width
        keep["mixed"] = attend(*parts)
        flat = D.DeviceArray(keep["mixed"].data_ptr(), lead + (HEADS * HEAD,), D.bfloat16,
                             keep["mixed"])
        keep["y"] = D.empty(lead + (DIM,), D.bfloat16)
        keep["n1"] = self.project(flat, 1, keep["y"])
        return keep["y"]

    def check_projections(self, keep):
        for i, name in ((0, "qkv"), (1, "y")):
            n, w = keep[f"n{i}"], self.weights[i]
            x, wv = R.values(n.out), R.values(w.out)
            x, scale = x.reshape(-1, x.shape[-1]), n.scale.numpy()
            want, mag = A.product(x, scale.reshape(len(x), -1), wv, w.scale.numpy())
            got = R.values(keep[name]).reshape(want.shape)
            R.assert_close(got, want, mag, 24 + scale.shape[-1], KIND, name)


def split(qkv):
    at = np.cumsum((0,) + CUT)
    return [qkv[..., at[i]:at[i + 1]].reshape(qkv.shape[:-1] + (h, HEAD))
            for i, h in enumerate((HEADS, KV, KV))]


def test_a_block_on_prompts_and_then_on_tokens():
    rng, block = np.random.default_rng(0), Block(1)
    batch, n, scale = 3, 150, HEAD ** -0.5
    real = [150, 0, 77]
    lengths = D.to_device(np.asarray(real), np.int32)
    x = R.to_device(rng.normal(size=(batch, n, DIM)), KIND)
    pool = D.zeros((batch + 1, HEADS, HEAD, HEAD), np.float32)
    keep = {}

    def prompt(q, k, v):
        return S.linear_attention(q, k, v, block.decay, scale=scale, n_real=lengths,
                                  final_state=pool[1:]).out

    block(x, keep, prompt)
    block.check_projections(keep)
    want = A.attention(*split(R.values(keep["qkv"])), block.log_decay, scale, real)
    R.assert_close(R.values(keep["mixed"]), want[0], want[1], 200 + 512 + n / 8, KIND, "attention")
    state = R.values(pool[1:])
    R.assert_close(state, want[2], want[3], 200 + n / 8, "float32", "state")
    slots = D.to_device(np.array([1, 2, 3]), np.int32)
    for t in range(3):
        x = R.to_device(rng.normal(size=(batch, DIM)), KIND)
        keep = {}
        block(x, keep, lambda q, k, v: S.linear_attention_step(
            pool, q, k, v, block.decay, scale=scale, slots=slots).out)
        block.check_projections(keep)
        want = A.attention(*split(R.values(keep["qkv"])[:, None]), block.log_decay, scale,
                           init=state)
        R.assert_close(R.values(keep["mixed"]), want[0][:, 0], want[1][:, 0], HEAD + 20, KIND,
                       f"token {t}")
        state = R.values(pool[1:])
        R.assert_close(state, want[2], want[3], 12, "float32", f"state {t}")
    assert np.all(R.values(pool[:1]) == 0)


def test_calls_replay_as_graphs_that_share_their_inputs():
    """Two recordings, each with workspaces of its own (split rows, shared key heads, planes), replayed
    one after the other and again on new inputs: the same bits as the calls themselves."""
    rng = np.random.default_rng(2)
    batch, n, heads, kv, dk, dv = 1, 700, 2, 1, 33, 50
    f = lambda *s: rng.normal(size=s).astype(np.float32)  # noqa: E731
    shapes = {"q": (batch, n, heads, dk), "k": (batch, n, kv, dk), "v": (batch, n, kv, dv),
              "d": (batch, n, heads, dv), "x": (30, 130), "w": (20, 130)}
    decay = R.to_device([-0.01, -0.3])
    inputs = [{name: f(*s) for name, s in shapes.items()} for _ in range(3)]

    def outputs():
        e = lambda *s: D.zeros(s, np.float32)  # noqa: E731
        return {"out": e(*shapes["d"]), "final": e(batch, heads, dk, dv), "dq": e(*shapes["q"]),
                "dk": e(*shapes["k"]), "dv": e(*shapes["v"]), "y": e(30, 20)}

    def forward(a, o):
        S.linear_attention(a["q"], a["k"], a["v"], decay, out=o["out"], final_state=o["final"])

    def backward(a, o):
        S.linear_attention_backward(a["d"], a["q"], a["k"], a["v"], decay, dq=o["dq"], dk=o["dk"],
                                    dv=o["dv"])
        x, w = S.quantize_q8(a["x"]), S.quantize_q8(a["w"], blocks=True)
        S.matmul_q8(x.out, x.scale, w.out, w.scale, out=o["y"])

    def run(recorded):
        arrays, o = {k: D.zeros(s, np.float32) for k, s in shapes.items()}, outputs()
        stream, results = D.Stream(), []
        D.synchronize()
        with D.use_stream(stream):
            graphs = []
            if recorded:
                for part in (forward, backward):
                    with D.Graph.capture(stream) as g:
                        part(arrays, o)
                    graphs.append(g)
            for values in inputs:
                for name, v in values.items():
                    arrays[name].copy_from(v, sync=True)
                for i, part in enumerate((forward, backward)):
                    graphs[i].replay(stream) if recorded else part(arrays, o)
                results.append({k: v.numpy() for k, v in o.items()})
        return results

    for a, b in zip(run(False), run(True)):
        for name in a:
            np.testing.assert_array_equal(a[name], b[name], err_msg=name)


def test_calls_on_two_streams_at_once():
    """The same work on two streams, each with its own outputs: the same bits."""
    rng = np.random.default_rng(3)
    q, k, v = (R.to_device(rng.normal(size=(2, 900, 2, 64)), KIND) for _ in range(3))
    decay = R.to_device([-0.02, -0.5])
    x, w = S.quantize_q8(R.to_device(rng.normal(size=(300, 512)), KIND)), S.quantize_q8(
        R.to_device(rng.normal(size=(400, 512)), KIND), blocks=True)
    D.synchronize()
    streams, got = [D.Stream(), D.Stream()], []
    for _ in range(4):
        for stream in streams:
            with D.use_stream(stream):
                a = S.linear_attention(q, k, v, decay, final_state=True)
                y = S.matmul_q8(x.out, x.scale, w.out, w.scale)
                got.append((a.out, a.final_state, y))
    D.synchronize()
    first = [R.values(a) for a in got[0]]
    for other in got[1:]:
        for a, b in zip(first, other):
            np.testing.assert_array_equal(a, R.values(b))


def test_another_librarys_arrays():
    """Transposed, sliced and broadcast views of torch tensors, on its stream."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(4)
    batch, n, heads, dim = 2, 70, 3, 32
    qkv = torch.from_numpy(rng.normal(size=(n, batch, 3, heads, dim)).astype(np.float32)).cuda()
    q, k, v = (qkv[:, :, i].transpose(0, 1) for i in range(3))  # token-major memory
    decay = torch.full((heads,), -0.1, device="cuda")
    torch.cuda.synchronize()
    got = S.linear_attention(q, k, v, decay, final_state=True)
    want = A.attention(*(t.cpu().numpy().astype(np.float64) for t in (q, k, v)),
                       decay.cpu().numpy(), 1.0)
    R.assert_close(R.values(got.out), want[0], want[1], 200 + n / 8, "float32", "out")
    # one row of keys and values for the whole batch: a batch stride of zero
    k1, v1 = (t[:1].expand(batch, -1, -1, -1) for t in (k, v))
    got = S.linear_attention(q, k1, v1, decay)
    want = A.attention(*(t.cpu().numpy().astype(np.float64) for t in (q, k1, v1)),
                       decay.cpu().numpy(), 1.0)
    R.assert_close(R.values(got.out), want[0], want[1], 200 + n / 8, "float32", "broadcast")
    x = torch.from_numpy(rng.normal(size=(40, 300)).astype(np.float32)).cuda()
    a = S.quantize_q8(x[:, 4:260])
    w = S.quantize_q8(x[:, :256], blocks=True)
    torch.cuda.synchronize()
    y = S.matmul_q8(a.out, a.scale, w.out, w.scale, dtype=np.float32)
    want, mag = A.product(R.values(a.out), a.scale.numpy(), R.values(w.out), w.scale.numpy())
    R.assert_close(R.values(y), want, mag, 26, "float32", "product")


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
def test_rows_of_many_tokens_keep_their_precision(kind):
    """No decay over thousands of tokens: the state's error grows with the chunks, not the tokens."""
    rng = np.random.default_rng(5)
    n = 6000
    q, k, v = (R.rounded(rng.normal(size=(1, n, 1, 16)), kind) for _ in range(3))
    want = A.attention(q, k, v, [0.0], 1.0)
    got = S.linear_attention(*(R.to_device(a, kind) for a in (q, k, v)), R.to_device([0.0]),
                             final_state=True)
    R.assert_close(R.values(got.final_state), want[2], want[3], 200 + n / 64, "float32", "state")
    R.assert_close(R.values(got.out), want[0], want[1],
                   200 + n / 64 + (0 if kind == "float32" else 512), kind, "out")
