"""Cases that measure the sequence operators' second part: linear attention with a decay for each
head (rows, single tokens, training), the matrix product in 8 bits with a scale for every 128
values, and the quantisation that makes its operands.

``run`` computes an operator either in its plain form (elementary torch operations in 32 bits,
rounded once at the end) or, where ``own`` is true, through ``salt_b200.sequence``.  Linear
attention's plain form goes through the rows in chunks: products within a chunk under a matrix of
decays, and one state that is carried from chunk to chunk.

Layouts: q is (batch, length, heads, dim_k), k and v are (batch, length, kv heads, dim_k or dim_v),
views of one projection's output; the states are float32 (batch, heads, dim_k, dim_v).  Rows end at
``n_real`` tokens; what lies past that is not read and comes back as zero.  8-bit values are e4m3;
the value is ``q * scale`` with a float32 scale for 128 neighbours of a row or for a block of
128 x 128.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
E4M3_MAX = 448.0
GROUP = 128
CHUNK = 128


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a single request's token: all latency
        {"name": "attn_step_one", "op": "attn_step", "batch": 1, "heads": 16, "kv": 16, "dk": 64,
         "dv": 64, "type": "bf16", "pool": 1},
        # a full serving batch: reading and writing the states is the work
        {"name": "attn_step_many", "op": "attn_step", "batch": 128, "heads": 32, "kv": 8,
         "dk": 128, "dv": 128, "type": "bf16", "pool": 160},
        # one long prompt: few heads' rows, so the length has to be split
        {"name": "attn_prompt_long", "op": "attn", "batch": 1, "len": 32768, "heads": 16, "kv": 16,
         "dk": 128, "dv": 128, "type": "bf16", "ragged": False, "initial": True},
        # a batch of ragged prompts with shared key heads
        {"name": "attn_prompt_batch", "op": "attn", "batch": 8, "len": 2048, "heads": 32, "kv": 8,
         "dk": 128, "dv": 128, "type": "bf16", "ragged": True, "initial": False},
        # 32 bits and sizes that are multiples of nothing, on states of earlier chunks
        {"name": "attn_prompt_odd", "op": "attn", "batch": 3, "len": 1021, "heads": 6, "kv": 3,
         "dk": 75, "dv": 50, "type": "f32", "ragged": True, "initial": True},
        # a training step's attention, forward and backward
        {"name": "attn_train", "op": "attn_train", "batch": 8, "len": 2048, "heads": 16, "kv": 16,
         "dk": 128, "dv": 128, "type": "bf16", "ragged": False, "initial": False},
        # training with shared key heads on ragged rows, in float16
        {"name": "attn_train_odd", "op": "attn_train", "batch": 3, "len": 1021, "heads": 12,
         "kv": 4, "dk": 64, "dv": 100, "type": "f16", "ragged": True, "initial": True},
        # one decoding step's rows through a projection: reading the weight is the work
        {"name": "q8_step", "op": "q8", "rows": 16, "k": 2048, "n": 4096, "type": "bf16",
         "bias": False},
        # a large prompt batch through the projection that follows the 8-bit norm
        {"name": "q8_prompt", "op": "q8", "rows": 16384, "k": 5120, "n": 5120, "type": "bf16",
         "bias": False},
        # rows, widths and a depth that are multiples of nothing
        {"name": "q8_odd", "op": "q8", "rows": 1021, "k": 2501, "n": 1002, "type": "f16",
         "bias": True},
        # a trained weight brought to 8 bits by blocks, as it lies and transposed
        {"name": "q8_weight", "op": "q8_quant", "rows": 4096, "dim": 5120, "type": "bf16",
         "blocks": True},
        # a projection's training step: both operands' quantisation, forward and two gradients
        {"name": "q8_train", "op": "q8_train", "rows": 8192, "k": 2048, "n": 4096, "type": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def _dim(rng, low, high):
    """A width: a multiple of 128, of 8, or any number."""
    step = rng.choice((128, 8, 1))
    return max(step, _log(rng, low, high) // step * step)


def draw(rng):
    op = rng.choice(("attn", "attn", "attn_step", "attn_train", "attn_train", "q8", "q8", "q8",
                     "q8_quant", "q8_train"))
    kind = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "q8":
        rows, k = _log(rng, 1, 16384), _dim(rng, 64, 8192)
        n = _dim(rng, 64, min(8192, max(128, 16384 * 5120 * 5120 // (rows * k))))
        return {"op": op, "rows": rows, "k": k, "n": n, "type": kind,
                "bias": rng.random() < 0.5}
    if op == "q8_quant":
        dim = _dim(rng, 64, 8192)
        return {"op": op, "rows": _log(rng, 1, 4096 * 5120 // dim), "dim": dim, "type": kind,
                "blocks": rng.random() < 0.5}
    if op == "q8_train":
        k, n = _dim(rng, 64, 4096), _dim(rng, 64, 4096)
        return {"op": op, "rows": _log(rng, 1, min(8192, 8192 * 2048 * 4096 // (k * n))), "k": k,
                "n": n, "type": kind}
    kv = rng.choice((1, 2, 4, 8))
    heads = kv * rng.choice((1, 1, 2, 4))
    dk, dv = (rng.choice((32, 64, 128, 128, rng.randrange(1, 129))) for _ in range(2))
    case = {"op": op, "heads": heads, "kv": kv, "dk": dk, "dv": dv, "type": kind}
    if op == "attn_step":
        batch = _log(rng, 1, 128)
        return case | {"batch": batch, "pool": batch + rng.randrange(0, 33)}
    batch = _log(rng, 1, 16)
    most = 32768 * 16 if op == "attn" else 8 * 2048 * 16
    return case | {"batch": batch, "len": _log(rng, 1, min(32768, most // (batch * heads))),
                   "ragged": rng.random() < 0.5, "initial": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs

class _Make:
    """Inputs on the GPU from one seed."""

    def __init__(self, case, seed):
        self.type = _TYPES[case["type"]]
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, scale=1.0, type=None):
        v = torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return v.mul_(scale).to(type or self.type)

    def lengths(self, case):
        """The rows' token counts: evenly from none to all, in an order of the seed's; or None."""
        if not case["ragged"]:
            return None
        spread = torch.tensor(_real(case), device="cuda", dtype=torch.int32)
        return spread[torch.randperm(case["batch"], generator=self.gen, device="cuda")]

    def empty(self, *shape, type=None):
        return torch.empty(*shape, device="cuda", dtype=type or self.type)


def _decays(heads):
    """log of 1 - 2^-1 to 1 - 2^-10: heads that forget in a token and heads that keep thousands."""
    at = torch.linspace(1, 10, heads, dtype=torch.float64) if heads > 1 else torch.tensor([5.0])
    return torch.log1p(-torch.exp2(-at.double())).float().cuda()


def prepare(case, seed):
    m, op = _Make(case, seed), case["op"]
    s = {"op": op, "case": case}
    f32, e4m3 = torch.float32, torch.float8_e4m3fn
    if op == "q8_quant":
        rows, dim = case["rows"], case["dim"]
        s["x"], s["blocks"] = m.normal(rows, dim, scale=dim ** -0.5), case["blocks"]
        up, over = -(-rows // GROUP), -(-dim // GROUP)
        s["q"], s["qt"] = m.empty(rows, dim, type=e4m3), m.empty(dim, rows, type=e4m3)
        s["scale"] = m.empty(up if s["blocks"] else rows, over, type=f32)
        s["scale_t"] = m.empty(over if s["blocks"] else dim, up, type=f32)
        return s
    if op.startswith("q8"):
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"] = m.normal(rows, k)
        s["w"] = m.normal(n, k, scale=k ** -0.5)
        s["y"] = m.empty(rows, n)
        if op == "q8_train":
            s["dy"] = m.normal(rows, n, scale=0.1)
            s["dx"], s["dw"] = m.empty(rows, k), m.empty(n, k, type=f32)
            return s
        # what the norm wrote in 8 bits, and the weight as it was laid out once
        s["x"], s["x_scale"] = _quantized(s["x"])
        s["w"], s["w_scale"] = _quantized(s["w"], blocks=True)
        s["bias"] = m.normal(n, scale=0.1) if case["bias"] else None
        return s
    batch, heads, kv, dk, dv = (case[k] for k in ("batch", "heads", "kv", "dk", "dv"))
    s["decay"], s["scale"] = _decays(heads), dk ** -0.5
    lead = (batch,) if op == "attn_step" else (batch, case["len"])
    cut = (heads * dk, kv * dk, kv * dv)
    q, k, v = m.normal(*lead, sum(cut)).split(cut, -1)
    s["q"], s["k"] = q.unflatten(-1, (heads, dk)), k.unflatten(-1, (kv, dk))
    s["v"] = v.unflatten(-1, (kv, dv))
    s["y"] = m.empty(*lead, heads, dv)
    if op == "attn_step":
        s["state"] = m.normal(case["pool"], heads, dk, dv, type=f32)
        s["slots"] = torch.randperm(case["pool"], generator=m.gen, device="cuda")[:batch].to(
            torch.int32)
        return s
    s["n_real"] = m.lengths(case)
    s["initial"], s["final"] = None, m.empty(batch, heads, dk, dv, type=f32)
    if case["initial"]:
        s["initial"] = m.normal(batch, heads, dk, dv, type=f32)
    if op == "attn_train":
        s["dy"] = m.normal(*lead, heads, dv, scale=0.1)
        s["dq"], s["dk"] = m.empty(*lead, heads, dk), m.empty(*lead, kv, dk)
        s["dv"] = m.empty(*lead, kv, dv)
        s["dinitial"] = None
        if case["initial"]:
            s["dinitial"] = m.empty(batch, heads, dk, dv, type=f32)
    return s


def _real(case):
    batch, n = case["batch"], case["len"]
    if not case["ragged"] or batch == 1:
        return [n] * batch
    return [n * i // (batch - 1) for i in range(batch)]


# ---------------------------------------------------------------- one pass

def run(s):
    return (_OWN if own else _PLAIN)[s["op"]](s)


def work(case):
    """Each input read once and each output written once, and the operator's arithmetic: for linear
    attention that of the recurrence."""
    e, op = _BYTES[case["type"]], case["op"]
    if op == "q8_quant":
        n = case["rows"] * case["dim"]
        return {"bytes": n * (e + 2), "flops": 3 * n}
    if op.startswith("q8"):
        rows, k, n = case["rows"], case["k"], case["n"]
        scales = 4 * -(-k // GROUP) * (rows + -(-n // GROUP))
        if op == "q8":
            return {"bytes": rows * k + n * k + scales + rows * n * e + case["bias"] * n * e,
                    "flops": 2 * rows * n * k}
        return {"bytes": e * (2 * rows * k + n * k + 2 * rows * n) + 4 * n * k,
                "flops": 6 * rows * n * k}
    batch, heads, kv, dk, dv = (case[k] for k in ("batch", "heads", "kv", "dk", "dv"))
    token = heads * dk + kv * (dk + dv)
    if op == "attn_step":
        return {"bytes": batch * ((token + heads * dv) * e + 8 * heads * dk * dv),
                "flops": 5 * batch * heads * dk * dv}
    n, live = batch * case["len"], sum(_real(case))
    states = 4 * batch * heads * dk * dv * (2 if case["initial"] else 1)
    if op == "attn":
        return {"bytes": (live * token + n * heads * dv) * e + states,
                "flops": 5 * live * heads * dk * dv}
    # forward: q, k, v, y; backward adds dy and the three gradients, and dinitial
    return {"bytes": (live * (token + heads * dv) + n * (token + heads * dv)) * e + 2 * states,
            "flops": 13 * live * heads * dk * dv}


# ---------------------------------------------------------------- the framework's calls

def _sequence():
    import salt_b200.sequence as sequence
    return sequence


def _own_attn(s):
    _sequence().linear_attention(s["q"], s["k"], s["v"], s["decay"], scale=s["scale"],
                                 n_real=s["n_real"], initial_state=s["initial"], out=s["y"],
                                 final_state=s["final"])
    return s["y"], s["final"]


def _own_attn_step(s):
    _sequence().linear_attention_step(s["state"], s["q"], s["k"], s["v"], s["decay"],
                                      scale=s["scale"], slots=s["slots"], out=s["y"])
    return s["y"], s["state"]


def _own_attn_train(s):
    a = _sequence()
    a.linear_attention(s["q"], s["k"], s["v"], s["decay"], scale=s["scale"], n_real=s["n_real"],
                       initial_state=s["initial"], out=s["y"], final_state=s["final"])
    a.linear_attention_backward(s["dy"], s["q"], s["k"], s["v"], s["decay"], scale=s["scale"],
                                n_real=s["n_real"], initial_state=s["initial"], dq=s["dq"],
                                dk=s["dk"], dv=s["dv"], dinitial=s["dinitial"])
    return {k: s[k] for k in _TRAINED}


def _own_q8(s):
    return _sequence().matmul_q8(s["x"], s["x_scale"], s["w"], s["w_scale"], bias=s["bias"],
                                 out=s["y"])


def _own_q8_quant(s):
    a = _sequence()
    a.quantize_q8(s["x"], blocks=s["blocks"], out=s["q"], scale=s["scale"])
    a.quantize_q8(s["x"], blocks=s["blocks"], transposed=True, out=s["qt"], scale=s["scale_t"])
    return s["q"].float(), s["scale"], s["qt"].float(), s["scale_t"]


def _own_q8_train(s):
    a = _sequence()
    w, wt = a.quantize_q8(s["w"], blocks=True), a.quantize_q8(s["w"], blocks=True, transposed=True)
    x, xt = a.quantize_q8(s["x"]), a.quantize_q8(s["x"], transposed=True)
    a.matmul_q8(x.out, x.scale, w.out, w.scale, out=s["y"])
    dy, dyt = a.quantize_q8(s["dy"]), a.quantize_q8(s["dy"], transposed=True)
    a.matmul_q8(dy.out, dy.scale, wt.out, wt.scale, out=s["dx"])
    a.matmul_q8(dyt.out, dyt.scale, xt.out, xt.scale, out=s["dw"])
    return s["y"], s["dx"], s["dw"]


_TRAINED = ("y", "final", "dq", "dk", "dv", "dinitial")
_OWN = {"attn": _own_attn, "attn_step": _own_attn_step, "attn_train": _own_attn_train,
        "q8": _own_q8, "q8_quant": _own_q8_quant, "q8_train": _own_q8_train}


# ---------------------------------------------------------------- plain forms: 8 bits

def _quantized(x, blocks=False):
    """(values in 8 bits, scales) of a matrix: by groups of 128 along its rows, or by blocks."""
    rows, dim = x.shape
    f = torch.nn.functional.pad(x.float(), (0, -dim % GROUP, 0, -rows % GROUP if blocks else 0))
    f = f.unflatten(-1, (-1, GROUP))  # (rows, groups, 128)
    most = f.abs().amax(-1)
    if blocks:
        most = most.unflatten(0, (-1, GROUP)).amax(1)
    # in 64 bits: a scale off by one unit takes values near a border to the other side of it
    scale = torch.where(most == 0, 1.0, most.double() / E4M3_MAX).float()
    by = scale.repeat_interleave(GROUP, 0) if blocks else scale
    q = (f / by[..., None]).flatten(1)[:rows, :dim]
    return q.to(torch.float8_e4m3fn), scale


def _values(q, scale):
    """The 32-bit values of 8-bit ones: scale has a row for each row or for every 128."""
    rows, dim = q.shape
    if scale.shape[0] != rows:
        scale = scale.repeat_interleave(GROUP, 0)[:rows]
    return q.float() * scale.repeat_interleave(GROUP, 1)[:, :dim]


def _plain_q8(s):
    y = _values(s["x"], s["x_scale"]) @ _values(s["w"], s["w_scale"]).T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["y"].dtype)


def _plain_q8_quant(s):
    q, scale = _quantized(s["x"], s["blocks"])
    qt, scale_t = _quantized(s["x"].T, s["blocks"])
    return q.float(), scale, qt.float(), scale_t


def _plain_q8_train(s):
    x, w = _values(*_quantized(s["x"])), _values(*_quantized(s["w"], True))
    y = x @ w.T
    dx = _values(*_quantized(s["dy"])) @ w
    dw = _values(*_quantized(s["dy"].T)) @ _values(*_quantized(s["x"].T)).T
    return y.to(s["y"].dtype), dx.to(s["dx"].dtype), dw


# ---------------------------------------------------------------- plain forms: linear attention

def _rows(s, name, heads):
    """(batch, heads, length, dim) in 32 bits, with zeros past the rows' ends."""
    v = s[name].float()
    if s["n_real"] is not None:
        live = torch.arange(v.shape[1], device="cuda") < s["n_real"][:, None]
        v = torch.where(live[..., None, None], v, 0)
    return v.transpose(1, 2).repeat_interleave(heads // v.shape[2], 1)


def _chunked(q, k, v, log_decay, start):
    """out[t] = q[t] S[t], S[t] = l S[t-1] + k[t]^T v[t] along the rows, from S = start or 0."""
    batch, heads, n, dk = q.shape
    chunk = min(CHUNK, n)
    q, k, v = (torch.nn.functional.pad(a, (0, 0, 0, -n % chunk)).unflatten(2, (-1, chunk))
               for a in (q, k, v))
    at = torch.arange(chunk, device="cuda", dtype=torch.float32)
    g = log_decay[:, None]
    apart = at[:, None] - at
    inner = torch.where(apart >= 0, torch.exp(g[..., None] * apart.clamp(min=0)), 0)
    front = torch.exp(g * (at + 1))[..., None]
    behind = torch.exp(g * (chunk - 1 - at))[..., None]
    whole = torch.exp(g * chunk)[..., None]
    out = ((q @ k.transpose(-1, -2)) * inner[:, None]) @ v
    added = (k * behind[:, None]).transpose(-1, -2) @ v
    state = torch.zeros_like(added[:, :, 0]) if start is None else start
    for c in range(q.shape[2]):
        out[:, :, c] += (q[:, :, c] * front) @ state
        state = state * whole + added[:, :, c]
    return out.flatten(2, 3)[:, :, :n]


def _real_lengths(s):
    batch, n = s["q"].shape[:2]
    if s["n_real"] is None:
        return torch.full((batch,), n, device="cuda")
    return s["n_real"].long()


def _moved(a, by):
    """Rows (batch, heads, length, dim) rolled to the right, each by its own count."""
    n = a.shape[2]
    at = (torch.arange(n, device="cuda") - by[:, None]) % n
    return a.gather(2, at[:, None, :, None].expand_as(a))


def _attn(s):
    heads = s["q"].shape[2]
    q, k, v = (_rows(s, name, heads) for name in ("q", "k", "v"))
    n = q.shape[2]
    y = _chunked(q, k, v, s["decay"], s["initial"])
    if s["n_real"] is not None:
        live = torch.arange(n, device="cuda") < s["n_real"][:, None]
        y = torch.where(live[:, None, :, None], y, 0)
    return y, q, k, v


def _final(s, k, v):
    """The state behind each row's last token, each token weighted by its distance from there."""
    real = _real_lengths(s)
    n = k.shape[2]
    g = s["decay"].double()[:, None]
    apart = (real[:, None, None] - 1 - torch.arange(n, device="cuda")).clamp(min=0)
    weight = torch.exp(g * apart).float()
    state = (k * weight[..., None]).transpose(-1, -2) @ v
    if s["initial"] is not None:
        state = state + torch.exp(g * real[:, None, None]).float()[..., None] * s["initial"]
    return state


def _plain_attn(s):
    y, _, k, v = _attn(s)
    return (y * s["scale"]).transpose(1, 2).to(s["y"].dtype), _final(s, k, v)


def _plain_attn_step(s):
    at, heads = s["slots"].long(), s["q"].shape[1]
    q, k, v = (s[name].float().repeat_interleave(heads // s[name].shape[1], 1)
               for name in ("q", "k", "v"))
    h = torch.exp(s["decay"])[:, None, None] * s["state"][at] + k[..., None] * v[..., None, :]
    s["state"][at] = h
    y = (q[..., None] * h).sum(-2) * s["scale"]
    return y.to(s["y"].dtype), s["state"]


def _plain_attn_train(s):
    y, q, k, v = _attn(s)
    g, kv, heads = s["decay"], s["k"].shape[2], s["q"].shape[2]
    kind = s["y"].dtype
    dy = _rows(s, "dy", heads) * s["scale"]
    real = _real_lengths(s)
    start = None if s["initial"] is None else s["initial"].transpose(-1, -2).contiguous()
    dq = _chunked(dy, v, k, g, start)
    back = lambda a: _moved(a.flip(2), real)  # noqa: E731  the rows' ends come first
    qr, kr, vr, dyr = (back(a) for a in (q, k, v, dy))
    dk = _moved(_chunked(vr, dyr, qr, g, None), -real).flip(2)
    dv = _moved(_chunked(kr, qr, dyr, g, None), -real).flip(2)
    live = (torch.arange(q.shape[2], device="cuda") < real[:, None])[:, None, :, None]
    dq, dk, dv = (torch.where(live, a, 0).transpose(1, 2) for a in (dq, dk, dv))
    shared = (kv, heads // kv)
    dk, dv = (a.unflatten(2, shared).sum(3) for a in (dk, dv))
    dinitial = None
    if s["initial"] is not None:
        at = torch.arange(1, q.shape[2] + 1, device="cuda")
        weight = torch.exp(g.double()[:, None] * at).float()
        dinitial = (q * weight[..., None]).transpose(-1, -2) @ dy
    return {"y": (y * s["scale"]).transpose(1, 2).to(kind), "final": _final(s, k, v),
            "dq": dq.to(kind), "dk": dk.to(kind), "dv": dv.to(kind), "dinitial": dinitial}


_PLAIN = {"attn": _plain_attn, "attn_step": _plain_attn_step, "attn_train": _plain_attn_train,
          "q8": _plain_q8, "q8_quant": _plain_q8_quant, "q8_train": _plain_q8_train}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits: attention one token after the other.
    The scales and the quotients that are rounded to 8 bits are float32 by definition."""
    s, op = prepare(case, seed), case["op"]
    if op == "q8":
        y = _exact_product(s["x"], s["x_scale"], s["w"], s["w_scale"])
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "q8_quant":
        q, scale = _exact_quantized(s["x"].double(), s["blocks"])
        qt, scale_t = _exact_quantized(s["x"].double().T, s["blocks"])
        return q.double(), scale.double(), qt.double(), scale_t.double()
    if op == "q8_train":
        x, w, dy = (s[k].double() for k in ("x", "w", "dy"))
        return (_exact_product(*_exact_quantized(x), *_exact_quantized(w, True)),
                _exact_product(*_exact_quantized(dy), *_exact_quantized(w.T, True)),
                _exact_product(*_exact_quantized(dy.T), *_exact_quantized(x.T)))
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v
         for k, v in s.items()}
    if op == "attn_step":
        at, share = s["slots"].long(), case["heads"] // case["kv"]
        k, v = (s[name].repeat_interleave(share, 1) for name in ("k", "v"))
        h = s["state"][at] * torch.exp(s["decay"]).reshape(-1, 1, 1)
        h = h + torch.einsum("bhk,bhv->bhkv", k, v)
        s["state"][at] = h
        return torch.einsum("bhk,bhkv->bhv", s["q"], h) * s["scale"], s["state"]
    return _exact_attn(case, s)


def _exact_quantized(x, blocks=False):
    """Group by group of columns, each magnitude, scale and quotient by its definition."""
    scales, values = [], []
    for at in range(0, x.shape[1], GROUP):
        part = x[:, at:at + GROUP]
        most = part.abs().max(1, keepdim=True).values
        if blocks:
            most = torch.cat([m.max().expand(len(m), 1) for m in most.split(GROUP)])
        scale = torch.where(most > 0, most / E4M3_MAX, torch.ones_like(most)).float()
        values.append((part / scale.double()).float().to(torch.float8_e4m3fn))
        scales.append(scale[::GROUP] if blocks else scale)
    return torch.cat(values, 1), torch.cat(scales, 1)


def _exact_product(x, x_scale, w, w_scale):
    out = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    if w_scale.shape[0] != w.shape[0]:
        w_scale = torch.cat([r.expand(GROUP, -1) for r in w_scale.split(1)])[:w.shape[0]]
    for g in range(x_scale.shape[1]):
        cut = slice(g * GROUP, (g + 1) * GROUP)
        left = x[:, cut].double() * x_scale[:, g:g + 1].double()
        out.addmm_(left, (w[:, cut].double() * w_scale[:, g:g + 1].double()).T)
    return out


def _exact_attn(case, s):
    share, n, scale = case["heads"] // case["kv"], case["len"], s["scale"]
    q = s["q"]
    k, v = (s[name].repeat_interleave(share, 2) for name in ("k", "v"))
    batch, heads, dk, dv = q.shape[0], q.shape[2], q.shape[3], v.shape[3]
    real = torch.full((batch,), n, device=q.device) if s["n_real"] is None else s["n_real"]
    decay = torch.exp(s["decay"]).reshape(-1, 1, 1)
    zero = torch.zeros(batch, heads, dk, dv, dtype=q.dtype, device=q.device)
    train, ragged = case["op"] == "attn_train", s["n_real"] is not None
    o = {"y": torch.zeros(batch, n, heads, dv, dtype=q.dtype, device=q.device),
         "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    h = zero if s["initial"] is None else s["initial"]
    for t in range(n):
        new = torch.einsum("bhk,bhv->bhkv", k[:, t], v[:, t]) + h * decay
        y = torch.einsum("bhk,bhkv->bhv", q[:, t], new) * scale
        dq = torch.einsum("bhv,bhkv->bhk", s["dy"][:, t], new) * scale if train else None
        if ragged:
            live = (t < real)[:, None, None]
            new, y = torch.where(live[..., None], new, h), torch.where(live, y, 0)
            dq = torch.where(live, dq, 0) if train else None
        h, o["y"][:, t] = new, y
        if train:
            o["dq"][:, t] = dq
    if not train:
        return o["y"], h
    o["final"], d = h, zero
    for t in reversed(range(n)):
        new = d + torch.einsum("bhk,bhv->bhkv", q[:, t], s["dy"][:, t]) * scale
        dk = torch.einsum("bhkv,bhv->bhk", new, v[:, t])
        dv = torch.einsum("bhkv,bhk->bhv", new, k[:, t])
        new = new * decay
        if ragged:
            live = (t < real)[:, None, None]
            new = torch.where(live[..., None], new, d)
            dk, dv = torch.where(live, dk, 0), torch.where(live, dv, 0)
        d, o["dk"][:, t], o["dv"][:, t] = new, dk, dv
    for name in ("dk", "dv"):
        o[name] = o[name].unflatten(2, (case["kv"], share)).sum(3)
    o["dinitial"] = None if s["initial"] is None else d
    return {name: o[name] for name in _TRAINED}
