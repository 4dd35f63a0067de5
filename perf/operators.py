"""Cases that measure the sequence operators: root-mean-square norm, short causal convolution and
selective state space scan, each for prompts, for single tokens where it keeps a state, and for
training.

``run`` computes an operator either in its plain form (elementary torch operations in 32 bits,
rounded once at the end) or, where ``own`` is true, through ``salt_b200.sequence``.  A scan's
plain form runs the affine maps (a, b) of all steps through log2(length) doubling steps.

Layouts: activations are (batch, length, channels) with contiguous channels; inputs that a block
cuts out of one projection (x and z; delta, B and C) are strided views of it.  Rows end at
``n_real`` tokens; what lies past that is not read and comes back as zero.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-5
E4M3_MAX = 448.0


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one decoding step's rows through the norm in front of a block: all latency
        {"name": "norm_step", "op": "norm", "rows": 16, "dim": 2048, "type": "bf16",
         "residual": "bf16"},
        # a large prompt batch, written in 8 bits for the projection that follows
        {"name": "norm_q8_prompt", "op": "norm_q8", "rows": 16384, "dim": 5120, "type": "bf16",
         "residual": "bf16", "group": 128},
        # training with a 32-bit residual stream, a width that is no multiple of a vector's
        {"name": "norm_back_odd", "op": "norm_back", "rows": 8190, "dim": 2500, "type": "bf16",
         "residual": "f32"},
        # one token for each of 64 requests, states in a pool
        {"name": "conv_step", "op": "conv_step", "batch": 64, "dim": 4096, "width": 4,
         "type": "bf16", "pool": 96},
        # ragged prompts that continue earlier chunks
        {"name": "conv_prompt", "op": "conv", "batch": 4, "len": 4096, "dim": 4096, "width": 4,
         "type": "bf16", "ragged": True, "initial": True},
        # a training step's convolution, forward and backward
        {"name": "conv_train", "op": "conv_train", "batch": 8, "len": 2048, "dim": 2048,
         "width": 4, "type": "bf16", "ragged": False, "initial": False},
        # a single request's token: all latency
        {"name": "scan_step_one", "op": "scan_step", "batch": 1, "dim": 1536, "state": 16,
         "groups": 1, "type": "bf16", "pool": 1},
        # a full serving batch: reading and writing the states is the work
        {"name": "scan_step_many", "op": "scan_step", "batch": 256, "dim": 8192, "state": 16,
         "groups": 1, "type": "bf16", "pool": 320},
        # one long prompt: few channels' rows, so the length has to be split
        {"name": "scan_prompt_long", "op": "scan", "batch": 1, "len": 16384, "dim": 2048,
         "state": 16, "groups": 1, "type": "bf16", "ragged": False, "initial": True},
        # a batch of ragged prompts
        {"name": "scan_prompt_batch", "op": "scan", "batch": 8, "len": 2048, "dim": 4096,
         "state": 16, "groups": 1, "type": "bf16", "ragged": True, "initial": False},
        # a training step's scan, forward and backward
        {"name": "scan_train", "op": "scan_train", "batch": 4, "len": 2048, "dim": 2048,
         "state": 16, "groups": 1, "type": "bf16", "ragged": False, "initial": False},
        # training in 32 bits with sizes that are multiples of nothing and shared B and C
        {"name": "scan_train_odd", "op": "scan_train", "batch": 3, "len": 1021, "dim": 1002,
         "state": 12, "groups": 2, "type": "f32", "ragged": True, "initial": True},
    ]


def _log(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))
    return v + (v == 3 * 1024)


def _dim(rng, low, high):
    """A width: a multiple of 128, of 8, or any number."""
    step = rng.choice((128, 8, 1))
    d = max(step, _log(rng, low, high) // step * step)
    return d + step if d == 3 * 1024 else d


def draw(rng):
    op = rng.choice(("norm", "norm_q8", "norm_back", "conv", "conv_step", "conv_train", "scan",
                     "scan", "scan_step", "scan_train"))
    kind = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op.startswith("norm"):
        dim = _dim(rng, 64, 8192)
        case = {"op": op, "rows": _log(rng, 1, min(32768, 40_000_000 // dim)), "dim": dim,
                "type": kind, "residual": rng.choice((kind, "f32"))}
        if op == "norm_q8":
            case["group"] = rng.choice((0, 32, 64, 128))
        return case
    if op.endswith("step"):
        batch = _log(rng, 1, 256)
        case = {"op": op, "batch": batch, "dim": _dim(rng, 64, 8192), "type": kind,
                "pool": batch + rng.randrange(0, 65)}
        if op == "conv_step":
            return case | {"width": rng.choice((2, 3, 4))}
        return _states(rng, case, 256 * 8192 * 16 / (batch * case["dim"]))
    batch, dim = _log(rng, 1, 16), _dim(rng, 64, 8192)
    case = {"op": op, "batch": batch, "dim": dim, "type": kind,
            "ragged": rng.random() < 0.5, "initial": rng.random() < 0.5}
    if op.startswith("conv"):
        most = 4 * 4096 * 4096 if op == "conv" else 8 * 2048 * 2048
        return case | {"len": _log(rng, 1, min(16384, most // (batch * dim))),
                       "width": rng.choice((2, 3, 4))}
    most = 8 * 2048 * 4096 * 16 if op == "scan" else 4 * 2048 * 2048 * 16
    case = _states(rng, case, most / (batch * dim))
    return case | {"len": _log(rng, 1, min(16384, most // (batch * dim * case["state"])))}


def _states(rng, case, most):
    state = rng.choice([n for n in (4, 8, 12, 16, 16, 16, 24, 32, 64) if n <= max(4, most)])
    fit = [g for g in (1, 1, 2, 4) if case["dim"] % g == 0]
    return case | {"state": state, "groups": rng.choice(fit)}


# ---------------------------------------------------------------- inputs

class _Make:
    """Inputs on the GPU from one seed."""

    def __init__(self, case, seed):
        self.type = _TYPES[case["type"]]
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, scale=1.0, type=None):
        v = torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return v.mul_(scale).to(type or self.type)

    def uniform(self, low, high, *shape):
        v = torch.rand(*shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return v * (high - low) + low

    def lengths(self, case):
        """The rows' token counts: evenly from none to all, in an order of the seed's; or None."""
        if not case["ragged"]:
            return None
        spread = torch.tensor(_real(case), device="cuda", dtype=torch.int32)
        return spread[torch.randperm(case["batch"], generator=self.gen, device="cuda")]

    def slots(self, batch, pool):
        return torch.randperm(pool, generator=self.gen, device="cuda")[:batch].to(torch.int32)

    def empty(self, *shape, type=None):
        return torch.empty(*shape, device="cuda", dtype=type or self.type)


def prepare(case, seed):
    m, op = _Make(case, seed), case["op"]
    s = {"op": op, "case": case}
    if op.startswith("norm"):
        rows, dim, wide = case["rows"], case["dim"], _TYPES[case["residual"]]
        s["weight"] = m.normal(dim, scale=0.2).add_(1)
        if op == "norm_back":
            s["x"] = m.normal(rows, dim, scale=2.0, type=wide)  # the residual stream it normed
            s["rstd"] = torch.rsqrt(s["x"].float().square().mean(-1) + EPS)
            s["dy"] = m.normal(rows, dim, scale=0.1)
            s["dresidual"] = m.normal(rows, dim, scale=0.1, type=wide)
            s["dx"] = m.empty(rows, dim, type=wide)
            s["dweight"] = m.empty(dim, type=torch.float32)
            return s
        s["x"], s["residual"] = m.normal(rows, dim), m.normal(rows, dim, scale=2.0, type=wide)
        s["residual_out"] = m.empty(rows, dim, type=wide)
        if op == "norm":
            s["y"] = m.empty(rows, dim)
        else:
            s["group"] = case["group"]
            s["y"] = m.empty(rows, dim, type=torch.float8_e4m3fn)
            s["scale"] = m.empty(rows, _parts(case), type=torch.float32)
        return s
    batch, dim = case["batch"], case["dim"]
    if op.startswith("conv"):
        width = case["width"]
        s["weight"], s["bias"] = m.normal(dim, width, scale=width ** -0.5), m.normal(dim, scale=0.1)
        if op == "conv_step":
            s["x"] = m.normal(batch, 2 * dim)[:, :dim]
            s["state"] = m.normal(case["pool"], dim, width - 1)
            s["slots"], s["y"] = m.slots(batch, case["pool"]), m.empty(batch, dim)
            return s
        n = case["len"]
        s["x"] = m.normal(batch, n, 2 * dim)[:, :, :dim]
        s["n_real"] = m.lengths(case)
        s["initial"] = m.normal(batch, dim, width - 1) if case["initial"] else None
        s["y"], s["final"] = m.empty(batch, n, dim), m.empty(batch, dim, width - 1)
        if op == "conv_train":
            s["dy"] = m.normal(batch, n, dim, scale=0.1)
            s["dx"], s["dinitial"] = m.empty(batch, n, dim), None
            if case["initial"]:
                s["dinitial"] = m.empty(batch, dim, width - 1)
            s["dweight"] = m.empty(dim, width, type=torch.float32)
            s["dbias"] = m.empty(dim, type=torch.float32)
        return s
    state, groups = case["state"], case["groups"]
    s["A"] = -(m.uniform(0.8, 1.2, dim, state) * torch.arange(1, state + 1, device="cuda"))
    s["D"] = m.normal(dim, scale=0.2, type=torch.float32).add_(1)
    step = torch.exp(m.uniform(math.log(1e-3), math.log(1e-1), dim))
    s["bias"] = torch.log(torch.expm1(step))  # softplus(bias) lies in [1e-3, 1e-1]
    lead = (batch,) if op == "scan_step" else (batch, case["len"])
    s["x"] = torch.nn.functional.silu(m.normal(*lead, dim))
    s["z"] = m.normal(*lead, 2 * dim)[..., dim:]
    s["delta"] = m.normal(*lead, dim, scale=0.5)
    both = m.normal(*lead, 2 * groups * state + 8)[..., 8:]
    s["B"] = both[..., :groups * state].unflatten(-1, (groups, state))
    s["C"] = both[..., groups * state:].unflatten(-1, (groups, state))
    s["y"] = m.empty(*lead, dim)
    if op == "scan_step":
        s["state"] = m.normal(case["pool"], dim, state, scale=0.1, type=torch.float32)
        s["slots"] = m.slots(batch, case["pool"])
        return s
    n = case["len"]
    s["n_real"] = m.lengths(case)
    s["initial"], s["dinitial"] = None, None
    if case["initial"]:
        s["initial"] = m.normal(batch, dim, state, scale=0.1, type=torch.float32)
    s["final"] = m.empty(batch, dim, state, type=torch.float32)
    if op == "scan_train":
        s["dy"] = m.normal(batch, n, dim, scale=0.1)
        s["dx"], s["ddelta"], s["dz"] = (m.empty(batch, n, dim) for _ in range(3))
        s["dB"], s["dC"] = (m.empty(batch, n, groups, state) for _ in range(2))
        s["dA"] = m.empty(dim, state, type=torch.float32)
        s["dD"], s["dbias"] = (m.empty(dim, type=torch.float32) for _ in range(2))
        if case["initial"]:
            s["dinitial"] = m.empty(batch, dim, state, type=torch.float32)
    return s


def _real(case):
    batch, n = case["batch"], case["len"]
    if not case["ragged"] or batch == 1:
        return [n] * batch
    return [n * i // (batch - 1) for i in range(batch)]


def _parts(case):
    return -(-case["dim"] // case["group"]) if case["group"] else 1


# ---------------------------------------------------------------- one pass

def run(s):
    return (_OWN if own else _PLAIN)[s["op"]](s)


def work(case):
    """Each input read once and each output written once, and the operator's arithmetic."""
    e, op = _BYTES[case["type"]], case["op"]
    if op.startswith("norm"):
        n, wide = case["rows"] * case["dim"], _BYTES[case["residual"]]
        if op == "norm":
            return {"bytes": n * (2 * e + 2 * wide), "flops": 5 * n}
        if op == "norm_q8":
            return {"bytes": n * (e + 2 * wide + 1) + 4 * case["rows"] * _parts(case),
                    "flops": 8 * n}
        return {"bytes": n * (e + 3 * wide) + 4 * case["rows"], "flops": 10 * n}
    batch, dim = case["batch"], case["dim"]
    if op.startswith("conv"):
        taps = case["width"]
        if op == "conv_step":
            return {"bytes": batch * dim * e * (2 + 2 * (taps - 1)) + dim * (taps + 1) * e,
                    "flops": batch * dim * (2 * taps + 5)}
        n, live = batch * case["len"] * dim, sum(_real(case)) * dim
        ends = batch * dim * (taps - 1) * e * (2 if case["initial"] else 1)
        if op == "conv":
            return {"bytes": (n + live) * e + ends, "flops": live * (2 * taps + 5)}
        return {"bytes": (2 * n + 3 * live) * e + ends, "flops": live * (8 * taps + 15)}
    state, groups = case["state"], case["groups"]
    if op == "scan_step":
        n = batch * dim
        return {"bytes": n * (4 * e + 8 * state) + 2 * batch * groups * state * e
                + 4 * dim * (state + 2), "flops": n * (7 * state + 15)}
    n, live, tokens = batch * case["len"] * dim, sum(_real(case)) * dim, sum(_real(case))
    ends = batch * dim * state * 4 * (2 if case["initial"] else 1)
    if op == "scan":
        return {"bytes": (n + 3 * live) * e + 2 * tokens * groups * state * e + ends,
                "flops": live * (7 * state + 15)}
    return {"bytes": (4 * n + 7 * live) * e + 6 * tokens * groups * state * e + ends,
            "flops": live * (27 * state + 50)}


# ---------------------------------------------------------------- the framework's calls

def _sequence():
    import salt_b200.sequence as sequence
    return sequence


def _own_norm(s):
    _sequence().rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, out=s["y"],
                         residual_out=s["residual_out"])
    return s["y"], s["residual_out"]


def _own_norm_q8(s):
    _sequence().rms_norm_q8(s["x"], s["weight"], residual=s["residual"], eps=EPS,
                            group=s["group"], out=s["y"], scale=s["scale"],
                            residual_out=s["residual_out"])
    return s["y"], s["scale"], s["residual_out"]


def _own_norm_back(s):
    _sequence().rms_norm_backward(s["dy"], s["x"], s["weight"], s["rstd"],
                                  dresidual=s["dresidual"], dx=s["dx"], dweight=s["dweight"])
    return s["dx"], s["dweight"]


def _own_conv(s):
    _sequence().causal_conv(s["x"], s["weight"], s["bias"], n_real=s["n_real"],
                            initial_state=s["initial"], silu=True, out=s["y"],
                            final_state=s["final"])
    return s["y"], s["final"]


def _own_conv_step(s):
    _sequence().causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], slots=s["slots"],
                                 silu=True, out=s["y"])
    return s["y"], s["state"]


def _own_conv_train(s):
    q = _sequence()
    q.causal_conv(s["x"], s["weight"], s["bias"], n_real=s["n_real"],
                  initial_state=s["initial"], silu=True, out=s["y"], final_state=s["final"])
    q.causal_conv_backward(s["dy"], s["x"], s["weight"], s["bias"], n_real=s["n_real"],
                           initial_state=s["initial"], silu=True, dx=s["dx"],
                           dweight=s["dweight"], dbias=s["dbias"], dinitial=s["dinitial"])
    return {k: s[k] for k in ("y", "final", "dx", "dweight", "dbias", "dinitial")}


def _own_scan(s):
    _sequence().selective_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                               delta_bias=s["bias"], softplus=True, n_real=s["n_real"],
                               initial_state=s["initial"], out=s["y"], final_state=s["final"])
    return s["y"], s["final"]


def _own_scan_step(s):
    _sequence().selective_scan_step(s["state"], s["x"], s["delta"], s["A"], s["B"], s["C"],
                                    D=s["D"], z=s["z"], delta_bias=s["bias"], softplus=True,
                                    slots=s["slots"], out=s["y"])
    return s["y"], s["state"]


def _own_scan_train(s):
    q = _sequence()
    f = q.selective_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                         delta_bias=s["bias"], softplus=True, n_real=s["n_real"],
                         initial_state=s["initial"], out=s["y"], final_state=s["final"],
                         checkpoints=True)
    q.selective_scan_backward(s["dy"], s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["D"],
                              z=s["z"], delta_bias=s["bias"], softplus=True,
                              n_real=s["n_real"], checkpoints=f.checkpoints, dx=s["dx"],
                              ddelta=s["ddelta"], dA=s["dA"], dB=s["dB"], dC=s["dC"],
                              dD=s["dD"], dz=s["dz"], ddelta_bias=s["dbias"],
                              dinitial=s["dinitial"])
    return {k: s[k] for k in _TRAINED}


_TRAINED = ("y", "final", "dx", "ddelta", "dz", "dA", "dB", "dC", "dD", "dbias", "dinitial")
_OWN = {"norm": _own_norm, "norm_q8": _own_norm_q8, "norm_back": _own_norm_back,
        "conv": _own_conv, "conv_step": _own_conv_step, "conv_train": _own_conv_train,
        "scan": _own_scan, "scan_step": _own_scan_step, "scan_train": _own_scan_train}


# ---------------------------------------------------------------- plain forms

def _silu(v):
    return v * torch.sigmoid(v)


def _silu_slope(v):
    p = torch.sigmoid(v)
    return p * (1 + v * (1 - p))


def _softplus(v):
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))


def _mask(s, length):
    """(batch, length, 1): which tokens are real; None where all are."""
    if s["n_real"] is None:
        return None
    return (torch.arange(length, device="cuda") < s["n_real"][:, None])[..., None]


def _kept(v, mask):
    return v if mask is None else torch.where(mask, v, 0)


def _normed(s):
    r = s["x"].float() + s["residual"].float()
    y = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    return r.to(s["residual"].dtype), y


def _plain_norm(s):
    r, y = _normed(s)
    return y.to(s["x"].dtype), r


def _plain_norm_q8(s):
    r, y = _normed(s)
    rows, dim = y.shape
    group = s["group"] or dim
    pad = torch.nn.functional.pad(y, (0, -dim % group)).unflatten(-1, (-1, group))
    most = pad.abs().amax(-1)
    scale = torch.where(most == 0, 1.0, most / E4M3_MAX)
    q = (pad / scale[..., None]).flatten(-2)[:, :dim]
    return q.to(torch.float8_e4m3fn), scale, r


def _plain_norm_back(s):
    dy, x, rstd = s["dy"].float(), s["x"].float(), s["rstd"][:, None]
    hat = x * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - hat * (g * hat).mean(-1, keepdim=True)) + s["dresidual"].float()
    return dx.to(s["x"].dtype), (dy * hat).sum(0)


def _conv_parts(s):
    """The padded inputs (batch, width - 1 + length, dim), the sums before the gate, the mask."""
    x = s["x"].float()
    batch, n, dim = x.shape
    taps = s["weight"].shape[1]
    mask = _mask(s, n)
    x = _kept(x, mask)
    before = x.new_zeros(batch, taps - 1, dim)
    if s["initial"] is not None:
        before = s["initial"].float().transpose(1, 2)
    full = torch.cat((before, x), 1)
    w = s["weight"].float()
    pre = s["bias"].float() + sum(full[:, k:k + n] * w[:, k] for k in range(taps))
    return full, pre, mask


def _conv_outputs(s, full, pre, mask):
    batch, n, dim = pre.shape
    taps = s["weight"].shape[1]
    y = _kept(_silu(pre), mask).to(s["x"].dtype)
    last = torch.full((batch,), n, device="cuda") if s["n_real"] is None else s["n_real"].long()
    at = last[:, None] + torch.arange(taps - 1, device="cuda")
    final = full.gather(1, at[..., None].expand(-1, -1, dim)).transpose(1, 2)
    return y, final.to(s["x"].dtype)


def _plain_conv(s):
    return _conv_outputs(s, *_conv_parts(s))


def _plain_conv_step(s):
    at = s["slots"].long()
    full = torch.cat((s["state"][at].float(), s["x"].float()[..., None]), -1)
    y = _silu((full * s["weight"].float()).sum(-1) + s["bias"].float())
    s["state"][at] = full[..., 1:].to(s["state"].dtype)
    return y.to(s["x"].dtype), s["state"]


def _plain_conv_train(s):
    full, pre, mask = _conv_parts(s)
    y, final = _conv_outputs(s, full, pre, mask)
    batch, n, dim = pre.shape
    taps = s["weight"].shape[1]
    w = s["weight"].float()
    g = _kept(s["dy"].float() * _silu_slope(pre), mask)
    dfull = torch.zeros_like(full)
    for k in range(taps):
        dfull[:, k:k + n] += g * w[:, k]
    dweight = torch.stack([(g * full[:, k:k + n]).sum((0, 1)) for k in range(taps)], -1)
    dinitial = None
    if s["initial"] is not None:
        dinitial = dfull[:, :taps - 1].transpose(1, 2).to(s["x"].dtype)
    return {"y": y, "final": final, "dx": _kept(dfull[:, taps - 1:], mask).to(s["x"].dtype),
            "dweight": dweight, "dbias": g.sum((0, 1)), "dinitial": dinitial}


def _affine(a, b):
    """h[t] = a[t] * h[t-1] + b[t] along dimension 1 from h = 0, by doubling."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat((b[:, :span], torch.addcmul(b[:, span:], a[:, span:], b[:, :-span])), 1)
        a = torch.cat((a[:, :span], a[:, span:] * a[:, :-span]), 1)
        span *= 2
    return b


def _spread(v, dim):
    """(..., groups, state) to (..., dim, state): each channel's group."""
    groups, state = v.shape[-2:]
    v = v.float().unsqueeze(-2).expand(*v.shape[:-1], dim // groups, state)
    return v.flatten(-3, -2)


def _scan_parts(s):
    n, dim = s["x"].shape[1:]
    mask = _mask(s, n)
    x, raw = _kept(s["x"].float(), mask), _kept(s["delta"].float() + s["bias"], mask)
    step = _kept(_softplus(raw), mask)
    over = None if mask is None else mask[..., None]
    b_in, c_in = (_spread(_kept(s[k].float(), over), dim) for k in ("B", "C"))
    a = torch.exp(step[..., None] * s["A"])
    b = (step * x)[..., None] * b_in
    if s["initial"] is not None:
        b[:, 0] += a[:, 0] * s["initial"]
    h = _affine(a, b)
    y = (h * c_in).sum(-1) + s["D"] * x
    return mask, x, raw, step, b_in, c_in, a, h, y


def _plain_scan(s):
    mask, *_, h, y = _scan_parts(s)
    return _kept(y * _silu(s["z"].float()), mask).to(s["x"].dtype), h[:, -1].clone()


def _plain_scan_step(s):
    at, dim = s["slots"].long(), s["x"].shape[1]
    x, z = s["x"].float(), s["z"].float()
    step = _softplus(s["delta"].float() + s["bias"])
    h = torch.exp(step[..., None] * s["A"]) * s["state"][at]
    h = h + (step * x)[..., None] * _spread(s["B"], dim)
    y = ((h * _spread(s["C"], dim)).sum(-1) + s["D"] * x) * _silu(z)
    s["state"][at] = h
    return y.to(s["x"].dtype), s["state"]


def _plain_scan_train(s):
    mask, x, raw, step, b_in, c_in, a, h, y = _scan_parts(s)
    kind, z, dy = s["x"].dtype, _kept(s["z"].float(), mask), _kept(s["dy"].float(), mask)
    batch, n, dim = x.shape
    groups, state = s["B"].shape[2:]
    g = dy * _silu(z)
    later = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), 1)
    dh = _affine(later.flip(1), (g[..., None] * c_in).flip(1)).flip(1)
    del later
    first = torch.zeros_like(h[:, :1]) if s["initial"] is None else s["initial"][:, None]
    moved = dh * a * torch.cat((first, h[:, :-1]), 1)
    through = (dh * b_in).sum(-1)
    dstep = (moved * s["A"]).sum(-1) + x * through
    draw = _kept(dstep * torch.sigmoid(raw), mask)
    split = (batch, n, groups, dim // groups, state)
    return {
        "y": _kept(y * _silu(s["z"].float()), mask).to(kind), "final": h[:, -1].clone(),
        "dx": _kept(step * through + g * s["D"], mask).to(kind), "ddelta": draw.to(kind),
        "dz": _kept(dy * y * _silu_slope(z), mask).to(kind),
        "dA": (moved * step[..., None]).sum((0, 1)),
        "dB": (dh * (step * x)[..., None]).reshape(split).sum(3).to(kind),
        "dC": (h * g[..., None]).reshape(split).sum(3).to(kind),
        "dD": (g * x).sum((0, 1)), "dbias": draw.sum((0, 1)),
        "dinitial": None if s["initial"] is None else dh[:, 0] * a[:, 0]}


_PLAIN = {"norm": _plain_norm, "norm_q8": _plain_norm_q8, "norm_back": _plain_norm_back,
          "conv": _plain_conv, "conv_step": _plain_conv_step, "conv_train": _plain_conv_train,
          "scan": _plain_scan, "scan_step": _plain_scan_step, "scan_train": _plain_scan_train}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits: one token after the other."""
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() and v.dtype.itemsize > 1
         else v for k, v in prepare(case, seed).items()}
    op = case["op"]
    if op.startswith("norm"):
        return _exact_norm(op, s)
    if op == "conv_step":
        at = s["slots"].long()
        taps = torch.cat((s["state"][at], s["x"].unsqueeze(-1)), -1)
        pre = torch.einsum("bdk,dk->bd", taps, s["weight"]) + s["bias"]
        s["state"][at] = taps[..., 1:]
        return pre / (1 + torch.exp(-pre)), s["state"]
    if op.startswith("conv"):
        return _exact_conv(op, s)
    if op == "scan_step":
        at = s["slots"].long()
        h, y = _exact_token(s, s["state"][at], s["x"], s["delta"], s["B"], s["C"])[:2]
        s["state"][at] = h
        return y * s["z"] / (1 + torch.exp(-s["z"])), s["state"]
    if case["batch"] * case["len"] * case["dim"] * case["state"] > 3e8 and op == "scan_train":
        return None
    return _exact_scan(op, s)


def _exact_norm(op, s):
    if op == "norm_back":
        hat = s["x"] * s["rstd"].unsqueeze(1)
        inner = torch.einsum("rd,rd,d->r", s["dy"], hat, s["weight"]) / hat.shape[1]
        dx = (s["dy"] * s["weight"] - hat * inner.unsqueeze(1)) * s["rstd"].unsqueeze(1)
        return dx + s["dresidual"], torch.einsum("rd,rd->d", s["dy"], hat)
    r = s["x"] + s["residual"]
    size = torch.sqrt(torch.einsum("rd,rd->r", r, r) / r.shape[1] + EPS)
    y = r / size.unsqueeze(1) * s["weight"]
    if op == "norm":
        return y, r
    dim, group = y.shape[1], s["group"] or y.shape[1]
    scales, values = [], []
    for at in range(0, dim, group):
        part = y[:, at:at + group]
        most = part.abs().max(1, keepdim=True).values
        scales.append(torch.where(most > 0, most / E4M3_MAX, torch.ones_like(most)))
        values.append((part / scales[-1]).to(torch.float8_e4m3fn).double())
    return torch.cat(values, 1), torch.cat(scales, 1), r


def _lengths(s):
    batch, n = s["x"].shape[:2]
    return [n] * batch if s["n_real"] is None else s["n_real"].tolist()


def _exact_conv(op, s):
    x, w = s["x"], s["weight"]
    batch, n, dim = x.shape
    taps = w.shape[1]
    out = {k: torch.zeros_like(x) for k in ("y", "dx")}
    out["final"] = torch.zeros(batch, dim, taps - 1, dtype=x.dtype, device=x.device)
    out["dweight"], out["dbias"] = torch.zeros_like(w), torch.zeros_like(s["bias"])
    out["dinitial"] = None if s["initial"] is None else torch.zeros_like(s["initial"])
    for i, real in enumerate(_lengths(s)):
        head = torch.zeros(dim, taps - 1, dtype=x.dtype, device=x.device)
        head = head if s["initial"] is None else s["initial"][i]
        line = torch.cat((head, x[i, :real].T), 1)  # (dim, taps - 1 + real)
        out["final"][i] = line[:, real:]
        if not real:
            continue
        seen = line.unfold(1, taps, 1)  # (dim, real, taps)
        pre = torch.einsum("dtk,dk->td", seen, w) + s["bias"]
        gate = 1 / (1 + torch.exp(-pre))
        out["y"][i, :real] = pre * gate
        if op == "conv":
            continue
        g = s["dy"][i, :real] * (gate + pre * gate * (1 - gate))
        out["dweight"] += torch.einsum("td,dtk->dk", g, seen)
        out["dbias"] += g.sum(0)
        back = torch.nn.functional.pad(g.T, (taps - 1, taps - 1)).unfold(1, taps, 1)
        dline = torch.einsum("dtk,dk->dt", back, w.flip(1))
        out["dx"][i, :real] = dline[:, taps - 1:].T
        if s["initial"] is not None:
            out["dinitial"][i] = dline[:, :taps - 1]
    if op == "conv":
        return out["y"], out["final"]
    return {k: out[k] for k in ("y", "final", "dx", "dweight", "dbias", "dinitial")}


def _exact_token(s, h, x, delta, b_in, c_in):
    """One token of every row: the new state, y before the gate, the step, its slope, a, B, C."""
    per = x.shape[1] // b_in.shape[1]
    raw = delta + s["bias"]
    step = torch.logaddexp(raw, torch.zeros_like(raw))
    b_in, c_in = (v.unsqueeze(2).expand(-1, -1, per, -1).flatten(1, 2) for v in (b_in, c_in))
    a = torch.exp(step.unsqueeze(-1) * s["A"])
    h = a * h + torch.einsum("bd,bdn->bdn", step * x, b_in)
    y = torch.einsum("bdn,bdn->bd", h, c_in) + s["D"] * x
    return h, y, step, 1 / (1 + torch.exp(-raw)), a, b_in, c_in


def _exact_scan(op, s):
    x, z = s["x"], s["z"]
    batch, n, dim = x.shape
    state = s["A"].shape[1]
    real = torch.tensor(_lengths(s), device=x.device)
    start = torch.zeros(batch, dim, state, dtype=x.dtype, device=x.device)
    start = start if s["initial"] is None else s["initial"]
    h, y, kept = start, torch.zeros_like(x), [start]
    for t in range(n):
        live = (t < real)[:, None]
        new, out = _exact_token(s, h, x[:, t], s["delta"][:, t], s["B"][:, t], s["C"][:, t])[:2]
        h = torch.where(live[..., None], new, h)
        y[:, t] = torch.where(live, out, 0)
        if op == "scan_train":
            kept.append(h)
    p = 1 / (1 + torch.exp(-z))
    if op == "scan":
        return y * z * p, h
    live = (torch.arange(n, device=x.device) < real[:, None]).unsqueeze(-1)
    dy = torch.where(live, s["dy"], 0)
    o = {"y": y * z * p, "final": h, "dz": dy * y * (p + z * p * (1 - p))}
    for k in ("dx", "ddelta"):
        o[k] = torch.zeros_like(x)
    for k in ("A", "D", "bias", "B", "C"):
        o["d" + k] = torch.zeros_like(s[k])
    carry = torch.zeros_like(start)
    groups = s["B"].shape[2]
    for t in reversed(range(n)):
        now = live[:, t]
        _, _, step, slope, a, b_in, c_in = _exact_token(s, kept[t], x[:, t], s["delta"][:, t],
                                                        s["B"][:, t], s["C"][:, t])
        g = dy[:, t] * z[:, t] * p[:, t]
        dh = torch.where(now[..., None], carry + g.unsqueeze(-1) * c_in, 0)
        old = dh * a * kept[t]
        into = torch.einsum("bdn,bdn->bd", dh, b_in)
        draw = (torch.einsum("bdn,dn->bd", old, s["A"]) + x[:, t] * into) * slope
        o["dx"][:, t] = torch.where(now, step * into + g * s["D"], 0)
        o["ddelta"][:, t] = torch.where(now, draw, 0)
        o["dbias"] += o["ddelta"][:, t].sum(0)
        o["dD"] += torch.where(now, g * x[:, t], 0).sum(0)
        o["dA"] += torch.einsum("bdn,bd->dn", old, step)
        o["dB"][:, t] = torch.einsum("bdn,bd->bdn", dh, step * x[:, t]).unflatten(
            1, (groups, -1)).sum(2)
        o["dC"][:, t] = torch.einsum("bdn,bd->bdn", kept[t + 1], g).unflatten(
            1, (groups, -1)).sum(2) * now[..., None]
        carry = torch.where(now[..., None], a * dh, carry)
    o["dinitial"] = None if s["initial"] is None else carry
    return {k: o[k] for k in _TRAINED}
