"""Measured cases of the sequence operators next to the convolution modules: group norm with an
activation and the gated linear recurrence, each forward and backward.

Activations are ``[N, T, C]`` (channels last) with int32 ``valid_lengths [N]``; frames at or past
an utterance's length are padding. ``own`` false runs the operators' plain form in 32 bits, true
the framework's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

STATE_FRAMES = 64  # frames between two saved states of the recurrence

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def _norm(name, n, t, c, groups, dtype, activation, ragged, statistics=False):
    return {"name": name, "op": "norm", "n": n, "t": t, "c": c, "groups": groups, "dtype": dtype,
            "activation": activation, "ragged": ragged, "statistics": statistics}


def _norm_gradient(name, n, t, c, groups, dtype, activation, ragged):
    return {"name": name, "op": "norm gradient", "n": n, "t": t, "c": c, "groups": groups,
            "dtype": dtype, "activation": activation, "ragged": ragged}


def _recurrence(name, n, t, c, dtype, ragged, states=False):
    return {"name": name, "op": "recurrence", "n": n, "t": t, "c": c, "dtype": dtype,
            "ragged": ragged, "states": states}


def _recurrence_gradient(name, n, t, c, dtype, ragged):
    return {"name": name, "op": "recurrence gradient", "n": n, "t": t, "c": c, "dtype": dtype,
            "ragged": ragged}


def listed():
    return [
        # One new frame of one stream through a convolution module's norm: latency alone.
        _norm("norm one frame", 1, 1, 512, 32, "f16", "silu", False),
        # The Conformer batch of 256 x 30 s at 80 ms, with the statistics that training keeps.
        _norm("norm batch f16", 256, 375, 1024, 32, "f16", "silu", True, True),
        # Odd channels and frames without an activation: groups of 17 channels, fp32.
        _norm("norm odd f32", 5, 733, 323, 19, "f32", "none", True),
        # A small fine-tuning batch of an 80-channel frontend, fp32.
        _norm_gradient("norm gradient short f32", 3, 37, 80, 8, "f32", "swoosh_r", True),
        # Training the first Zipformer stack: 256 x 30 s at 40 ms, 192 channels.
        _norm_gradient("norm gradient batch bf16", 256, 750, 192, 6, "bf16", "swoosh_r", True),
        # Long-form training, one group: statistics over all of a 240 s utterance.
        _norm_gradient("norm gradient long f16", 16, 3000, 1024, 1, "f16", "silu", True),
        # One decoding step of 64 streams: the serving form, states carried between calls.
        _recurrence("recurrence one frame", 64, 1, 512, "bf16", False),
        # The Conformer batch, inference.
        _recurrence("recurrence batch bf16", 256, 375, 1024, "bf16", True),
        # Two recordings of 16 minutes, few rows and a long axis, states kept for training.
        _recurrence("recurrence long f16", 2, 12000, 512, "f16", False, True),
        # Odd everything, fp32.
        _recurrence_gradient("recurrence gradient odd f32", 5, 333, 77, "f32", True),
        # The Conformer batch, training.
        _recurrence_gradient("recurrence gradient batch f16", 256, 375, 1024, "f16", True),
        # Training on the two long recordings.
        _recurrence_gradient("recurrence gradient long bf16", 2, 12000, 512, "bf16", False),
    ]


def _spread(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "norm gradient", "recurrence", "recurrence gradient"])
    n, t = _spread(rng, 1, 256), _spread(rng, 1, 12000)
    if op.startswith("norm"):
        groups = rng.choice([1, _spread(rng, 1, 64), _spread(rng, 1, 64)])
        # A group of a few values has hardly any variance: its gradient is rounding alone.
        c = groups * _spread(rng, 1 if t >= 64 else 8, max(8, 1024 // groups))
    else:
        c = _spread(rng, 8, 1024)
    n = max(1, min(n, 40_000_000 // (t * c)))
    case = {"op": op, "n": n, "t": t, "c": c, "dtype": rng.choice(["f32", "f16", "bf16"]),
            "ragged": rng.random() < 0.7}
    if op.startswith("norm"):
        case |= {"groups": groups, "activation": rng.choice(["none", "silu", "swoosh_r"])}
    if op == "norm":
        case["statistics"] = rng.random() < 0.5
    if op == "recurrence":
        case["states"] = rng.random() < 0.5
    return case


def _lengths(case):
    """Valid frames of each utterance, in order: all of them, or spread evenly from a sixth of T."""
    n, t = case["n"], case["t"]
    if not case["ragged"]:
        return [t] * n
    low = max(1, t // 6)
    return [low + round((t - low) * (i + 0.5) / n) for i in range(n)]


def _chunks(t):
    return -(-t // STATE_FRAMES)


# ---- inputs -----------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    n, t, c, dtype = case["n"], case["t"], case["c"], TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        v = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
        return v.mul_(scale).add_(shift)

    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    lengths = lengths[torch.randperm(n, generator=gen, device="cuda")].contiguous()
    s = {"case": case, "lengths": lengths}
    if case["op"].startswith("norm"):
        # Channels of an encoder differ in offset and spread.
        x = normal(n, t, c).mul_(normal(c, scale=0.2).exp_()).add_(normal(c, scale=0.5))
        s["x"] = x.to(dtype)
        s["weight"] = normal(c, scale=0.1, shift=1.0).to(dtype)
        s["bias"] = normal(c, scale=0.1).to(dtype)
        if case["op"] == "norm gradient":
            s["grad_out"] = normal(n, t, c, scale=0.1).to(dtype)
            s["mean"], s["rstd"] = _statistics(s["x"], lengths, case["groups"])
    else:
        s["x"] = normal(n, t, c).to(dtype)
        # Gates that mostly keep: a memory of a few to a few hundred frames.
        s["gate"] = normal(n, t, c, scale=1.5, shift=2.0).to(dtype)
        initial = normal(n, c)
        if case["op"] == "recurrence":
            s["initial"] = initial
        else:
            s["grad_out"] = normal(n, t, c, scale=0.1).to(dtype)
            s["grad_final"] = normal(n, c, scale=0.1)
            keep, add = _steps(s["x"], s["gate"], lengths)
            s["states"] = _saved(_scan(keep, add, initial), initial, lengths)
    return s


# ---- the plain form ---------------------------------------------------------------------------

def _valid(lengths, t):
    """[N, T, 1]: frames below the utterance's length."""
    return (torch.arange(t, device=lengths.device) < lengths[:, None])[:, :, None]


def _grouped(v, groups):
    return v.view(v.shape[0], v.shape[1], groups, -1)


def _statistics(x, lengths, groups):
    valid = _valid(lengths, x.shape[1])[..., None]
    v = _grouped(x.float(), groups)
    count = (lengths.float() * v.shape[3]).clamp(min=1.0)[:, None]
    mean = torch.where(valid, v, 0.0).sum((1, 3)) / count
    centred = torch.where(valid, v - mean[:, None, :, None], 0.0)
    var = (centred * centred).sum((1, 3)) / count
    return mean, 1.0 / torch.sqrt(var + EPS)


def _normalised(x, mean, rstd):
    """xhat [N, T, C]."""
    v = _grouped(x.float(), mean.shape[1])
    return ((v - mean[:, None, :, None]) * rstd[:, None, :, None]).view(x.shape)


def _sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _activated(z, activation):
    if activation == "silu":
        return z * _sigmoid(z)
    if activation == "swoosh_r":
        v = z - 1.0
        return v.clamp(min=0.0) + torch.log1p(torch.exp(-v.abs())) - 0.08 * z - 0.313261687
    return z


def _slope(z, activation):
    if activation == "silu":
        p = _sigmoid(z)
        return p * (1.0 + z * (1.0 - p))
    if activation == "swoosh_r":
        return _sigmoid(z - 1.0) - 0.08
    return torch.ones_like(z)


def _norm_plain(s):
    case, x = s["case"], s["x"]
    mean, rstd = _statistics(x, s["lengths"], case["groups"])
    z = _normalised(x, mean, rstd) * s["weight"].float() + s["bias"].float()
    out = torch.where(_valid(s["lengths"], x.shape[1]), _activated(z, case["activation"]), 0.0)
    return (out.to(x.dtype), mean, rstd) if case["statistics"] else out.to(x.dtype)


def _norm_gradient_plain(s):
    case, x, groups = s["case"], s["x"], s["mean"].shape[1]
    weight = s["weight"].float()
    valid = _valid(s["lengths"], x.shape[1])
    xhat = torch.where(valid, _normalised(x, s["mean"], s["rstd"]), 0.0)
    z = xhat * weight + s["bias"].float()
    dz = torch.where(valid, s["grad_out"].float() * _slope(z, case["activation"]), 0.0)
    grad_weight, grad_bias = (dz * xhat).sum((0, 1)), dz.sum((0, 1))
    dxhat = _grouped(dz * weight, groups)
    xhat = _grouped(xhat, groups)
    count = (s["lengths"].float() * xhat.shape[3]).clamp(min=1.0)[:, None]
    first = (dxhat.sum((1, 3)) / count)[:, None, :, None]
    second = ((dxhat * xhat).sum((1, 3)) / count)[:, None, :, None]
    dx = (s["rstd"][:, None, :, None] * (dxhat - first - xhat * second)).view(x.shape)
    return (torch.where(valid, dx, 0.0).to(x.dtype), grad_weight.to(x.dtype),
            grad_bias.to(x.dtype))


def _steps(x, gate, lengths):
    """h_t = keep_t h_{t-1} + add_t; a padded frame keeps the state as it is."""
    valid, g = _valid(lengths, x.shape[1]), gate.float()
    keep = torch.where(valid, 1.0 / (1.0 + torch.exp(-g)), 1.0)
    add = torch.where(valid, x.float() / (1.0 + torch.exp(g)), 0.0)
    return keep, add


def _scan(keep, add, initial):
    """All h_t at once: in step k, every frame takes in the 2^k frames before those it has."""
    step = 1
    while step < keep.shape[1]:
        add = torch.cat((add[:, :step], add[:, step:] + keep[:, step:] * add[:, :-step]), 1)
        keep = torch.cat((keep[:, :step], keep[:, step:] * keep[:, :-step]), 1)
        step *= 2
    return add + keep * initial[:, None]


def _saved(h, initial, lengths):
    """The state before every STATE_FRAMES-th frame; zero where that frame is padding."""
    t = h.shape[1]
    before = torch.cat((initial[:, None], h[:, STATE_FRAMES - 1:t - 1:STATE_FRAMES]), 1)
    return torch.where(_valid(lengths, t)[:, ::STATE_FRAMES], before, 0.0)


def _recurrence_plain(s):
    x, initial = s["x"], s["initial"]
    keep, add = _steps(x, s["gate"], s["lengths"])
    h = _scan(keep, add, initial)
    out = torch.where(_valid(s["lengths"], x.shape[1]), h, 0.0).to(x.dtype)
    if s["case"]["states"]:
        return out, h[:, -1].contiguous(), _saved(h, initial, s["lengths"])
    return out, h[:, -1].contiguous()


def _recurrence_gradient_plain(s):
    x, initial = s["x"], s["states"][:, 0]
    valid, g = _valid(s["lengths"], x.shape[1]), s["gate"].float()
    keep, add = _steps(x, s["gate"], s["lengths"])
    before = torch.cat((initial[:, None], _scan(keep, add, initial)[:, :-1]), 1)
    grad = torch.where(valid, s["grad_out"].float(), 0.0)
    keep_next = torch.cat((keep[:, 1:], torch.ones_like(keep[:, :1])), 1)
    total = _scan(keep_next.flip(1), grad.flip(1), s["grad_final"]).flip(1)
    pass_on = 1.0 / (1.0 + torch.exp(g))
    grad_x = torch.where(valid, pass_on * total, 0.0)
    grad_gate = torch.where(valid, keep * pass_on * (before - x.float()) * total, 0.0)
    return grad_x.to(x.dtype), grad_gate.to(x.dtype), keep[:, 0] * total[:, 0]


# ---- one pass ---------------------------------------------------------------------------------

def _run_own(s):
    import fast_gpu_asr_b200 as fga

    case = s["case"]
    if case["op"] == "norm":
        return fga.group_norm_activation(
            s["x"], s["lengths"], s["weight"], s["bias"], case["groups"], eps=EPS,
            activation=case["activation"], return_statistics=case["statistics"])
    if case["op"] == "norm gradient":
        return fga.group_norm_activation_backward(
            s["grad_out"], s["x"], s["lengths"], s["weight"], s["bias"], s["mean"], s["rstd"],
            activation=case["activation"])
    if case["op"] == "recurrence":
        return fga.gated_linear_recurrence(s["x"], s["gate"], s["lengths"], s["initial"],
                                           return_states=case["states"])
    return fga.gated_linear_recurrence_backward(s["grad_out"], s["x"], s["gate"], s["lengths"],
                                                s["states"], s["grad_final"])


def run(state):
    if own:
        return _run_own(state)
    plain = {"norm": _norm_plain, "norm gradient": _norm_gradient_plain,
             "recurrence": _recurrence_plain, "recurrence gradient": _recurrence_gradient_plain}
    return plain[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    n, t, c = case["n"], case["t"], case["c"]
    size = TYPES[case["dtype"]].itemsize
    lengths = _lengths(case)
    valid, every = sum(lengths) * c, n * t * c
    saved = 4 * c * sum(_chunks(m) for m in lengths)
    if case["op"] == "norm":
        b = size * (valid + every + 2 * c) + 4 * n + (8 * n * case["groups"] if case["statistics"]
                                                      else 0)
        return {"bytes": b, "flops": 16 * valid}
    if case["op"] == "norm gradient":
        b = size * (2 * valid + every + 4 * c) + 4 * n + 8 * n * case["groups"]
        return {"bytes": b, "flops": 30 * valid}
    if case["op"] == "recurrence":
        b = size * (2 * valid + every) + 4 * n + 8 * n * c
        return {"bytes": b + (4 * n * c * _chunks(t) if case["states"] else 0), "flops": 8 * valid}
    return {"bytes": size * (3 * valid + 2 * every) + 4 * n + 8 * n * c + saved,
            "flops": 16 * valid}


# ---- the definition in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _norm_exact, "norm gradient": _norm_gradient_exact,
            "recurrence": _recurrence_exact,
            "recurrence gradient": _recurrence_gradient_exact}[case["op"]](s)


def _act_exact(z, activation):
    """(value, derivative)."""
    if activation == "silu":
        p = torch.special.expit(z)
        return z * p, p + z * p * torch.special.expit(-z)
    if activation == "swoosh_r":
        value = torch.logaddexp(z - 1.0, torch.zeros_like(z)) - 0.08 * z - 0.313261687
        return value, torch.special.expit(z - 1.0) - 0.08
    return z, torch.ones_like(z)


def _norm_exact(s):
    case = s["case"]
    n, t, c, g = case["n"], case["t"], case["c"], case["groups"]
    out = torch.zeros(n, t, c, dtype=torch.float64, device="cuda")
    mean, rstd = (torch.zeros(n, g, dtype=torch.float64, device="cuda") for _ in range(2))
    w, b = s["weight"].double(), s["bias"].double()
    for i, m in enumerate(s["lengths"].tolist()):
        v = s["x"][i, :m].double().view(m, g, c // g)
        var, mu = torch.var_mean(v, dim=(0, 2), correction=0)
        mean[i], rstd[i] = mu, (var + EPS) ** -0.5
        xhat = (v - mu[:, None]) * rstd[i][:, None]
        out[i, :m] = _act_exact(xhat.reshape(m, c) * w + b, case["activation"])[0]
    return (out, mean, rstd) if case["statistics"] else out


def _norm_gradient_exact(s):
    case = s["case"]
    n, t, c, g = case["n"], case["t"], case["c"], case["groups"]
    dx = torch.zeros(n, t, c, dtype=torch.float64, device="cuda")
    w, b = s["weight"].double(), s["bias"].double()
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for i, m in enumerate(s["lengths"].tolist()):
        mu, r = s["mean"][i].double()[:, None], s["rstd"][i].double()[:, None]
        xhat = (s["x"][i, :m].double().view(m, g, c // g) - mu) * r
        slope = _act_exact(xhat.reshape(m, c) * w + b, case["activation"])[1]
        dz = s["grad_out"][i, :m].double() * slope
        dw += (dz * xhat.reshape(m, c)).sum(0)
        db += dz.sum(0)
        d = (dz * w).view(m, g, c // g)
        first = d.mean((0, 2))[:, None]
        second = (d * xhat).mean((0, 2))[:, None]
        dx[i, :m] = ((d - first - xhat * second) * r).reshape(m, c)
    return dx, dw, db


def _recurrence_exact(s):
    case, x, lengths = s["case"], s["x"].double(), s["lengths"][:, None]
    f, h = torch.special.expit(s["gate"].double()), s["initial"].double()
    out = torch.zeros_like(x)
    states = torch.zeros(x.shape[0], _chunks(x.shape[1]), x.shape[2], dtype=torch.float64,
                         device="cuda")
    for i in range(x.shape[1]):
        live = i < lengths
        if i % STATE_FRAMES == 0:
            states[:, i // STATE_FRAMES] = h * live
        h = torch.where(live, torch.lerp(x[:, i], h, f[:, i]), h)
        out[:, i] = h * live
    return (out, h, states) if case["states"] else (out, h)


def _recurrence_gradient_exact(s):
    x, grad, lengths = s["x"].double(), s["grad_out"].double(), s["lengths"][:, None]
    f, p = torch.special.expit(s["gate"].double()), torch.special.expit(-s["gate"].double())
    h = s["states"][:, 0].double()
    away = torch.empty_like(x)  # h_{t-1} - x_t
    for i in range(x.shape[1]):
        away[:, i] = h - x[:, i]
        h = torch.where(i < lengths, x[:, i] + f[:, i] * away[:, i], h)
    grad_x, grad_gate = torch.zeros_like(x), torch.zeros_like(x)
    carry = s["grad_final"].double()
    for i in reversed(range(x.shape[1])):
        live = i < lengths
        total = grad[:, i] + carry
        grad_x[:, i] = p[:, i] * total * live
        grad_gate[:, i] = f[:, i] * p[:, i] * away[:, i] * total * live
        carry = torch.where(live, f[:, i] * total, carry)
    return grad_x, grad_gate, carry
