"""Inputs and error bounds of the group-norm and recurrence tests.

The bounds count roundings. ``U`` is half a step of fp32 (2^-24, the relative error of one
operation), ``HALF[t]`` that of the storage type. CUDA's ``__expf`` and fast division are
within a few steps of fp32 plus the rounding of the argument, whose effect grows with the
argument: ``(4 + |v|) 2 U`` relative is what the bounds below grant an exponential of v. A sum
through a chain of d additions is off by at most ``d U`` times the sum of magnitudes.
"""

from __future__ import annotations

import numpy as np
import torch

from oracle import sequence_oracle as oracle

U = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -133}
DTYPES = ("float32", "float16", "bfloat16")
INT32_MIN, INT32_MAX = np.iinfo(np.int32).min, np.iinfo(np.int32).max
# Additions that one value passes on its way into a sum: what a thread adds up serially (at
# most 16 vectors of 8), a block's and a cluster's trees, and the chunks of a long axis.
CHAIN = 256


def store(v, dtype):
    """float64 of ``v`` rounded to the storage type."""
    t = torch.from_numpy(np.ascontiguousarray(v, dtype=np.float32))
    return t.to(getattr(torch, dtype)).double().numpy()


def to_cuda(v, dtype):
    return torch.from_numpy(np.ascontiguousarray(v, dtype=np.float32)).to(
        "cuda", getattr(torch, dtype))


def host(t):
    return t.detach().double().cpu().numpy()


def mixed_lengths(n, t, seed):
    """Full, empty and clamped utterances among random ones."""
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, t + 1, n).astype(np.int64)
    special = (t, 0, INT32_MAX, INT32_MIN, 1)
    for i in range(n):
        if i % 2 == 0:
            lengths[i] = special[i // 2 % len(special)]
    return lengths.astype(np.int32)


def poison(v, lengths, value=np.nan):
    """Padded frames that must not be read."""
    v = v.copy()
    for i, m in enumerate(np.clip(np.asarray(lengths, np.int64), 0, v.shape[1])):
        v[i, m:] = value
    return v


def assert_within(got, expected, bound, what=""):
    got, expected = np.asarray(got, np.float64), np.asarray(expected, np.float64)
    assert got.shape == expected.shape, (what, got.shape, expected.shape)
    bad = ~(np.abs(got - expected) <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4],
                           expected[bad][:4], np.broadcast_to(bound, got.shape)[bad][:4])


# ---- group norm -------------------------------------------------------------------------------

def norm_inputs(n, t, c, dtype, seed, offset=0.5):
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 1, (n, t, c)) * np.exp(rng.normal(0, 0.2, c)) + rng.normal(0, offset, c)
    w, b = rng.normal(1, 0.1, c), rng.normal(0, 0.1, c)
    return store(x, dtype), store(w, dtype), store(b, dtype), store(rng.normal(0, 1, (n, t, c)),
                                                                   dtype)


def _per_channel(stat, c):
    """[N, G] -> [N, 1, C]."""
    return np.repeat(stat, c // stat.shape[1], axis=1)[:, None, :]


def _largest(x, lengths, groups):
    """max |x| over each group's valid frames, [N, G]."""
    n, t, c = x.shape
    big = np.zeros((n, groups))
    for i, m in enumerate(np.clip(np.asarray(lengths, np.int64), 0, t)):
        if m:
            big[i] = np.abs(x[i, :m]).reshape(m, groups, -1).max((0, 2))
    return big


def norm_bounds(x, lengths, w, b, groups, mean, rstd, out, dtype):
    """Bounds of (out, mean, rstd).

    mean: CHAIN U max|x|. The variance sums squares of x - mean (each off by 3 U) and takes
    the squared error of the mean on top: rstd is off by half of (CHAIN + 8) U, plus
    (rstd dmean)^2 / 2, relative (both granted whole). z = (x - mean) rstd w + b then carries
    w rstd dmean + |w xhat| (drstd + 4 U) + 2 U (|z| + |b|); the activations have slopes of at
    most 1.1 and are evaluated to 16 U (1 + |z|); one rounding to the storage type."""
    c = x.shape[2]
    dmean = CHAIN * U * _largest(x, lengths, groups)
    drstd = (CHAIN + 8) * U + (rstd * dmean) ** 2
    valid = np.arange(x.shape[1])[None, :, None] < np.clip(
        np.asarray(lengths, np.int64), 0, x.shape[1])[:, None, None]
    xhat = np.where(valid, (np.where(valid, x, 0) - _per_channel(mean, c)) * _per_channel(rstd, c), 0)
    z = xhat * w + b
    dz = (np.abs(w) * _per_channel(rstd * dmean, c)
          + np.abs(w * xhat) * (_per_channel(drstd, c) + 4 * U) + 2 * U * (np.abs(z) + np.abs(b)))
    value = 1.1 * dz + 16 * U * (1 + np.abs(z))
    value = value + HALF[dtype] * (np.abs(out) + value) + TINY[dtype]
    return np.where(valid, value, 0.0), dmean, rstd * drstd


def norm_gradient_bounds(dout, x, lengths, w, b, mean, rstd, grads, activation, dtype):
    """Bounds of (grad_x, grad_weight, grad_bias).

    xhat is off by 3 U |xhat| and z by 6 U (|w xhat| + |b|); the slopes change by at most 0.5
    per unit of z and are evaluated to 16 U. So dz is off by e = |dout| (20 U + 3 U (|w xhat|
    + |b|)). The sums add CHAIN U of their magnitudes (four times that over a whole batch,
    which the parameters' gradients pass through), the last formula four roundings."""
    n, t, c = x.shape
    groups = mean.shape[1]
    valid = np.arange(t)[None, :, None] < np.clip(np.asarray(lengths, np.int64), 0, t)[:, None, None]
    r = _per_channel(rstd, c)
    xhat = np.where(valid, (np.where(valid, x, 0) - _per_channel(mean, c)) * r, 0)
    dout = np.where(valid, dout, 0)
    dz = np.abs(dout * oracle.slope(xhat * w + b, activation))
    e = np.abs(dout) * (20 * U + 3 * U * (np.abs(w * xhat) + np.abs(b)))
    count = np.maximum(np.clip(np.asarray(lengths, np.int64), 0, t) * (c // groups), 1)[:, None]

    def mean_of(v):
        return _per_channel(v.reshape(n, t, groups, -1).sum((1, 3)) / count, c)

    a, ax, aw = np.abs(w) * dz, np.abs(xhat), np.abs(w) * e
    ds1 = mean_of(aw) + (CHAIN + 4) * U * mean_of(a)
    ds2 = mean_of(aw * ax) + (CHAIN + 8) * U * mean_of(a * ax)
    gx = r * (aw + ds1 + ax * ds2 + 6 * U * (a + mean_of(a) + ax * mean_of(a * ax)))
    gx = gx + HALF[dtype] * (np.abs(grads[0]) + gx) + TINY[dtype]
    gw = (e * ax).sum((0, 1)) + (4 * CHAIN + 4) * U * (dz * ax).sum((0, 1))
    gb = e.sum((0, 1)) + 4 * CHAIN * U * dz.sum((0, 1))
    return (np.where(valid, gx, 0.0), gw + HALF[dtype] * (np.abs(grads[1]) + gw) + TINY[dtype],
            gb + HALF[dtype] * (np.abs(grads[2]) + gb) + TINY[dtype])


# ---- recurrence -------------------------------------------------------------------------------

def recurrence_inputs(n, t, c, dtype, seed):
    rng = np.random.default_rng(seed)
    x, gate = rng.normal(0, 1, (n, t, c)), rng.normal(1.5, 2.0, (n, t, c))
    dout = rng.normal(0, 1, (n, t, c))
    initial, dfinal = rng.normal(0, 1, (n, c)), rng.normal(0, 1, (n, c))
    return (*(store(v, dtype) for v in (x, gate, dout)),
            *(store(v, "float32") for v in (initial, dfinal)))


def recurrence_errors(x, gate, lengths, initial, out):
    """Error of h after every frame, [N, T, C], and of the final state, [N, C].

    A frame takes h to f h + p x with p off by (8 + 2|gate|) U relative, f by the same
    amount absolutely, and some roundings of values no larger than the larger of |h| and |x|,
    which a frame meets once in its own chunk and once more for each product of a chunk's f:
    8 U of it. Errors of earlier frames shrink by f like the state."""
    n, t, c = x.shape
    before = np.zeros((n, c)) if initial is None else initial
    error, e = np.zeros((n, t, c)), np.zeros((n, c))
    for i in range(t):
        live = (i < np.asarray(lengths, np.int64))[:, None]
        f, p, g = oracle.sigmoid(gate[:, i]), oracle.sigmoid(-gate[:, i]), np.abs(gate[:, i])
        h, hx = np.abs(before), np.abs(x[:, i])
        step = f * e + U * ((8 + 2 * g) * p * (h + hx) + 8 * np.maximum(h, hx))
        e = np.where(live, step, e)
        error[:, i] = np.where(live, e, 0.0)
        before = np.where(live, out[:, i], before)
    return error, e


def recurrence_bounds(x, gate, lengths, initial, expected, dtype):
    """Bounds of (out, final, states)."""
    out, _, states = expected
    error, final = recurrence_errors(x, gate, lengths, initial, out)
    saved = np.zeros_like(states)
    for j in range(1, states.shape[1]):
        saved[:, j] = error[:, j * oracle.STATE_FRAMES - 1]
    return error + HALF[dtype] * (np.abs(out) + error) + TINY[dtype] * (error > 0), final, saved


def recurrence_gradient_bounds(dout, x, gate, lengths, initial, dfinal, out, grads, dtype):
    """Bounds of (grad_x, grad_gate, grad_initial): the same walk backwards for the carry f G,
    then one product each; h[t-1] is off as in the forward call."""
    n, t, c = x.shape
    before0 = np.zeros((n, c)) if initial is None else initial
    error, _ = recurrence_errors(x, gate, lengths, initial, out)
    carry = np.zeros((n, c)) if dfinal is None else dfinal.copy()
    e = np.zeros((n, c))
    bx, bg = np.zeros_like(x), np.zeros_like(x)
    for i in reversed(range(t)):
        live = (i < np.asarray(lengths, np.int64))[:, None]
        f, p, g = oracle.sigmoid(gate[:, i]), oracle.sigmoid(-gate[:, i]), np.abs(gate[:, i])
        before = out[:, i - 1] if i else before0
        eh = error[:, i - 1] if i else 0.0
        total = np.abs(dout[:, i] + carry)
        largest = np.maximum(np.abs(dout[:, i]), np.abs(carry))
        dt = e + 4 * U * largest
        away = np.abs(before - x[:, i])
        bx[:, i] = np.where(live, p * dt + p * total * (8 + 2 * g) * U, 0.0)
        bg[:, i] = np.where(live, f * p * (away * dt + total * (
            eh + 2 * U * (np.abs(before) + np.abs(x[:, i])) + away * (16 + 4 * g) * U)), 0.0)
        e = np.where(live, f * dt + total * U * ((8 + 2 * g) * p + 8 * f), e)
        carry = np.where(live, f * (dout[:, i] + carry), carry)
    tiny = TINY[dtype]
    bx = bx + HALF[dtype] * (np.abs(grads[0]) + bx) + tiny * (bx > 0)
    bg = bg + HALF[dtype] * (np.abs(grads[1]) + bg) + tiny * (bx > 0)
    return bx, bg, e
