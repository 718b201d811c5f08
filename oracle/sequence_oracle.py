"""Group norm with an activation and the gated linear recurrence in float64, from their
formulas, with the gradients (test infrastructure only). No reference plugin.

Arrays are ``[N, T, C]``; ``lengths`` are clamped to ``[0, T]`` and padded frames are neither
read nor anything but zero in an output.
"""

from __future__ import annotations

import numpy as np

STATE_FRAMES = 64


def _lengths(lengths, t):
    return np.clip(np.asarray(lengths, np.int64), 0, t)


def sigmoid(v):
    e = np.exp(-np.abs(v))
    return np.where(v < 0, e, 1.0) / (1.0 + e)


def activate(z, activation):
    if activation == "silu":
        return z * sigmoid(z)
    if activation == "swoosh_r":
        return np.logaddexp(z - 1.0, 0.0) - 0.08 * z - 0.313261687
    return z.copy()


def slope(z, activation):
    if activation == "silu":
        return sigmoid(z) * (1.0 + z * sigmoid(-z))
    if activation == "swoosh_r":
        return sigmoid(z - 1.0) - 0.08
    return np.ones_like(z)


def group_norm_activation(x, lengths, weight, bias, groups, eps=1e-5, activation="silu"):
    """(out, mean, rstd)."""
    x, weight, bias = (np.asarray(v, np.float64) for v in (x, weight, bias))
    n, t, c = x.shape
    out = np.zeros_like(x)
    mean, rstd = np.zeros((n, groups)), np.full((n, groups), float(eps) ** -0.5)
    for i, m in enumerate(_lengths(lengths, t)):
        if m == 0:
            continue
        v = x[i, :m].reshape(m, groups, c // groups)
        mean[i] = v.mean((0, 2))
        centred = v - mean[i][:, None]
        rstd[i] = ((centred * centred).mean((0, 2)) + eps) ** -0.5
        xhat = (centred * rstd[i][:, None]).reshape(m, c)
        out[i, :m] = activate(xhat * weight + bias, activation)
    return out, mean, rstd


def group_norm_activation_backward(grad_out, x, lengths, weight, bias, mean, rstd,
                                   activation="silu"):
    """(grad_x, grad_weight, grad_bias)."""
    grad_out, x, weight, bias, mean, rstd = (
        np.asarray(v, np.float64) for v in (grad_out, x, weight, bias, mean, rstd))
    n, t, c = x.shape
    groups = mean.shape[1]
    grad_x, grad_weight, grad_bias = np.zeros_like(x), np.zeros(c), np.zeros(c)
    for i, m in enumerate(_lengths(lengths, t)):
        if m == 0:
            continue
        xhat = (x[i, :m].reshape(m, groups, -1) - mean[i][:, None]) * rstd[i][:, None]
        flat = xhat.reshape(m, c)
        dz = grad_out[i, :m] * slope(flat * weight + bias, activation)
        grad_weight += (dz * flat).sum(0)
        grad_bias += dz.sum(0)
        d = (dz * weight).reshape(m, groups, -1)
        first, second = d.mean((0, 2))[:, None], (d * xhat).mean((0, 2))[:, None]
        grad_x[i, :m] = ((d - first - xhat * second) * rstd[i][:, None]).reshape(m, c)
    return grad_x, grad_weight, grad_bias


def gated_linear_recurrence(x, gate, lengths, initial=None):
    """(out, final, states)."""
    x, gate = np.asarray(x, np.float64), np.asarray(gate, np.float64)
    n, t, c = x.shape
    out, states = np.zeros_like(x), np.zeros((n, -(-t // STATE_FRAMES), c))
    h = np.zeros((n, c)) if initial is None else np.asarray(initial, np.float64).copy()
    for i, m in enumerate(_lengths(lengths, t)):
        for j in range(m):
            if j % STATE_FRAMES == 0:
                states[i, j // STATE_FRAMES] = h[i]
            h[i] = sigmoid(gate[i, j]) * h[i] + sigmoid(-gate[i, j]) * x[i, j]
            out[i, j] = h[i]
    return out, h, states


def gated_linear_recurrence_backward(grad_out, x, gate, lengths, initial, grad_final=None):
    """(grad_x, grad_gate, grad_initial)."""
    grad_out, x, gate = (np.asarray(v, np.float64) for v in (grad_out, x, gate))
    n, t, c = x.shape
    before = np.zeros((n, c)) if initial is None else np.asarray(initial, np.float64)
    out, _, _ = gated_linear_recurrence(x, gate, lengths, before)
    carry = np.zeros((n, c)) if grad_final is None else np.asarray(grad_final, np.float64).copy()
    grad_x, grad_gate = np.zeros_like(x), np.zeros_like(x)
    for i, m in enumerate(_lengths(lengths, t)):
        for j in reversed(range(m)):
            f, p = sigmoid(gate[i, j]), sigmoid(-gate[i, j])
            total = grad_out[i, j] + carry[i]
            grad_x[i, j] = p * total
            grad_gate[i, j] = f * p * ((out[i, j - 1] if j else before[i]) - x[i, j]) * total
            carry[i] = f * total
    return grad_x, grad_gate, carry
