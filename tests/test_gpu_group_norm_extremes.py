"""Group norm with activation where parameters are NaN, infinite or next to the type's largest
number: what comes out is what the formulas give, in every activation, type and way of launching.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import sequence_cases as cases
from fast_gpu_asr_b200 import group_norm_activation, group_norm_activation_backward
from oracle import sequence_oracle as oracle

pytestmark = pytest.mark.gpu

ACTIVATIONS = ("none", "silu", "swoosh_r")
# Vectors of one group, of several, rows that start anywhere, clusters, streams of both kinds, a
# group wider than a block.
SHAPES = [(2, 40, 48, 6), (2, 29, 30, 2), (3, 33, 35, 5), (2, 700, 256, 2), (1, 12000, 40, 5),
          (1, 9000, 67, 1), (1, 300, 4104, 1), (1, 17000, 24, 2)]


def inputs(n, t, c, dtype, seed):
    x, w, b, dout = cases.norm_inputs(n, t, c, dtype, seed)
    return x, np.array([t] * (n - 1) + [max(1, t // 2)], np.int32), w, b, dout


def call(x, lengths, w, b, dout, groups, activation, dtype):
    """((out, mean, rstd), gradients) of the kernels."""
    gx, gw, gb, gd = (cases.to_cuda(v, dtype) for v in (x, w, b, dout))
    lens = torch.from_numpy(lengths).cuda()
    got = group_norm_activation(gx, lens, gw, gb, groups, activation=activation,
                                return_statistics=True)
    return got, group_norm_activation_backward(gd, gx, lens, gw, gb, *got[1:],
                                               activation=activation)


def formulas(x, lengths, w, b, dout, groups, activation, got):
    with np.errstate(all="ignore"):
        out = oracle.group_norm_activation(x, lengths, w, b, groups, 1e-5, activation)
        grads = oracle.group_norm_activation_backward(
            dout, x, lengths, w, b, cases.host(got[1]), cases.host(got[2]), activation)
    return out, grads


def assert_same_kind(got, want, what):
    """NaN where the formula has one, infinite where it is, finite elsewhere."""
    got = cases.host(got)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, "NaN")
    assert np.array_equal(np.where(np.isinf(got), got, 0), np.where(np.isinf(want), want, 0)), (
        what, "inf")


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("n,t,c,groups", SHAPES)
@pytest.mark.parametrize("which", ["weight", "bias"])
def test_a_nan_parameter_shows(which, n, t, c, groups, activation, dtype):
    """NaN in its channel's out and parameters' gradients and throughout its group's grad_x
    (without an activation, whose slope does not see the bias, only in what the formula has it)."""
    x, lengths, w, b, dout = inputs(n, t, c, dtype, 3)
    at = c // 2
    (w if which == "weight" else b)[at] = np.nan
    got, grads = call(x, lengths, w, b, dout, groups, activation, dtype)
    want, want_grads = formulas(x, lengths, w, b, dout, groups, activation, got)
    valid = slice(0, lengths[0])
    assert np.isnan(want[0][0, valid, at]).all()
    if activation != "none":
        width = c // groups
        group = slice(at // width * width, at // width * width + width)
        assert np.isnan(want_grads[0][0, valid, group]).all()
        assert np.isnan(want_grads[1][at]) and np.isnan(want_grads[2][at])
    for v, e, what in zip((got[0], *grads), (want[0], *want_grads),
                          ("out", "grad_x", "grad_weight", "grad_bias")):
        assert_same_kind(v, e, what)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("n,t,c,groups", SHAPES[:5])
def test_infinite_biases(n, t, c, groups, activation, dtype):
    """As the formulas have it: SiLU is inf and NaN at the two infinities, Swoosh-R NaN and inf;
    the slopes are NaN for SiLU, and 0.92 and -0.08 for Swoosh-R."""
    for value in (np.inf, -np.inf):
        x, lengths, w, b, dout = inputs(n, t, c, dtype, 4)
        b[c // 2] = value
        got, grads = call(x, lengths, w, b, dout, groups, activation, dtype)
        want, want_grads = formulas(x, lengths, w, b, dout, groups, activation, got)
        for v, e, what in zip((got[0], *grads), (want[0], *want_grads),
                              ("out", "grad_x", "grad_weight", "grad_bias")):
            assert_same_kind(v, e, (what, value))


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("n,t,c,groups", SHAPES)
def test_biases_up_to_the_largest(n, t, c, groups, activation, dtype):
    """Biases of the type's largest and lowest numbers and of steps towards them, in some
    channels, next to ordinary ones.

    out is off by a rounding of z = w xhat + b (2 U |b|), the slope's rounding (the formula's
    0.92 is fp32: 3 U) and the store's. For the gradients such a bias is one of +-120, at which
    the slopes are already what they are at infinity to within exp(-119) (1 + 120) < 2^-160, as
    long as |w xhat| stays below 20; so that is what the bounds are taken from."""
    x, lengths, w, b, dout = inputs(n, t, c, dtype, 5)
    most = torch.finfo(getattr(torch, dtype)).max
    channels = np.linspace(0, c - 1, 6).astype(int)
    steps = most * np.array([1.0, -1.0, 0.75, -0.75, 0.4375, -0.4375])
    ordinary = b.copy()
    b[channels] = cases.store(steps, dtype)
    ordinary[channels] = np.sign(steps) * 120.0
    got, grads = call(x, lengths, w, b, dout, groups, activation, dtype)
    want, _ = formulas(x, lengths, w, b, dout, groups, activation, got)
    _, want_grads = formulas(x, lengths, w, ordinary, dout, groups, activation, got)
    bounds = cases.norm_bounds(x, lengths, w, b, groups, want[1], want[2], want[0], dtype)
    for v, e, bound, what in zip(got, want, bounds, ("out", "mean", "rstd")):
        cases.assert_within(cases.host(v), e, bound, what)
    bounds = cases.norm_gradient_bounds(dout, x, lengths, w, ordinary, cases.host(got[1]),
                                        cases.host(got[2]), want_grads, activation, dtype)
    for v, e, bound, what in zip(grads, want_grads, bounds, ("grad_x", "grad_weight", "grad_bias")):
        cases.assert_within(cases.host(v), e, bound, what)
