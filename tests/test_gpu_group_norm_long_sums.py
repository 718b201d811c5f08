"""GPU tests of group norm where a thread adds up the most rows that a launch gives it, with bounds
from what is really added in a row.

Streams give a thread up to 64 rows. In a group of whole vectors each adds the four pairs of its
eight 16-bit values to one sum: 256 additions, one more for the pair's halves, then up to 8
entries and 5 steps across a warp for the block, and as much again for the blocks: below
``LONGEST = 288``. What is added are differences from the thread's first values, at most 2
max|x| each, where the shared bounds take max|x|: twice that. Rows on chip are fewer, at most 23 a
thread (129 vectors a row leave 127 of 256 threads idle, and 48 KB hold 23 such rows). Parameters'
gradients pass a thread's rows one by one (64) and then every 32nd block row of the batch and 5
steps across threads.

The exponentials and reciprocals behind the shared bounds are ``ex2.approx``, ``lg2.approx`` and
``rcp.approx``: 2 steps of fp32, 2^-22 absolute next to 1, and 1 step, after the rounding of an
argument that is a product with log2 e."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import sequence_cases as cases
from fast_gpu_asr_b200 import group_norm_activation, group_norm_activation_backward
from oracle import sequence_oracle as oracle

pytestmark = pytest.mark.gpu

LONGEST = 288
U = cases.U


def problem(n, t, c, dtype, outlier):
    """On the GPU: x, weight, bias, grad_out and lengths of which every third is full. With
    `outlier` every utterance's first frame, and so each first block's pivots, lie 30 away."""
    gen = torch.Generator("cuda").manual_seed(n + t + c)
    dt = getattr(torch, dtype)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    x = normal(n, t, c) * (normal(c) * 0.2).exp() + normal(c) * 0.5
    if outlier:
        x[:, 0] += 30.0
    w, b = normal(c) * 0.1 + 1, normal(c) * 0.1
    lens = torch.randint(1, t + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)
    lens[::3] = t
    return x.to(dt), w.to(dt), b.to(dt), normal(n, t, c).to(dt), lens


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("outlier", [False, True])
@pytest.mark.parametrize("n,t,c,rows", [(296, 256, 2048, 64), (300, 23, 1032, 23)])
def test_statistics_of_the_longest_sums(n, t, c, rows, outlier, dtype, monkeypatch):
    """With an outlier in its first vector a thread's squares about it are up to (1 + rows) times
    those about the mean, and so is their rounding error."""
    monkeypatch.setattr(cases, "CHAIN", 2 * LONGEST * (1 + rows if outlier else 1))
    x, w, b, _, lens = problem(n, t, c, dtype, outlier)
    got = group_norm_activation(x, lens, w, b, 1, return_statistics=True)
    some = [0, 1, n // 2, n - 1]  # the oracle takes the utterances one by one
    hx, hw, hb = cases.host(x[some]), cases.host(w), cases.host(b)
    lengths = lens[some].cpu().numpy()
    want = oracle.group_norm_activation(hx, lengths, hw, hb, 1, float(np.float32(1e-5)))
    bounds = cases.norm_bounds(hx, lengths, hw, hb, 1, want[1], want[2], want[0], dtype)
    for v, e, bound, what in zip(got, want, bounds, ("out", "mean", "rstd")):
        cases.assert_within(cases.host(v[some]), e, bound, what)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_gradients_of_the_longest_sums(dtype, monkeypatch):
    n, t, c = 1200, 64, 2048
    monkeypatch.setattr(cases, "CHAIN", LONGEST)
    x, w, b, dout, lens = problem(n, t, c, dtype, False)
    _, mean, rstd = group_norm_activation(x, lens, w, b, 1, return_statistics=True)
    grads = group_norm_activation_backward(dout, x, lens, w, b, mean, rstd)

    some = [0, 1, n // 2, n - 1]
    hx, hw, hb, hd = (cases.host(v) for v in (x[some], w, b, dout[some]))
    lengths, mu, r = lens[some].cpu().numpy(), cases.host(mean[some]), cases.host(rstd[some])
    want = oracle.group_norm_activation_backward(hd, hx, lengths, hw, hb, mu, r)
    bound = cases.norm_gradient_bounds(hd, hx, lengths, hw, hb, mu, r, want, "silu", dtype)[0]
    cases.assert_within(cases.host(grads[0][some]), want[0], bound, "grad_x")

    # The parameters' sums over the whole batch, and of what each term is off by (as in
    # norm_gradient_bounds), in float64 on the GPU.
    w, b = w.double(), b.double()
    sums = torch.zeros(6, c, dtype=torch.float64, device="cuda")
    for i, m in enumerate(lens.tolist()):
        xhat = (x[i, :m].double() - mean[i].double()) * rstd[i].double()
        d, z = dout[i, :m].double(), xhat * w + b
        s = torch.sigmoid(z)
        dz = d * s * (1 + z * (1 - s))
        e = d.abs() * (20 * U + 3 * U * ((w * xhat).abs() + b.abs()))
        for k, v in enumerate((dz * xhat, dz, (dz * xhat).abs(), dz.abs(), e * xhat.abs(), e)):
            sums[k] += v.sum(0)
    gw, gb, aw, ab, ew, eb = sums.cpu().numpy()
    chain = 64 + -(-n // 32) + 5
    for got, want, size, off, what in ((grads[1], gw, aw, ew, "grad_weight"),
                                       (grads[2], gb, ab, eb, "grad_bias")):
        bound = off + (chain + 4) * U * size
        bound = bound + cases.HALF[dtype] * (np.abs(want) + bound) + cases.TINY[dtype]
        cases.assert_within(cases.host(got), want, bound, what)
