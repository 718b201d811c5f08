"""GPU tests of group norm with activation, forward and backward, against the float64 oracle.

The bounds count roundings (``sequence_cases``). Shapes cover one frame to long axes, group
sizes from one channel to all of them, odd channel counts, and every way a launch splits an
utterance; padded frames hold NaN, which no output may show."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import sequence_cases as cases
from fast_gpu_asr_b200 import (_lib, group_norm_activation, group_norm_activation_backward,
                               normalization)
from oracle import sequence_oracle as oracle

pytestmark = pytest.mark.gpu

ACTIVATIONS = ("none", "silu", "swoosh_r")


def lengths_on_gpu(lengths):
    return torch.from_numpy(np.asarray(lengths, np.int32)).cuda()


def check(n, t, c, groups, dtype, activation, lengths=None, offset=0.5, seed=None):
    """One forward and one backward call, every element against the oracle."""
    seed = 7 * n + 11 * t + 13 * c + groups if seed is None else seed
    x, w, b, dout = cases.norm_inputs(n, t, c, dtype, seed, offset)
    lengths = cases.mixed_lengths(n, t, seed) if lengths is None else np.asarray(lengths, np.int32)
    gpu = [cases.to_cuda(v, dtype) for v in (cases.poison(x, lengths), w, b,
                                             cases.poison(dout, lengths))]
    lens = lengths_on_gpu(lengths)
    out, mean, rstd = group_norm_activation(gpu[0], lens, gpu[1], gpu[2], groups,
                                            activation=activation, return_statistics=True)
    expected = oracle.group_norm_activation(x, lengths, w, b, groups, float(np.float32(1e-5)),
                                            activation)
    bounds = cases.norm_bounds(x, lengths, w, b, groups, expected[1], expected[2], expected[0],
                               dtype)
    for got, want, bound, what in zip((out, mean, rstd), expected, bounds, ("out", "mean", "rstd")):
        cases.assert_within(cases.host(got), want, bound, (what, n, t, c, groups, dtype))
    assert out.dtype == gpu[0].dtype and mean.dtype == rstd.dtype == torch.float32
    alone = group_norm_activation(gpu[0], lens, gpu[1], gpu[2], groups, activation=activation)
    assert torch.equal(alone, out)

    grads = group_norm_activation_backward(gpu[3], gpu[0], lens, gpu[1], gpu[2], mean, rstd,
                                           activation=activation)
    mu, r = cases.host(mean), cases.host(rstd)
    want = oracle.group_norm_activation_backward(dout, x, lengths, w, b, mu, r, activation)
    bounds = cases.norm_gradient_bounds(dout, x, lengths, w, b, mu, r, want, activation, dtype)
    for got, e, bound, what in zip(grads, want, bounds, ("grad_x", "grad_weight", "grad_bias")):
        cases.assert_within(cases.host(got), e, bound, (what, n, t, c, groups, dtype))
        assert got.dtype == gpu[0].dtype


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("n,t,c,groups", [
    (1, 1, 16, 2), (2, 3, 8, 1), (5, 17, 24, 3), (4, 65, 64, 64), (3, 37, 80, 8)])
def test_small(n, t, c, groups, activation, dtype):
    check(n, t, c, groups, dtype, activation)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("n,t,c,groups", [
    (2, 33, 1, 1), (2, 40, 3, 3), (2, 29, 7, 1), (3, 50, 30, 2), (2, 31, 130, 10),
    (2, 20, 323, 19), (2, 45, 129, 1), (1, 9, 2050, 2), (2, 21, 96, 32)])
def test_odd_channels(n, t, c, groups, dtype):
    check(n, t, c, groups, dtype, "silu")


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("n,t,c,groups", [
    (2, 375, 1024, 32), (2, 375, 1024, 1), (3, 750, 192, 6), (2, 188, 384, 384),
    (1, 1500, 512, 32), (2, 1000, 64, 1), (1, 3000, 256, 2), (1, 5000, 96, 3),
    (1, 700, 4104, 1), (1, 12000, 40, 5)])
def test_every_split(n, t, c, groups, dtype):
    check(n, t, c, groups, dtype, "swoosh_r" if c % 3 else "silu",
          lengths=[t] if n == 1 else None)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_many_rows(dtype):
    check(150, 12, 64, 4, dtype, "silu")
    check(600, 1, 32, 4, dtype, "none", lengths=[1] * 600)


def test_offset_far_above_the_spread():
    """Means hundreds of times the spread: the variance is taken about the mean."""
    check(3, 300, 64, 4, "float32", "silu", lengths=[300, 211, 1], offset=300.0)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_constant_groups_and_extremes(dtype):
    """A variance of zero, and values at which exponentials overflow."""
    lens = lengths_on_gpu([5])
    x = torch.full((1, 5, 8), 3.0, device="cuda", dtype=getattr(torch, dtype))
    w, b = torch.ones(8, device="cuda", dtype=x.dtype), torch.zeros(8, device="cuda", dtype=x.dtype)
    out, mean, rstd = group_norm_activation(x, lens, w, b, 2, activation="none",
                                            return_statistics=True)
    assert torch.equal(out, torch.zeros_like(out)) and torch.all(mean == 3.0)
    np.testing.assert_allclose(rstd.cpu().numpy(), 1e-5 ** -0.5, rtol=1e-6)
    b = torch.tensor([-1000.0, -90.0, -50.0, -1.0, 1.0, 50.0, 90.0, 1000.0], device="cuda")
    for activation in ACTIVATIONS:
        out = group_norm_activation(x, lens, w, b.to(x.dtype), 2, activation=activation)
        want = oracle.activate(b.double().cpu().numpy(), activation)
        bound = (cases.HALF[dtype] + 16 * cases.U) * (1 + np.abs(want)) + 1e-6
        cases.assert_within(cases.host(out), np.broadcast_to(want, (1, 5, 8)), bound, activation)
        grads = group_norm_activation_backward(torch.ones_like(x), x, lens, w, b.to(x.dtype), mean,
                                               rstd, activation=activation)
        assert all(torch.isfinite(g).all() for g in grads)
        want = 5 * oracle.slope(b.double().cpu().numpy(), activation)
        cases.assert_within(cases.host(grads[2]), want,
                            (cases.HALF[dtype] + 64 * cases.U) * (5 + np.abs(want)), activation)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_the_lowest_bias_closes_a_channel(dtype):
    """A bias of the type's lowest value: silu gives zero and so do its gradients."""
    x, w, b, dout = cases.norm_inputs(2, 9, 8, dtype, 4)
    lens = lengths_on_gpu([9, 3])
    args = [cases.to_cuda(v, dtype) for v in (x, w, b, dout)]
    args[2][5] = torch.finfo(args[2].dtype).min
    out, mean, rstd = group_norm_activation(args[0], lens, args[1], args[2], 2,
                                            return_statistics=True)
    assert torch.isfinite(out).all() and not out[:, :, 5].any() and out[0, :, 4].all()
    grads = group_norm_activation_backward(args[3], args[0], lens, args[1], args[2], mean, rstd)
    assert all(torch.isfinite(g).all() for g in grads)
    assert grads[1][5] == 0 and grads[2][5] == 0
    for activation in ("none", "swoosh_r"):
        out = group_norm_activation(args[0], lens, args[1], args[2], 2, activation=activation)
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_a_nan_stays_in_its_group(dtype):
    n, t, c, groups = 2, 40, 48, 6
    x, w, b, dout = cases.norm_inputs(n, t, c, dtype, 3)
    x[1, 7, 19] = np.nan  # group 2 of utterance 1
    lens = lengths_on_gpu([t, t])
    args = [cases.to_cuda(v, dtype) for v in (x, w, b, dout)]
    out, mean, rstd = group_norm_activation(args[0], lens, args[1], args[2], groups,
                                            return_statistics=True)
    grad = group_norm_activation_backward(args[3], args[0], lens, args[1], args[2], mean, rstd)[0]
    inside = np.zeros((n, t, c), bool)
    inside[1, :, 16:24] = True
    for v in (out, grad):
        assert np.array_equal(np.isnan(cases.host(v)), inside)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_unaligned_buffers_and_guards(dtype, shift):
    """Bindings that start `shift` elements into their storage, with sentinels around."""
    n, t, c, groups = 3, 50, 64, 4
    x, w, b, dout = cases.norm_inputs(n, t, c, dtype, 8)
    lengths = [50, 0, 23]
    lens = lengths_on_gpu(lengths)
    dt = getattr(torch, dtype)

    def shifted(v):
        room = torch.full((v.size + 64,), 77.0, dtype=dt, device="cuda")
        room[shift:shift + v.size] = cases.to_cuda(v, dtype).flatten()
        return room, room[shift:shift + v.size].view(v.shape)

    (_, gx), (_, gw), (_, gb), (_, gd) = (shifted(v) for v in (x, w, b, dout))
    room, out = shifted(np.zeros((n, t, c)))
    aligned = [cases.to_cuda(v, dtype) for v in (x, w, b, dout)]
    want, mean, rstd = group_norm_activation(aligned[0], lens, aligned[1], aligned[2], groups,
                                             return_statistics=True)
    group_norm_activation(gx, lens, gw, gb, groups, out=out)
    assert torch.all(room[:shift] == 77.0) and torch.all(room[shift + out.numel():] == 77.0)
    expected = oracle.group_norm_activation(x, lengths, w, b, groups, 1e-5, "silu")
    bound = cases.norm_bounds(x, lengths, w, b, groups, expected[1], expected[2], expected[0],
                              dtype)[0]
    cases.assert_within(cases.host(out), expected[0], bound)
    grads = group_norm_activation_backward(gd, gx, lens, gw, gb, mean, rstd)
    mu, r = cases.host(mean), cases.host(rstd)
    want = oracle.group_norm_activation_backward(dout, x, lengths, w, b, mu, r, "silu")
    bounds = cases.norm_gradient_bounds(dout, x, lengths, w, b, mu, r, want, "silu", dtype)
    for got, e, bound in zip(grads, want, bounds):
        cases.assert_within(cases.host(got), e, bound)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("n,t,c,groups", [(2, 100, 65, 5), (1, 9, 3, 1), (1, 3000, 129, 3),
                                          (2, 5000, 1, 1), (3, 70, 130, 130), (40, 900, 258, 2)])
def test_tensors_that_start_differently(n, t, c, groups, dtype):
    x, w, b, dout = cases.norm_inputs(n, t, c, dtype, 8)
    lengths = [t] * n
    lens = lengths_on_gpu(lengths)

    def starting(v, shift):
        room = torch.full((v.size + 64,), float("nan"), dtype=getattr(torch, dtype), device="cuda")
        room[shift:shift + v.size] = cases.to_cuda(v, dtype).flatten()
        return room[shift:shift + v.size].view(v.shape)

    gx, gw, gb, gd = (starting(v, s) for v, s in ((x, 1), (w, 3), (b, 0), (dout, 6)))
    out = starting(np.zeros((n, t, c)), 5)
    _, mean, rstd = group_norm_activation(gx, lens, gw, gb, groups, out=out,
                                          return_statistics=True)
    expected = oracle.group_norm_activation(x, lengths, w, b, groups, 1e-5, "silu")
    bounds = cases.norm_bounds(x, lengths, w, b, groups, expected[1], expected[2], expected[0],
                               dtype)
    for v, want, bound in zip((out, mean, rstd), expected, bounds):
        cases.assert_within(cases.host(v), want, bound)
    grads = group_norm_activation_backward(gd, gx, lens, gw, gb, mean, rstd)
    mu, r = cases.host(mean), cases.host(rstd)
    want = oracle.group_norm_activation_backward(dout, x, lengths, w, b, mu, r, "silu")
    bounds = cases.norm_gradient_bounds(dout, x, lengths, w, b, mu, r, want, "silu", dtype)
    for v, e, bound in zip(grads, want, bounds):
        cases.assert_within(cases.host(v), e, bound)


@pytest.mark.parametrize("n,t,c,groups", [(4, 60, 128, 8), (2, 2500, 64, 1), (1, 700, 1040, 1)])
def test_streams_graphs_and_repeats_give_the_same_bits(n, t, c, groups):
    x, w, b, dout = (cases.to_cuda(v, "bfloat16") for v in cases.norm_inputs(n, t, c, "bfloat16", 5))
    lens = lengths_on_gpu(cases.mixed_lengths(n, t, 5))

    def both(stream=None):
        out, mean, rstd = group_norm_activation(x, lens, w, b, groups, return_statistics=True,
                                                stream=stream)
        return (out, mean, rstd, *group_norm_activation_backward(dout, x, lens, w, b, mean, rstd,
                                                                 stream=stream))

    first = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    on_side = both(side)
    side.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            captured = both()
        graphs.append((g, captured))
    for _ in range(2):
        for g, captured in graphs:
            for v in captured:
                v.fill_(float("nan"))
            g.replay()
    torch.cuda.synchronize()
    for other in (on_side, graphs[0][1], graphs[1][1], both()):
        assert all(torch.equal(p, q) for p, q in zip(first, other))
    # A replay reads its inputs anew.
    x.mul_(2.0)
    graphs[0][0].replay()
    assert all(torch.equal(p, q) for p, q in zip(graphs[0][1], both()))


def test_calls_from_two_threads():
    import threading

    problems = []
    for seed, (n, t, c, groups) in enumerate(((3, 900, 64, 1), (4, 100, 96, 12))):
        x, w, b, dout = (cases.to_cuda(v, "float16")
                         for v in cases.norm_inputs(n, t, c, "float16", seed))
        lens = lengths_on_gpu([t] * n)

        def call(x=x, w=w, b=b, dout=dout, lens=lens, groups=groups):
            out, mean, rstd = group_norm_activation(x, lens, w, b, groups, return_statistics=True)
            return (out, *group_norm_activation_backward(dout, x, lens, w, b, mean, rstd))

        problems.append((call, call()))
    torch.cuda.synchronize()
    wrong = []

    def work(call, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = call()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want)):
                    wrong.append(1)

    threads = [threading.Thread(target=work, args=p) for p in problems for _ in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


def test_a_given_workspace_is_enough():
    n, t, c = 2, 3000, 256
    x, w, b, dout = (cases.to_cuda(v, "float16") for v in cases.norm_inputs(n, t, c, "float16", 6))
    lens = lengths_on_gpu([t, 1234])
    size = normalization.group_norm_activation_workspace_size(x, lens, w, b, 1)
    ws = torch.full((size + 256,), 171, dtype=torch.uint8, device="cuda")
    want = group_norm_activation(x, lens, w, b, 1)
    got = group_norm_activation(x, lens, w, b, 1, workspace=ws[:max(size, 1)])
    assert torch.equal(want, got) and torch.all(ws[size:] == 171)


@pytest.mark.parametrize("n,t,c,groups", [(2, 3000, 256, 1), (200, 400, 256, 8), (1, 60, 512, 32)])
def test_a_given_backward_workspace_is_enough(n, t, c, groups):
    x, w, b, dout = (cases.to_cuda(v, "float16") for v in cases.norm_inputs(n, t, c, "float16", 6))
    lens = lengths_on_gpu([t] + [t // 2] * (n - 1))
    _, mean, rstd = group_norm_activation(x, lens, w, b, groups, return_statistics=True)
    size = normalization.group_norm_activation_backward_workspace_size(x, lens, w, b, groups)
    ws = torch.full((size + 256,), 171, dtype=torch.uint8, device="cuda")
    want = group_norm_activation_backward(dout, x, lens, w, b, mean, rstd)
    got = group_norm_activation_backward(dout, x, lens, w, b, mean, rstd, workspace=ws[:size])
    assert all(torch.equal(p, q) for p, q in zip(want, got)) and torch.all(ws[size:] == 171)


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last utterance as in a call of its own."""
    n, t, c, groups = 3, 1 << 19, 1408, 11
    lens = lengths_on_gpu([0, 5, 700])
    x = torch.empty(n, t, c, dtype=torch.bfloat16, device="cuda")
    x[2, :700] = torch.randn(700, c, device="cuda")
    x[1, :5] = torch.randn(5, c, device="cuda")
    w, b = torch.randn(2, c, device="cuda").to(x.dtype)
    out, mean, rstd = group_norm_activation(x, lens, w, b, groups, return_statistics=True)
    want, mu, r = group_norm_activation(x[2:, :700].contiguous(), lens[2:].contiguous(), w, b,
                                        groups, return_statistics=True)
    torch.testing.assert_close(mean[2:], mu, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(rstd[2:], r, rtol=1e-5, atol=0)
    torch.testing.assert_close(out[2:, :700], want, rtol=2 ** -7, atol=1e-3)
    assert not out[2, 700:].any() and not out[0].any()
    del out
    dout = torch.ones_like(x)
    grads = group_norm_activation_backward(dout, x, lens, w, b, mean, rstd)
    small = group_norm_activation_backward(dout[2:, :700].contiguous(), x[2:, :700].contiguous(),
                                           lens[2:].contiguous(), w, b, mu, r)
    torch.testing.assert_close(grads[0][2:, :700], small[0], rtol=2 ** -7, atol=1e-3)
    assert not grads[0][2, 700:].any() and not grads[0][0].any()


# ---- refusals ---------------------------------------------------------------------------------

def test_refusals():
    x = torch.zeros(2, 6, 16, device="cuda")
    lens = lengths_on_gpu([6, 6])
    w, b = torch.ones(16, device="cuda"), torch.zeros(16, device="cuda")
    mean, rstd = torch.zeros(2, 4, device="cuda"), torch.ones(2, 4, device="cuda")
    for bad in (0, -1, 3, 17):
        with pytest.raises(_lib.AttentionError):
            group_norm_activation(x, lens, w, b, bad)
    with pytest.raises(_lib.AttentionError, match="BAD_FIELD"):
        group_norm_activation(x, lens, w, b, 4, activation="gelu")
    with pytest.raises(_lib.AttentionError, match="BAD_FIELD"):
        group_norm_activation(x, lens, w, b, 4, eps=0.0)
    with pytest.raises(_lib.AttentionError, match="BAD_DESCRIPTOR"):
        group_norm_activation(x, lens.long(), w, b, 4)
    with pytest.raises(_lib.AttentionError, match="BAD_DESCRIPTOR"):
        group_norm_activation(x, lens, w.half(), b, 4)
    with pytest.raises(_lib.AttentionError, match="UNSUPPORTED"):
        group_norm_activation(x, lens, w, b, 4, out=x)
    with pytest.raises(ValueError, match="contiguous"):
        group_norm_activation(x[:, :, ::2], lens, w[::2], b[::2], 4)
    with pytest.raises(ValueError, match="CUDA tensor"):
        group_norm_activation(x, lens.cpu(), w, b, 4)
    with pytest.raises(ValueError, match="requires grad"):
        group_norm_activation(x, lens, w.clone().requires_grad_(), b, 4)
    with torch.no_grad():
        group_norm_activation(x, lens, w.clone().requires_grad_(), b, 4)
    with pytest.raises(_lib.AttentionError, match="BAD_SHAPE"):
        group_norm_activation_backward(x, x, lens, w, b, mean[:, :3].contiguous(),
                                       rstd[:, :3].contiguous())
    with pytest.raises(_lib.AttentionError, match="BAD_SHAPE"):
        group_norm_activation_backward(x[:, :5].contiguous(), x, lens, w, b, mean, rstd)
    with pytest.raises(_lib.AttentionError, match="BAD_DESCRIPTOR"):
        group_norm_activation_backward(x, x, lens, w, b, mean.half(), rstd.half())
