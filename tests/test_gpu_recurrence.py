"""GPU tests of the gated linear recurrence, forward and backward, against the float64 oracle,
and of the operators in a row as an encoder layer uses them.

The bounds count roundings (``sequence_cases``). Padded frames hold NaN, which no output may
show."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import sequence_cases as cases
from fast_gpu_asr_b200 import (_lib, gated_linear_recurrence, gated_linear_recurrence_backward,
                               group_norm_activation, group_norm_activation_backward,
                               parakeet_conformer_convolution, recurrence)
from oracle import sequence_oracle as oracle

pytestmark = pytest.mark.gpu


def lengths_on_gpu(lengths):
    return torch.from_numpy(np.asarray(lengths, np.int32)).cuda()


def check(n, t, c, dtype, lengths=None, with_state=True, seed=None):
    seed = 7 * n + 11 * t + 13 * c if seed is None else seed
    x, gate, dout, initial, dfinal = cases.recurrence_inputs(n, t, c, dtype, seed)
    lengths = cases.mixed_lengths(n, t, seed) if lengths is None else np.asarray(lengths, np.int32)
    if not with_state:
        initial = dfinal = None
    gx, gg, gd = (cases.to_cuda(cases.poison(v, lengths), dtype) for v in (x, gate, dout))
    gi = cases.to_cuda(initial, "float32") if with_state else None
    gf = cases.to_cuda(dfinal, "float32") if with_state else None
    lens = lengths_on_gpu(lengths)
    got = gated_linear_recurrence(gx, gg, lens, gi, return_states=True)
    expected = oracle.gated_linear_recurrence(x, gate, lengths, initial)
    bounds = cases.recurrence_bounds(x, gate, lengths, initial, expected, dtype)
    for v, want, bound, what in zip(got, expected, bounds, ("out", "final", "states")):
        cases.assert_within(cases.host(v), want, bound, (what, n, t, c, dtype))
    without = gated_linear_recurrence(gx, gg, lens, gi)
    assert torch.equal(without[0], got[0]) and torch.equal(without[1], got[1])

    grads = gated_linear_recurrence_backward(gd, gx, gg, lens, got[2], gf)
    want = oracle.gated_linear_recurrence_backward(dout, x, gate, lengths, initial, dfinal)
    bounds = cases.recurrence_gradient_bounds(dout, x, gate, lengths, initial, dfinal,
                                              expected[0], want, dtype)
    for v, e, bound, what in zip(grads, want, bounds, ("grad_x", "grad_gate", "grad_initial")):
        cases.assert_within(cases.host(v), e, bound, (what, n, t, c, dtype))
    assert grads[0].dtype == grads[1].dtype == gx.dtype


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("with_state", [True, False])
@pytest.mark.parametrize("t", [1, 2, 8, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 257])
def test_lengths(t, with_state, dtype):
    check(6, t, 70, dtype, with_state=with_state)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("c", [1, 2, 3, 7, 32, 63, 64, 65, 77, 130, 512])
def test_channels(c, dtype):
    check(3, 70, c, dtype)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("n,t,c", [(2, 375, 1024), (1, 1500, 33), (2, 3000, 64), (1, 5000, 16),
                                   (40, 200, 256), (1, 12000, 66), (1, 13000, 8)])
def test_every_split(n, t, c, dtype):
    check(n, t, c, dtype, lengths=[t] if n == 1 else None)


def test_many_streams_one_frame():
    check(300, 1, 48, "bfloat16", lengths=[1] * 300)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_saturated_gates(dtype):
    """A gate of -inf or the type's lowest value takes x, +inf or the highest keeps the state,
    and the gradients of both are zeros or the gradient itself.

    Below -87.3 the kernels' f stays at 2^-126, the smallest normal number: what should be a
    zero f (h - x) G is at most 2^-126 * 4 * 3 here (|h - x| <= 4, |G| <= 3), and f G at most
    2^-126 * 3."""
    dt = getattr(torch, dtype)
    low, high = torch.finfo(dt).min, torch.finfo(dt).max
    gates = torch.tensor([[-np.inf, low, np.inf, high, -np.inf, np.inf]], device="cuda")
    t, c = gates.shape[1], 4
    gate = gates.to(dt)[:, :, None].expand(1, t, c).contiguous()
    x = torch.arange(1, t + 1, device="cuda").to(dt)[None, :, None].expand(1, t, c).contiguous()
    lens = lengths_on_gpu([t])
    out, final, states = gated_linear_recurrence(x, gate, lens, return_states=True)
    want = torch.tensor([1.0, 2, 2, 2, 5, 5], device="cuda")
    assert torch.equal(out[0, :, 0].float(), want) and torch.all(final == 5.0)
    dout = torch.ones_like(x)
    gx, gg, gi = gated_linear_recurrence_backward(dout, x, gate, lens, states)
    want = torch.tensor([1.0, 3, 0, 0, 2, 0], device="cuda")
    assert torch.equal(gx[0, :, 0].float(), want)
    assert gg.abs().max() <= 12 * 2.0 ** -126 and gi.abs().max() <= 3 * 2.0 ** -126


@pytest.mark.parametrize("gate", [-60.0, -12.0, 12.0, 60.0])
def test_far_gates(gate):
    """Gates where 1 - f or f itself would round to nothing."""
    n, t, c = 2, 300, 10
    x, g, dout, initial, dfinal = cases.recurrence_inputs(n, t, c, "float32", 31)
    g = cases.store(g * 0.1 + gate, "float32")
    lengths = [300, 129]
    lens = lengths_on_gpu(lengths)
    args = [cases.to_cuda(v, "float32") for v in (x, g, dout, initial, dfinal)]
    got = gated_linear_recurrence(args[0], args[1], lens, args[3], return_states=True)
    expected = oracle.gated_linear_recurrence(x, g, lengths, initial)
    for v, want, bound in zip(got, expected, cases.recurrence_bounds(x, g, lengths, initial,
                                                                     expected, "float32")):
        cases.assert_within(cases.host(v), want, bound)
    grads = gated_linear_recurrence_backward(args[2], args[0], args[1], lens, got[2], args[4])
    want = oracle.gated_linear_recurrence_backward(dout, x, g, lengths, initial, dfinal)
    bounds = cases.recurrence_gradient_bounds(dout, x, g, lengths, initial, dfinal, expected[0],
                                              want, "float32")
    for v, e, bound in zip(grads, want, bounds):
        cases.assert_within(cases.host(v), e, bound)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("where", ["x", "gate"])
@pytest.mark.parametrize("n,t,c", [(2, 300, 66), (1, 3000, 65)])
def test_a_nan_stays_in_its_channel_and_its_future(n, t, c, where, dtype):
    x, gate, dout, initial, dfinal = cases.recurrence_inputs(n, t, c, dtype, 9)
    (x if where == "x" else gate)[0, 150, 9] = np.nan
    lens = lengths_on_gpu([t] * n)
    gx, gg, gd = (cases.to_cuda(v, dtype) for v in (x, gate, dout))
    out, final, states = gated_linear_recurrence(gx, gg, lens, return_states=True)
    bad = np.zeros((n, t, c), bool)
    bad[0, 150:, 9] = True
    assert np.array_equal(np.isnan(cases.host(out)), bad)
    grad_x, grad_gate, _ = gated_linear_recurrence_backward(gd, gx, gg, lens, states)
    if where == "x":
        assert np.array_equal(np.isnan(cases.host(grad_gate)), bad)
        assert not torch.isnan(grad_x).any()
    else:  # what comes before it in the channel takes the gradient through the gate
        past = np.zeros_like(bad)
        past[0, :151, 9] = True
        assert np.array_equal(np.isnan(cases.host(grad_x)), past)
        assert np.array_equal(np.isnan(cases.host(grad_gate)), bad | past)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_a_stream_in_pieces(dtype):
    """Pieces of any size, one frame among them, with the state passed on in place."""
    n, t, c = 3, 200, 40
    x, gate, _, initial, _ = cases.recurrence_inputs(n, t, c, dtype, 12)
    lengths = [200, 77, 0]
    gx, gg = cases.to_cuda(x, dtype), cases.to_cuda(gate, dtype)
    expected = oracle.gated_linear_recurrence(x, gate, lengths, initial)
    bounds = cases.recurrence_bounds(x, gate, lengths, initial, expected, dtype)
    state = cases.to_cuda(initial, "float32")
    pieces, at = [], 0
    for size in (1, 64, 1, 1, 17, 100, 16):
        part = slice(at, at + size)
        left = lengths_on_gpu(np.clip(np.asarray(lengths) - at, 0, size))
        out, final = gated_linear_recurrence(gx[:, part].contiguous(), gg[:, part].contiguous(),
                                             left, state, final_state=state)
        assert final is state
        pieces.append(out)
        at += size
    assert at == t
    cases.assert_within(cases.host(torch.cat(pieces, 1)), expected[0], bounds[0])
    cases.assert_within(cases.host(state), expected[1], bounds[1])


@pytest.mark.parametrize("n,t,c", [(4, 1, 48), (2, 70, 64), (1, 6000, 64), (2, 3000, 130)])
def test_state_in_place_gives_the_same_bits(n, t, c):
    x, gate, _, initial, _ = cases.recurrence_inputs(n, t, c, "bfloat16", 13)
    gx, gg = cases.to_cuda(x, "bfloat16"), cases.to_cuda(gate, "bfloat16")
    lens = lengths_on_gpu([t] * (n - 1) + [0])
    state = cases.to_cuda(initial, "float32")
    out, final = gated_linear_recurrence(gx, gg, lens, state.clone())
    again, _ = gated_linear_recurrence(gx, gg, lens, state, final_state=state)
    assert torch.equal(out, again) and torch.equal(final, state)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_unaligned_buffers_and_guards(dtype, shift):
    n, t, c = 2, 140, 66
    x, gate, dout, initial, dfinal = cases.recurrence_inputs(n, t, c, dtype, 21)
    lengths = [140, 75]
    lens = lengths_on_gpu(lengths)

    def shifted(v, dt):
        room = torch.full((v.size + 64,), 77.0, dtype=getattr(torch, dt), device="cuda")
        room[shift:shift + v.size] = cases.to_cuda(v, dt).flatten()
        return room, room[shift:shift + v.size].view(v.shape)

    gx, gg, gd = (shifted(v, dtype)[1] for v in (x, gate, dout))
    gi, gf = (shifted(v, "float32")[1] for v in (initial, dfinal))
    room, out = shifted(np.zeros((n, t, c)), dtype)
    state_room, final = shifted(np.zeros((n, c)), "float32")
    _, _, states = gated_linear_recurrence(gx, gg, lens, gi, out=out, final_state=final,
                                           return_states=True)
    for r, v in ((room, out), (state_room, final)):
        assert torch.all(r[:shift] == 77.0) and torch.all(r[shift + v.numel():] == 77.0)
    expected = oracle.gated_linear_recurrence(x, gate, lengths, initial)
    bounds = cases.recurrence_bounds(x, gate, lengths, initial, expected, dtype)
    for v, want, bound in zip((out, final, states), expected, bounds):
        cases.assert_within(cases.host(v), want, bound)
    grads = gated_linear_recurrence_backward(gd, gx, gg, lens, states, gf)
    want = oracle.gated_linear_recurrence_backward(dout, x, gate, lengths, initial, dfinal)
    bounds = cases.recurrence_gradient_bounds(dout, x, gate, lengths, initial, dfinal,
                                              expected[0], want, dtype)
    for v, e, bound in zip(grads, want, bounds):
        cases.assert_within(cases.host(v), e, bound)


def starting(v, dtype, shift):
    """`v` on the GPU, `shift` elements into a storage of NaN."""
    room = torch.full((v.size + 64,), float("nan"), dtype=getattr(torch, dtype), device="cuda")
    room[shift:shift + v.size] = cases.to_cuda(v, dtype).flatten()
    return room[shift:shift + v.size].view(v.shape)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("n,t,c", [(2, 100, 65), (1, 9, 3), (1, 1500, 33), (3, 70, 130), (2, 64, 1)])
def test_tensors_that_start_differently(n, t, c, dtype):
    x, gate, dout, initial, dfinal = cases.recurrence_inputs(n, t, c, dtype, 23)
    lengths = [t] * n
    lens = lengths_on_gpu(lengths)
    gx, gg, gd = (starting(v, dtype, s) for v, s in ((x, 1), (gate, 0), (dout, 5)))
    gi, gf = (cases.to_cuda(v, "float32") for v in (initial, dfinal))
    out = starting(np.zeros((n, t, c)), dtype, 3)
    got = gated_linear_recurrence(gx, gg, lens, gi, out=out, return_states=True)
    expected = oracle.gated_linear_recurrence(x, gate, lengths, initial)
    bounds = cases.recurrence_bounds(x, gate, lengths, initial, expected, dtype)
    for v, want, bound in zip(got, expected, bounds):
        cases.assert_within(cases.host(v), want, bound)
    grads = gated_linear_recurrence_backward(gd, gx, gg, lens, got[2], gf)
    want = oracle.gated_linear_recurrence_backward(dout, x, gate, lengths, initial, dfinal)
    bounds = cases.recurrence_gradient_bounds(dout, x, gate, lengths, initial, dfinal,
                                              expected[0], want, dtype)
    for v, e, bound in zip(grads, want, bounds):
        cases.assert_within(cases.host(v), e, bound)


@pytest.mark.parametrize("n,t,c", [(4, 60, 128), (1, 5000, 64), (3, 700, 65)])
def test_streams_graphs_and_repeats_give_the_same_bits(n, t, c):
    x, gate, dout, initial, dfinal = cases.recurrence_inputs(n, t, c, "float16", 5)
    x, gate, dout = (cases.to_cuda(v, "float16") for v in (x, gate, dout))
    initial, dfinal = (cases.to_cuda(v, "float32") for v in (initial, dfinal))
    lens = lengths_on_gpu([t] + [t // 3] * (n - 1))

    def both(stream=None):
        got = gated_linear_recurrence(x, gate, lens, initial, return_states=True, stream=stream)
        return (*got, *gated_linear_recurrence_backward(dout, x, gate, lens, got[2], dfinal,
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


@pytest.mark.parametrize("n,t,c", [(1, 5000, 64), (3, 700, 65), (2, 60, 64), (1, 128, 40)])
def test_a_given_workspace_is_enough(n, t, c):
    x, gate, dout, initial, dfinal = cases.recurrence_inputs(n, t, c, "float16", 6)
    x, gate, dout = (cases.to_cuda(v, "float16") for v in (x, gate, dout))
    initial, dfinal = (cases.to_cuda(v, "float32") for v in (initial, dfinal))
    lens = lengths_on_gpu([t] + [t // 3] * (n - 1))
    size = recurrence.gated_linear_recurrence_workspace_size(x, lens)
    size_back = recurrence.gated_linear_recurrence_backward_workspace_size(x, lens)
    assert (size > 0) == (size_back > 0) == (t > 128)
    ws = torch.full((size + 256,), 171, dtype=torch.uint8, device="cuda")
    ws_back = torch.full((size_back + 256,), 171, dtype=torch.uint8, device="cuda")
    want = gated_linear_recurrence(x, gate, lens, initial, return_states=True)
    got = gated_linear_recurrence(x, gate, lens, initial, return_states=True, workspace=ws[:size])
    want += gated_linear_recurrence_backward(dout, x, gate, lens, want[2], dfinal)
    got += gated_linear_recurrence_backward(dout, x, gate, lens, got[2], dfinal,
                                            workspace=ws_back[:size_back])
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    assert torch.all(ws[size:] == 171) and torch.all(ws_back[size_back:] == 171)
    if size:
        with pytest.raises(_lib.AttentionError, match="WORKSPACE"):
            gated_linear_recurrence(x, gate, lens, initial, workspace=ws[:size - 1])


def test_a_decoding_loop_in_a_graph():
    """The streaming step captured once, its state updated in place by every replay."""
    n, t, c = 5, 12, 64
    x, gate, _, initial, _ = cases.recurrence_inputs(n, t, c, "bfloat16", 17)
    gx, gg = cases.to_cuda(x, "bfloat16"), cases.to_cuda(gate, "bfloat16")
    state, lens = cases.to_cuda(initial, "float32"), lengths_on_gpu([1] * n)
    step_x, step_g = gx[:, :1].contiguous(), gg[:, :1].contiguous()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, _ = gated_linear_recurrence(step_x, step_g, lens, state, final_state=state)
    expected = oracle.gated_linear_recurrence(x, gate, [t] * n, initial)
    bounds = cases.recurrence_bounds(x, gate, [t] * n, initial, expected, "bfloat16")
    for i in range(t):
        step_x.copy_(gx[:, i:i + 1])
        step_g.copy_(gg[:, i:i + 1])
        g.replay()
        cases.assert_within(cases.host(out)[:, 0], expected[0][:, i], bounds[0][:, i])
    cases.assert_within(cases.host(state), expected[1], bounds[1])


def test_offsets_past_32_bits():
    n, t, c = 3, 1 << 19, 1408
    lengths = [0, 5, 700]
    lens = lengths_on_gpu(lengths)
    x = torch.empty(n, t, c, dtype=torch.bfloat16, device="cuda")
    gate = torch.empty_like(x)
    for i, m in enumerate(lengths):
        x[i, :m] = torch.randn(m, c, device="cuda")
        gate[i, :m] = torch.randn(m, c, device="cuda")
    initial = torch.randn(n, c, device="cuda")
    out, final, states = gated_linear_recurrence(x, gate, lens, initial, return_states=True)
    cut = [v[2:, :700].contiguous() for v in (x, gate)]
    want = gated_linear_recurrence(*cut, lens[2:].contiguous(), initial[2:].contiguous(),
                                   return_states=True)
    torch.testing.assert_close(out[2:, :700], want[0], rtol=2 ** -7, atol=1e-4)
    torch.testing.assert_close(final[2:], want[1], rtol=1e-5, atol=1e-5)
    assert not out[2, 700:].any() and not out[0].any() and torch.equal(final[0], initial[0])
    dout = out
    grads = gated_linear_recurrence_backward(dout, x, gate, lens, states)
    small = gated_linear_recurrence_backward(dout[2:, :700].contiguous(), *cut,
                                             lens[2:].contiguous(), want[2])
    for p, q in zip(grads[:2], small[:2]):
        torch.testing.assert_close(p[2:, :700], q, rtol=2 ** -6, atol=1e-3)
        assert not p[2, 700:].any() and not p[0].any()
    torch.testing.assert_close(grads[2][2:], small[2], rtol=1e-4, atol=1e-4)


# ---- the operators in a row -------------------------------------------------------------------

class Recurrence(torch.autograd.Function):
    """The two halves as an autograd function, as the integration notes show it."""

    @staticmethod
    def forward(ctx, x, gate, lengths):
        out, final, states = gated_linear_recurrence(x, gate, lengths, return_states=True)
        ctx.save_for_backward(x, gate, lengths, states)
        return out, final

    @staticmethod
    def backward(ctx, grad_out, grad_final):
        x, gate, lengths, states = ctx.saved_tensors
        grad_x, grad_gate, _ = gated_linear_recurrence_backward(
            grad_out.contiguous(), x, gate, lengths, states, grad_final.contiguous())
        return grad_x, grad_gate, None


class Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, lengths, weight, bias, groups):
        out, mean, rstd = group_norm_activation(x, lengths, weight, bias, groups,
                                                return_statistics=True)
        ctx.save_for_backward(x, lengths, weight, bias, mean, rstd)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        grads = group_norm_activation_backward(grad_out.contiguous(), *ctx.saved_tensors)
        return grads[0], None, grads[1], grads[2], None


def test_recurrence_then_norm_trains_like_the_formulas():
    """Recurrence -> group norm + SiLU under autograd, fp32, against torch's own autograd of
    the formulas in float64. Every value passes both operators in fp32: 1e-4 of the largest
    gradient is over 1000 roundings."""
    n, t, c, groups = 3, 90, 32, 4
    lengths = [90, 41, 7]
    x, gate, dout, _, _ = cases.recurrence_inputs(n, t, c, "float32", 41)
    _, w, b, _ = cases.norm_inputs(1, 1, c, "float32", 42)
    lens = lengths_on_gpu(lengths)
    leaves = [cases.to_cuda(v, "float32").requires_grad_() for v in (x, gate, w, b)]
    out, final = Recurrence.apply(leaves[0], leaves[1], lens)
    y = Norm.apply(out, lens, leaves[2], leaves[3], groups)
    ((y * cases.to_cuda(dout, "float32")).sum() + final.square().sum()).backward()

    ref = [torch.tensor(v, requires_grad=True) for v in (x, gate, w, b)]
    loss = 0.0
    for i, m in enumerate(lengths):
        h, hs = torch.zeros(c, dtype=torch.float64), []
        for j in range(m):
            f = torch.sigmoid(ref[1][i, j])
            h = f * h + (1 - f) * ref[0][i, j]
            hs.append(h)
        z = torch.nn.functional.group_norm(torch.stack(hs).T[None], groups, ref[2], ref[3])[0].T
        loss = loss + (torch.nn.functional.silu(z) * torch.tensor(dout[i, :m])).sum()
        loss = loss + h.square().sum()
    loss.backward()
    for leaf, r in zip(leaves, ref):
        want = r.grad.numpy()
        cases.assert_within(cases.host(leaf.grad), want, 1e-4 * np.abs(want).max())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_convolution_recurrence_norm(dtype):
    """A layer's time mixers on one stream: convolution -> recurrence -> group norm. Each
    operator is held to its own bound on what the one before it gave."""
    n, t, c, groups = 4, 130, 64, 4
    lengths = [130, 64, 1, 0]
    lens = lengths_on_gpu(lengths)
    x, gate, _, _, _ = cases.recurrence_inputs(n, t, c, dtype, 51)
    _, w, b, _ = cases.norm_inputs(1, 1, c, dtype, 52)
    taps = cases.to_cuda(np.random.default_rng(1).normal(0, 0.3, (9, c)), dtype)
    gx, gg, gw, gb = (cases.to_cuda(v, dtype) for v in (x, gate, w, b))
    mixed = parakeet_conformer_convolution(gx, lens, taps, gb)
    out, final = gated_linear_recurrence(mixed, gg, lens)
    y = group_norm_activation(out, lens, gw, gb, groups)
    assert not y[3].any() and not y[1, 64:].any() and torch.isfinite(y).all()
    m = cases.host(mixed)
    expected = oracle.gated_linear_recurrence(m, gate, lengths)
    bounds = cases.recurrence_bounds(m, gate, lengths, None, expected, dtype)
    cases.assert_within(cases.host(out), expected[0], bounds[0])
    cases.assert_within(cases.host(final), expected[1], bounds[1])
    o = cases.host(out)
    want = oracle.group_norm_activation(o, lengths, w, b, groups)
    bound = cases.norm_bounds(o, lengths, w, b, groups, want[1], want[2], want[0], dtype)[0]
    cases.assert_within(cases.host(y), want[0], bound)


# ---- refusals ---------------------------------------------------------------------------------

def test_refusals():
    x = torch.zeros(2, 70, 16, device="cuda")
    lens, state = lengths_on_gpu([6, 6]), torch.zeros(2, 16, device="cuda")
    states = torch.zeros(2, 2, 16, device="cuda")
    with pytest.raises(_lib.AttentionError, match="BAD_SHAPE"):
        gated_linear_recurrence(x, x[:, :69].contiguous(), lens)
    with pytest.raises(_lib.AttentionError, match="BAD_DESCRIPTOR"):
        gated_linear_recurrence(x, x.half(), lens)
    with pytest.raises(_lib.AttentionError, match="BAD_DESCRIPTOR"):
        gated_linear_recurrence(x, x, lens, state.half())
    with pytest.raises(_lib.AttentionError, match="BAD_SHAPE"):
        gated_linear_recurrence(x, x, lens, state[:1])
    with pytest.raises(_lib.AttentionError, match="UNSUPPORTED"):
        gated_linear_recurrence(x, x, lens, out=x)
    with pytest.raises(ValueError, match="contiguous"):
        gated_linear_recurrence(x.transpose(0, 1), x.transpose(0, 1), lens)
    with pytest.raises(ValueError, match="CUDA tensor"):
        gated_linear_recurrence(x, x, lens.cpu())
    with pytest.raises(ValueError, match="requires grad"):
        gated_linear_recurrence(x.clone().requires_grad_(), x, lens)
    with pytest.raises(_lib.AttentionError, match="BAD_SHAPE"):
        gated_linear_recurrence_backward(x, x, x, lens, states[:, :1].contiguous())
    with pytest.raises(_lib.AttentionError, match="BAD_SHAPE"):
        gated_linear_recurrence_backward(x, x, x, lens, states, state[:, :8].contiguous())
    with pytest.raises(_lib.AttentionError, match="OVERFLOW"):
        gated_linear_recurrence(x[:0], x[:0], lens[:0])
