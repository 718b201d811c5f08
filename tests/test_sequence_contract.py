"""Group norm with activation and the gated linear recurrence without a device: the contract
checks of their C entry points, the refusals of the Python functions, and the oracle (against
torch's float64 autograd and against differences)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fast_gpu_asr_b200 import _lib, normalization, recurrence
from oracle import sequence_oracle as oracle

F32, F16, BF16, I32 = _lib.FGA_FLOAT, _lib.FGA_HALF, _lib.FGA_BF16, _lib.FGA_INT32
D = _lib.TensorDesc.make
OK, NULL, DESC, SHAPE, OVERFLOW, FIELD, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3, 4, 5, 9, 10


def norm_descs(n=2, t=9, c=24, g=4, dtype=F16, **override):
    d = dict(x=D(dtype, (n, t, c)), lengths=D(I32, (n,)), weight=D(dtype, (c,)),
             bias=D(dtype, (c,)), out=D(dtype, (n, t, c)), mean=D(F32, (n, g)),
             rstd=D(F32, (n, g)))
    d.update(override)
    return d


def norm_status(d, g=4, eps=1e-5, activation="silu"):
    return normalization.group_norm_activation_check(
        [d[k] for k in ("x", "lengths", "weight", "bias")], [d[k] for k in ("out", "mean", "rstd")],
        g, eps, activation)


def norm_backward_status(d, activation="silu", **override):
    e = dict(grad_out=d["x"], gx=d["x"], gw=d["weight"], gb=d["bias"])
    e.update(override)
    ins = [e["grad_out"], *(d[k] for k in ("x", "lengths", "weight", "bias", "mean", "rstd"))]
    return normalization.group_norm_activation_backward_check(ins, [e["gx"], e["gw"], e["gb"]],
                                                              activation)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_norm_accepts(library, dtype):
    assert norm_status(norm_descs(dtype=dtype)) == OK
    assert norm_backward_status(norm_descs(dtype=dtype)) == OK
    assert norm_status(norm_descs(1, 1, 1, 1, dtype), 1) == OK
    for activation in ("none", "silu", "swoosh_r"):
        assert norm_status(norm_descs(dtype=dtype), activation=activation) == OK


@pytest.mark.parametrize("override,status", [
    (dict(lengths=D(I32, (3,))), SHAPE), (dict(lengths=D(F32, (2,))), DESC),
    (dict(weight=D(F16, (23,))), SHAPE), (dict(bias=D(F32, (24,))), DESC),
    (dict(mean=D(F32, (2, 5))), SHAPE), (dict(mean=D(F32, (3, 4)), rstd=D(F32, (3, 4))), SHAPE),
    (dict(rstd=D(F16, (2, 4))), DESC), (dict(x=D(F16, (2, 9))), DESC),
    (dict(x=D(I32, (2, 9, 24))), DESC),
    (dict(x=D(F16, (0, 9, 24))), OVERFLOW),
], ids=lambda v: str(v)[:20])
def test_norm_refuses(library, override, status):
    d = norm_descs(**override)
    assert norm_status(d) == status
    assert norm_backward_status(d) == status


def test_norm_refuses_more(library):
    d = norm_descs()
    assert norm_status(norm_descs(out=D(BF16, (2, 9, 24)))) == DESC
    assert norm_status(norm_descs(out=D(F16, (2, 8, 24)))) == SHAPE
    assert norm_status(norm_descs(g=5), 5) == SHAPE  # 5 does not divide 24
    assert norm_backward_status(norm_descs(g=5)) == SHAPE
    for g in (0, -4):
        assert norm_status(d, g) == FIELD
    for eps in (0.0, -1e-5, float("inf"), float("nan"), 1e-60):
        assert norm_status(d, eps=eps) == FIELD
    for activation in ("relu", None, 1):
        assert norm_status(d, activation=activation) == FIELD
        assert norm_backward_status(d, activation) == FIELD
    assert norm_backward_status(d, grad_out=D(F16, (2, 9, 23))) == SHAPE
    assert norm_backward_status(d, gw=D(F32, (24,))) == DESC
    assert norm_backward_status(d, gb=D(F16, (25,))) == SHAPE
    # Frames or channels of the batch past 32 bits; their product may be.
    big = norm_descs(1 << 16, 1 << 16, 8, 4)
    assert norm_status(big) == OVERFLOW
    big = norm_descs(1 << 16, 1 << 14, 16, 4)
    assert norm_status(big) == OK


def recurrence_descs(n=2, t=130, c=24, dtype=F16, **override):
    chunks = -(-t // 64)
    d = dict(x=D(dtype, (n, t, c)), gate=D(dtype, (n, t, c)), lengths=D(I32, (n,)),
             state=D(F32, (n, c)), out=D(dtype, (n, t, c)), final=D(F32, (n, c)),
             states=D(F32, (n, chunks, c)))
    d.update(override)
    return d


def recurrence_status(d):
    return recurrence.gated_linear_recurrence_check(
        [d[k] for k in ("x", "gate", "lengths", "state")], [d[k] for k in ("out", "final", "states")])


def recurrence_backward_status(d, **override):
    e = dict(grad_out=d["x"], gx=d["x"], gg=d["gate"], gi=d["state"])
    e.update(override)
    return recurrence.gated_linear_recurrence_backward_check(
        [e["grad_out"], *(d[k] for k in ("x", "gate", "lengths", "states", "final"))],
        [e["gx"], e["gg"], e["gi"]])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("t", [1, 63, 64, 65])
def test_recurrence_accepts(library, dtype, t):
    assert recurrence_status(recurrence_descs(t=t, dtype=dtype)) == OK
    assert recurrence_backward_status(recurrence_descs(t=t, dtype=dtype)) == OK


@pytest.mark.parametrize("override,status", [
    (dict(gate=D(F32, (2, 130, 24))), DESC), (dict(gate=D(F16, (2, 129, 24))), SHAPE),
    (dict(lengths=D(I32, (1,))), SHAPE), (dict(states=D(F32, (2, 2, 24))), SHAPE),
    (dict(states=D(F32, (2, 4, 24))), SHAPE), (dict(states=D(F16, (2, 3, 24))), DESC),
    (dict(state=D(F32, (2, 23)), final=D(F32, (2, 23))), SHAPE),
    (dict(state=D(F16, (2, 24)), final=D(F16, (2, 24))), DESC),
    (dict(x=D(F16, (2, 130, 24, 1))), DESC), (dict(x=D(F16, (2, 0, 24))), OVERFLOW),
], ids=lambda v: str(v)[:20])
def test_recurrence_refuses(library, override, status):
    d = recurrence_descs(**override)
    assert recurrence_status(d) == status
    assert recurrence_backward_status(d) == status


def test_buffers_are_checked_before_any_launch(library):
    """Null, misaligned and overlapping buffers and short workspaces, with made-up addresses:
    every call here is refused on the host."""
    ins = _lib.desc_array([recurrence_descs()[k] for k in ("x", "gate", "lengths", "state")])
    outs = _lib.desc_array([recurrence_descs()[k] for k in ("out", "final", "states")])
    step = 1 << 20
    good_in, good_out = [step * i for i in (1, 2, 3, 4)], [step * i for i in (5, 6, 7)]

    def status(i, o):
        return library.fga_gated_linear_recurrence_enqueue(
            ins, outs, _lib.pointer_array(i), _lib.pointer_array(o), None, 0, None)

    for k in (0, 1, 2):
        assert status([p if q != k else None for q, p in enumerate(good_in)], good_out) == NULL
    for k in (0, 1):
        assert status(good_in, [p if q != k else None for q, p in enumerate(good_out)]) == NULL
    assert status([good_in[0] + 1, *good_in[1:]], good_out) == UNSUPPORTED
    assert status(good_in, [good_out[0], good_out[1] + 2, good_out[2]]) == UNSUPPORTED
    assert status(good_in, [good_in[0], *good_out[1:]]) == UNSUPPORTED          # out is x
    assert status(good_in, [good_in[1] + 64, *good_out[1:]]) == UNSUPPORTED     # inside gate
    assert status(good_in, [good_out[0], good_out[0] + 64, good_out[2]]) == UNSUPPORTED
    assert status(good_in, [good_out[0], good_in[3] + 4, good_out[2]]) == UNSUPPORTED

    d = norm_descs(8, 30000, 1024, 1)
    ins = _lib.desc_array([d[k] for k in ("x", "lengths", "weight", "bias")])
    outs = _lib.desc_array([d[k] for k in ("out", "mean", "rstd")])
    step = 1 << 30
    i, o = _lib.pointer_array([step * k for k in (1, 2, 3, 4)]), [step * k for k in (5, 6, 7)]
    size = library.fga_group_norm_activation_workspace_size(ins, 4, 1)
    assert size == 0 or library.fga_group_norm_activation_enqueue(
        ins, outs, i, _lib.pointer_array(o), 1, 1e-5, 1, o[0] + 64, size, None) == WORKSPACE
    for ws, have in ((None, size), (step * 8, size - 1), (step * 8 + 8, size)):
        if size:
            assert library.fga_group_norm_activation_enqueue(
                ins, outs, i, _lib.pointer_array(o), 1, 1e-5, 1, ws, have, None) == WORKSPACE
    assert library.fga_group_norm_activation_enqueue(
        ins, outs, i, _lib.pointer_array([step, *o[1:]]), 1, 1e-5, 1, step * 8, 1 << 30,
        None) == UNSUPPORTED
    d = norm_descs(8, 300, 1024, 4)
    ins = _lib.desc_array([d["x"], *(d[k] for k in ("x", "lengths", "weight", "bias", "mean",
                                                    "rstd"))])
    size = library.fga_group_norm_activation_backward_workspace_size(ins, 7)
    outs = _lib.desc_array([d["x"], d["weight"], d["bias"]])
    i = _lib.pointer_array([step * k for k in range(1, 8)])
    o = _lib.pointer_array([step * k for k in (8, 9, 10)])
    if size:
        assert library.fga_group_norm_activation_backward_enqueue(
            ins, outs, i, o, 1, None, size, None) == WORKSPACE


def test_state_frames_match_the_header():
    from pathlib import Path

    header = (Path(__file__).resolve().parents[1] / "include" / "fga_convolution.h").read_text()
    assert f"#define FGA_RECURRENCE_STATE_FRAMES {_lib.RECURRENCE_STATE_FRAMES}\n" in header
    assert oracle.STATE_FRAMES == recurrence.STATE_FRAMES == _lib.RECURRENCE_STATE_FRAMES


def test_python_refuses_what_is_no_tensor(library):
    for bad in (None, [1.0], np.zeros((1, 2, 3))):
        with pytest.raises(ValueError, match="x must be a tensor"):
            normalization.group_norm_activation(bad, bad, bad, bad, 1)
        with pytest.raises(ValueError, match="x must be a tensor"):
            recurrence.gated_linear_recurrence(bad, bad, bad)
        with pytest.raises(ValueError, match="x must be a tensor"):
            recurrence.gated_linear_recurrence_backward(bad, bad, bad, bad, bad)
    with pytest.raises(_lib.AttentionError, match="BAD_DESCRIPTOR"):
        recurrence.gated_linear_recurrence(torch.zeros(2, 3), torch.zeros(2, 3), None)


# ---- the oracle -------------------------------------------------------------------------------

LENGTHS = [7, 0, 12, 100]


def torch_activation(z, name):
    if name == "silu":
        return torch.nn.functional.silu(z)
    if name == "swoosh_r":
        return torch.nn.functional.softplus(z - 1.0) - 0.08 * z - 0.313261687
    return z


@pytest.mark.parametrize("activation", ["none", "silu", "swoosh_r"])
@pytest.mark.parametrize("groups", [1, 3, 12])
def test_norm_oracle_matches_autograd(activation, groups):
    rng = np.random.default_rng(3)
    n, t, c = len(LENGTHS), 12, 12
    x, dout = rng.normal(0, 1, (n, t, c)), rng.normal(0, 1, (n, t, c))
    w, b = rng.normal(1, 0.2, c), rng.normal(0, 0.2, c)
    tx, tw, tb = (torch.tensor(v, requires_grad=True) for v in (x, w, b))
    loss, expected = 0.0, np.zeros_like(x)
    for i, m in enumerate(LENGTHS):
        m = min(m, t)
        if m == 0:
            continue
        y = torch.nn.functional.group_norm(tx[i, :m].T[None], groups, tw, tb, 1e-5)[0].T
        y = torch_activation(y, activation)
        expected[i, :m] = y.detach().numpy()
        loss = loss + (y * torch.tensor(dout[i, :m])).sum()
    loss.backward()
    out, mean, rstd = oracle.group_norm_activation(x, LENGTHS, w, b, groups, 1e-5, activation)
    np.testing.assert_allclose(out, expected, rtol=1e-10, atol=1e-12)
    grads = oracle.group_norm_activation_backward(dout, x, LENGTHS, w, b, mean, rstd, activation)
    for got, leaf in zip(grads, (tx, tw, tb)):
        np.testing.assert_allclose(got, leaf.grad.numpy(), rtol=1e-9, atol=1e-11)


def test_recurrence_oracle_matches_autograd():
    rng = np.random.default_rng(4)
    n, t, c = len(LENGTHS), 12, 5
    x, gate, dout = (rng.normal(0, 1, (n, t, c)) for _ in range(3))
    initial, dfinal = rng.normal(0, 1, (n, c)), rng.normal(0, 1, (n, c))
    tx, tg, ti = (torch.tensor(v, requires_grad=True) for v in (x, gate, initial))
    loss = 0.0
    for i, m in enumerate(LENGTHS):
        h = ti[i]
        for j in range(min(m, t)):
            f = torch.sigmoid(tg[i, j])
            h = f * h + (1 - f) * tx[i, j]
            loss = loss + (h * torch.tensor(dout[i, j])).sum()
        loss = loss + (h * torch.tensor(dfinal[i])).sum()
    loss.backward()
    grads = oracle.gated_linear_recurrence_backward(dout, x, gate, LENGTHS, initial, dfinal)
    for got, leaf in zip(grads, (tx, tg, ti)):
        np.testing.assert_allclose(got, leaf.grad.numpy(), rtol=1e-10, atol=1e-12)


def test_gradient_oracles_match_differences():
    """Central differences of the forward oracles, a few directions each."""
    rng = np.random.default_rng(5)
    n, t, c, step = 2, 6, 4, 1e-5
    lengths = [6, 3]
    x, gate, dout = (rng.normal(0, 1, (n, t, c)) for _ in range(3))
    w, b, initial, dfinal = (rng.normal(0.5, 1, s) for s in (c, c, (n, c), (n, c)))

    def norm_loss(x, w, b):
        return (oracle.group_norm_activation(x, lengths, w, b, 2, 1e-5, "silu")[0] * dout).sum()

    def recurrence_loss(x, gate, initial):
        out, final, _ = oracle.gated_linear_recurrence(x, gate, lengths, initial)
        return (out * dout).sum() + (final * dfinal).sum()

    _, mean, rstd = oracle.group_norm_activation(x, lengths, w, b, 2, 1e-5, "silu")
    norm = oracle.group_norm_activation_backward(dout, x, lengths, w, b, mean, rstd, "silu")
    rec = oracle.gated_linear_recurrence_backward(dout, x, gate, lengths, initial, dfinal)
    for loss, args, grads in ((norm_loss, (x, w, b), norm),
                              (recurrence_loss, (x, gate, initial), rec)):
        for k, grad in enumerate(grads):
            way = rng.normal(0, 1, grad.shape)
            up, down = list(args), list(args)
            up[k], down[k] = args[k] + step * way, args[k] - step * way
            slope = (loss(*up) - loss(*down)) / (2 * step)
            np.testing.assert_allclose((grad * way).sum(), slope, rtol=1e-6, atol=1e-8)
