"""Gated linear recurrence over ``[N, T, C]`` and its gradients, called on torch CUDA tensors
through the C ABI (``include/fga_convolution.h``).

A time mixer beside the depthwise convolution, with unbounded left context and a state of one
value per channel::

    f = sigmoid(gate);  h[t] = f[t] * h[t-1] + (1 - f[t]) * x[t];  out[t] = h[t]

The state is float32 and passes from call to call, so a recording may be cut anywhere; ``T =
1`` is the streaming step. ``valid_lengths`` is int32 ``[N]`` as in the convolutions, clamped
to ``[0, T]``: what padded frames hold is not used, they leave the state as it is, and padded
frames of the outputs are zeros. No reference plugin.

The operators record no autograd graph: a call on tensors that require grad is refused while
grad mode is on, and one on tensors that carry forward-mode tangents. The two functions are
the halves of a ``torch.autograd.Function``.

Tensors must be contiguous and live on the current CUDA device. Work is enqueued on
``stream`` (default: torch's current stream), outputs and workspace are allocated on it, and
nothing is synchronised. A ``workspace`` passed in must not serve two calls in flight; a few
long rows need one (``gated_linear_recurrence_workspace_size``), many or short rows none.
"""

from __future__ import annotations

import torch

from . import _lib
from ._call import Operator, descs, require

_FORWARD = Operator("gated_linear_recurrence",
                    ("x", "gate", "valid_lengths", "initial_state"),
                    ("out", "final_state", "states"))
_BACKWARD = Operator("gated_linear_recurrence_backward",
                     ("grad_out", "x", "gate", "valid_lengths", "states", "grad_final_state"),
                     ("grad_x", "grad_gate", "grad_initial_state"))

STATE_FRAMES = _lib.RECURRENCE_STATE_FRAMES


def gated_linear_recurrence_check(input_descs, output_descs) -> int:
    """Status of the shape and type checks (no device needed)."""
    return _lib.library().fga_gated_linear_recurrence_check(
        _lib.desc_array(input_descs), len(input_descs), _lib.desc_array(output_descs),
        len(output_descs))


def gated_linear_recurrence_backward_check(input_descs, output_descs) -> int:
    return _lib.library().fga_gated_linear_recurrence_backward_check(
        _lib.desc_array(input_descs), len(input_descs), _lib.desc_array(output_descs),
        len(output_descs))


def gated_linear_recurrence_workspace_size(x: torch.Tensor, valid_lengths: torch.Tensor) -> int:
    """Bytes of device memory that a forward call on ``x`` takes as ``workspace``."""
    state = (torch.float32, (x.shape[0], x.shape[2]))
    ins = descs([(x.dtype, x.shape)] * 2 + [(valid_lengths.dtype, valid_lengths.shape), state])
    return _lib.library().fga_gated_linear_recurrence_workspace_size(ins, 4)


def gated_linear_recurrence_backward_workspace_size(x: torch.Tensor,
                                                    valid_lengths: torch.Tensor) -> int:
    """Bytes of device memory that a backward call on ``x`` takes as ``workspace``."""
    n, t, c = x.shape
    ins = descs([(x.dtype, x.shape)] * 3 + [(valid_lengths.dtype, valid_lengths.shape),
                                            (torch.float32, (n, -(-t // STATE_FRAMES), c)),
                                            (torch.float32, (n, c))])
    return _lib.library().fga_gated_linear_recurrence_backward_workspace_size(ins, 6)


def _state_like(other, x):
    """A float32 ``[N, C]``: like ``other``, which the call's checks hold to that, if given (0.5
    us less than by shape)."""
    if other is not None:
        return torch.empty_like(other)
    return x.new_empty((x.shape[0], x.shape[2]), dtype=torch.float32)


def gated_linear_recurrence(x: torch.Tensor, gate: torch.Tensor, valid_lengths: torch.Tensor,
                            initial_state: torch.Tensor | None = None, *,
                            return_states: bool = False, out: torch.Tensor | None = None,
                            final_state: torch.Tensor | None = None, stream=None,
                            workspace: torch.Tensor | None = None):
    """``(out, final_state)``, or ``(out, final_state, states)`` with ``return_states``.

    ``gate`` holds logits; ``initial_state`` is float32 ``[N, C]`` (default zeros).
    ``final_state`` is the state after the last valid frame; a buffer may be passed for it,
    ``initial_state`` itself for an update in place. ``states`` (float32 ``[N, ceil(T / 64),
    C]``, the state before every 64th frame, zero where that frame is padding) is what the
    backward call takes."""
    require("x", x, 3)
    n, t, c = x.shape
    saved = (n, -(-t // STATE_FRAMES), c)

    def allocate():
        return (torch.empty_like(x) if out is None else out,
                _state_like(initial_state, x) if final_state is None else final_state,
                x.new_empty(saved, dtype=torch.float32) if return_states else None)

    outputs = _FORWARD((x, gate, valid_lengths, initial_state), (out, final_state), allocate,
                       lambda name: (torch.float32, saved if name == "states" else (n, c)),
                       workspace=workspace, stream=stream)
    return outputs if return_states else outputs[:2]


def gated_linear_recurrence_backward(grad_out: torch.Tensor, x: torch.Tensor,
                                     gate: torch.Tensor, valid_lengths: torch.Tensor,
                                     states: torch.Tensor,
                                     grad_final_state: torch.Tensor | None = None, *,
                                     stream=None, workspace: torch.Tensor | None = None):
    """``(grad_x, grad_gate, grad_initial_state)`` from the forward call's inputs and its
    ``states``. ``grad_final_state`` is float32 ``[N, C]`` (default zeros), and so is
    ``grad_initial_state``."""
    require("x", x, 3)
    n, _, c = x.shape
    return _BACKWARD((grad_out, x, gate, valid_lengths, states, grad_final_state), (),
                     lambda: (torch.empty_like(x), torch.empty_like(x),
                              _state_like(grad_final_state, x)),
                     lambda name: (torch.float32, (n, c)), workspace=workspace, stream=stream)
