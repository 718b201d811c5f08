"""Group norm with an activation over ``[N, T, C]`` and its gradients, called on torch CUDA
tensors through the C ABI (``include/fga_convolution.h``).

For convolution modules whose norm cannot be folded into the depthwise convolution's weights,
because its statistics come from the utterance itself: group norm, and with one group or one
channel per group the layer and instance forms over time. No reference plugin.

``valid_lengths`` is int32 ``[N]`` as in the convolutions, clamped to ``[0, T]``: statistics
and gradients cover the valid frames, what padded frames hold is not used, and padded frames
of ``out`` and ``grad_x`` are zeros. All arithmetic is fp32, with one rounding at the store.

The operators record no autograd graph: a call on tensors that require grad is refused while
grad mode is on, and one on tensors that carry forward-mode tangents. The two functions are
the halves of a ``torch.autograd.Function``.

Tensors must be contiguous and live on the current CUDA device. Work is enqueued on
``stream`` (default: torch's current stream), outputs and workspace are allocated on it, and
nothing is synchronised. A ``workspace`` passed in must not serve two calls in flight.
"""

from __future__ import annotations

import torch

from . import _lib
from ._call import Operator, descs, require

_FORWARD = Operator("group_norm_activation", ("x", "valid_lengths", "weight", "bias"),
                    ("out", "mean", "rstd"))
_BACKWARD = Operator("group_norm_activation_backward",
                     ("grad_out", "x", "valid_lengths", "weight", "bias", "mean", "rstd"),
                     ("grad_x", "grad_weight", "grad_bias"))


def _activation(name) -> int:
    """The ``fga_activation`` value, -1 (which the C ABI refuses) for an unknown name."""
    return _lib.ACTIVATIONS.get(name, -1) if isinstance(name, str) else -1


def group_norm_activation_check(input_descs, output_descs, num_groups: int, eps: float,
                                activation: str) -> int:
    """Status of the shape, type and field checks (no device needed)."""
    return _lib.library().fga_group_norm_activation_check(
        _lib.desc_array(input_descs), len(input_descs), _lib.desc_array(output_descs),
        len(output_descs), int(num_groups), float(eps), _activation(activation))


def group_norm_activation_backward_check(input_descs, output_descs, activation: str) -> int:
    return _lib.library().fga_group_norm_activation_backward_check(
        _lib.desc_array(input_descs), len(input_descs), _lib.desc_array(output_descs),
        len(output_descs), _activation(activation))


def group_norm_activation_workspace_size(x: torch.Tensor, valid_lengths: torch.Tensor,
                                         weight: torch.Tensor, bias: torch.Tensor,
                                         num_groups: int) -> int:
    """Bytes of device memory that a call with these bindings takes as ``workspace``."""
    return _lib.library().fga_group_norm_activation_workspace_size(
        descs([(t.dtype, t.shape) for t in (x, valid_lengths, weight, bias)]), 4, int(num_groups))


def group_norm_activation_backward_workspace_size(x: torch.Tensor, valid_lengths: torch.Tensor,
                                                  weight: torch.Tensor, bias: torch.Tensor,
                                                  num_groups: int) -> int:
    """Bytes of device memory that a backward call with these bindings takes as ``workspace``."""
    stats = (torch.float32, (x.shape[0], int(num_groups)))
    ins = [(t.dtype, t.shape) for t in (x, x, valid_lengths, weight, bias)] + [stats] * 2
    return _lib.library().fga_group_norm_activation_backward_workspace_size(descs(ins), 7)


def group_norm_activation(x: torch.Tensor, valid_lengths: torch.Tensor, weight: torch.Tensor,
                          bias: torch.Tensor, num_groups: int, *, eps: float = 1e-5,
                          activation: str = "silu", return_statistics: bool = False,
                          out: torch.Tensor | None = None, stream=None,
                          workspace: torch.Tensor | None = None):
    """``act((x - mean) rstd weight + bias)`` with each group's mean and rstd over the valid
    frames of its utterance, ``[N, T, C]``.

    ``activation`` is ``"none"``, ``"silu"`` or ``"swoosh_r"``; ``weight`` and ``bias`` are
    ``[C]`` of ``x``'s type. With ``return_statistics``: ``(out, mean, rstd)``, the latter
    float32 ``[N, num_groups]``, which the backward call takes."""
    require("x", x, 3)
    num_groups = int(num_groups)

    def allocate():
        y = torch.empty_like(x) if out is None else out
        if not return_statistics or num_groups < 1:
            return y, None, None
        shape = (x.shape[0], num_groups)
        return y, x.new_empty(shape, dtype=torch.float32), x.new_empty(shape, dtype=torch.float32)

    outputs = _FORWARD((x, valid_lengths, weight, bias), (out,), allocate,
                       lambda name: (torch.float32, (x.shape[0], num_groups)),
                       (num_groups, float(eps), _activation(activation)), (num_groups,),
                       workspace, stream)
    return outputs if return_statistics else outputs[0]


def group_norm_activation_backward(grad_out: torch.Tensor, x: torch.Tensor,
                                   valid_lengths: torch.Tensor, weight: torch.Tensor,
                                   bias: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, *,
                                   activation: str = "silu", stream=None,
                                   workspace: torch.Tensor | None = None):
    """``(grad_x, grad_weight, grad_bias)`` from the forward call's inputs and its ``mean``
    and ``rstd`` (which give the number of groups). The parameters' gradients are sums over
    the batch, in the parameters' type."""
    require("x", x, 3)
    require("weight", weight, 1)
    require("bias", bias, 1)
    return _BACKWARD((grad_out, x, valid_lengths, weight, bias, mean, rstd), (),
                     lambda: (torch.empty_like(x), torch.empty_like(weight),
                              torch.empty_like(bias)),
                     None, (_activation(activation),), (), workspace, stream)
