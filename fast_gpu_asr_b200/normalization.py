"""Group norm with an activation over ``[N, T, C]`` and its gradients, called on torch CUDA
tensors through the C ABI (``include/fga_convolution.h``).

For convolution modules whose norm cannot be folded into the depthwise convolution's weights,
because its statistics come from the utterance itself: group norm, and with one group or one
channel per group the layer and instance forms over time. No reference plugin.

``valid_lengths`` is int32 ``[N]`` as in the convolutions, clamped to ``[0, T]``: statistics
and gradients cover the valid frames, padded frames are not read, and padded frames of
``out`` and ``grad_x`` are zeros. All arithmetic is fp32, with one rounding at the store.

The operators record no autograd graph: a call on tensors that require grad is refused while
grad mode is on. The two functions are the halves of a ``torch.autograd.Function``.

Tensors must be contiguous and live on the current CUDA device. Work is enqueued on
``stream`` (default: torch's current stream), outputs and workspace are allocated on it, and
nothing is synchronised. A ``workspace`` passed in must not serve two calls in flight.
"""

from __future__ import annotations

import torch

from . import _lib
from ._call import Absent, descs, enqueue, launch_stream, require


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
        descs((x, valid_lengths, weight, bias)), 4, int(num_groups))


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
    handle, context = launch_stream(stream)
    shape = (x.shape[0], num_groups)
    with context:
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        if return_statistics and num_groups > 0:
            mean = torch.empty(shape, dtype=torch.float32, device=x.device)
            rstd = torch.empty(shape, dtype=torch.float32, device=x.device)
        else:
            mean = rstd = Absent(torch.float32, shape)
    enqueue("group_norm_activation", (x, valid_lengths, weight, bias),
            ("x", "valid_lengths", "weight", "bias"), (out, mean, rstd), ("out", "mean", "rstd"),
            (num_groups, float(eps), _activation(activation)), workspace, handle, context,
            size_fields=(num_groups,))
    return (out, mean, rstd) if return_statistics else out


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
    handle, context = launch_stream(stream)
    with context:
        outputs = tuple(torch.empty_like(t, memory_format=torch.contiguous_format)
                        for t in (x, weight, bias))
    enqueue("group_norm_activation_backward",
            (grad_out, x, valid_lengths, weight, bias, mean, rstd),
            ("grad_out", "x", "valid_lengths", "weight", "bias", "mean", "rstd"), outputs,
            ("grad_x", "grad_weight", "grad_bias"), (_activation(activation),), workspace,
            handle, context)
    return outputs
