"""One call of a C ABI entry point on torch CUDA tensors, for the operators whose bindings
include optional ones and a shape-dependent workspace (``normalization``, ``recurrence``).

A call of a few microseconds of GPU work is bound by what Python does around it, so the
descriptor arrays of a set of shapes and types are built once and reused; they hold no
address.
"""

from __future__ import annotations

import contextlib
from functools import lru_cache

import torch

from . import _lib
from .attention import _check, _torch_stream, _workspace, dtype_code


class Absent:
    """An optional binding that is not given: its descriptor without a buffer."""

    __slots__ = ("dtype", "shape")

    def __init__(self, dtype: torch.dtype, shape):
        self.dtype, self.shape = dtype, tuple(shape)


@lru_cache(maxsize=1024)
def _descs(spec):
    return _lib.desc_array([_lib.TensorDesc.make(dtype_code(d), s) for d, s in spec])


def descs(tensors):
    """Descriptor array of tensors, ``Absent`` bindings among them (shared: read only)."""
    return _descs(tuple([(t.dtype, t.shape) for t in tensors]))


def require(name: str, t, rank: int) -> None:
    """What an output's shape is taken from has to be a tensor of that rank."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor (got {type(t).__name__})")
    if t.dim() != rank:
        raise _lib.AttentionError(_lib.STATUS_CODES["FGA_ERROR_BAD_DESCRIPTOR"],
                                  f"{name} of rank {t.dim()}")


def _pointer(t, name: str, device: int, grad: bool):
    if isinstance(t, Absent):
        return None
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor (got {type(t).__name__})")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (got {t.device})")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous (row-major linear)")
    if grad and t.requires_grad:
        raise ValueError(f"{name} requires grad: this operator records no autograd graph; call "
                         "it under torch.no_grad() and use its backward function")
    return t.data_ptr()


def pointers(tensors, names):
    device = torch.cuda.current_device()
    grad = torch.is_grad_enabled()
    return _lib.pointer_array([_pointer(t, n, device, grad) for t, n in zip(tensors, names)])


def launch_stream(stream):
    """``(handle, context)``: the ``cudaStream_t`` of the launch, and the context in which
    outputs and workspace are allocated, so that they belong to that stream."""
    if stream is None:
        return torch.cuda.current_stream().cuda_stream, contextlib.nullcontext()
    stream = _torch_stream(stream)
    return stream.cuda_stream, torch.cuda.stream(stream)


def enqueue(op: str, tensors, names, outputs, out_names, fields, workspace, stream, context,
            size_fields=()):
    """Size the workspace and enqueue ``fga_<op>_enqueue``; raise on a nonzero status."""
    lib = _lib.library()
    ins, outs = descs(tensors), descs(outputs)
    in_ptrs, out_ptrs = pointers(tensors, names), pointers(outputs, out_names)
    size = getattr(lib, f"fga_{op}_workspace_size")(ins, len(tensors), *size_fields)
    ws, ws_bytes = None, 0
    if size:
        with context:
            ws, ws_bytes = _workspace(size, tensors[0].device, workspace, None)
    status = getattr(lib, f"fga_{op}_enqueue")(ins, outs, in_ptrs, out_ptrs, *fields, ws,
                                               ws_bytes, stream)
    if status:
        _check(status, op)
