"""One call of a C ABI entry point on torch CUDA tensors, for the operators whose bindings
include optional ones and a shape-dependent workspace (``normalization``, ``recurrence``).

A call whose GPU work takes a few microseconds is bound by what Python does around it. So what
follows from the shapes and types alone - the descriptor arrays, the workspace's size - is kept
for the next call of the same shapes and types; nothing is kept by address or identity.
"""

from __future__ import annotations

import ctypes
import struct
import threading

import torch
from torch.autograd import forward_ad

from . import _lib
from .attention import _check, _torch_stream, dtype_code

_MOST_PLANS = 1024
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _current_stream(device: int) -> int:
    if _raw_stream is not None:
        return _raw_stream(device)
    return torch.cuda.current_stream(device).cuda_stream


def require(name: str, t, rank: int) -> None:
    """What an output's shape is taken from has to be a tensor of that rank."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor (got {type(t).__name__})")
    if t.dim() != rank:
        raise _lib.AttentionError(_lib.STATUS_CODES["FGA_ERROR_BAD_DESCRIPTOR"],
                                  f"{name} of rank {t.dim()}")


def _dual() -> bool:
    """Whether tensors may carry forward-mode tangents."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def _has_tangent(t) -> bool:
    return forward_ad.unpack_dual(t).tangent is not None


def _refuse(name: str, t, device: int, grad: bool) -> None:
    """Why a binding cannot be launched on."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor (got {type(t).__name__})")
    if _dual() and _has_tangent(t):
        raise ValueError(f"{name} carries a forward-mode tangent, which this operator would lose: "
                         "call it on forward_ad.unpack_dual(...).primal")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (got {t.device})")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous (row-major linear)")
    if grad and t.requires_grad:
        raise ValueError(f"{name} requires grad: this operator records no autograd graph; call "
                         "it under torch.no_grad() and use its backward function")


def descs(bindings):
    """Descriptor array of ``(dtype, shape)`` bindings."""
    return _lib.desc_array([_lib.TensorDesc.make(dtype_code(d), s) for d, s in bindings])


def _by_address(name: str):
    """An entry point that takes its arrays as addresses or bytes: ctypes spends less on those
    than on typed pointers (a call refused by the library: 7.2 us and 3.5)."""
    _, argtypes = _lib.SYMBOLS[name]
    fn = _lib.library()[name]
    fn.restype = ctypes.c_int32
    fn.argtypes = [ctypes.c_void_p if hasattr(a, "contents") else a for a in argtypes]
    return fn


class _Plan:
    """What a call takes that follows from its shapes and types."""

    __slots__ = ("ins", "outs", "workspace", "_keep")

    def __init__(self, ins, outs, workspace: int):
        self.ins, self.outs, self.workspace = ctypes.addressof(ins), ctypes.addressof(outs), workspace
        self._keep = (ins, outs)


class Operator:
    """The entry point ``fga_<name>_enqueue`` with its bindings' names."""

    def __init__(self, name: str, inputs: tuple[str, ...], outputs: tuple[str, ...]):
        self.name, self.inputs, self.outputs = name, inputs, outputs
        self._pack_in = struct.Struct(f"{len(inputs)}Q").pack
        self._pack_out = struct.Struct(f"{len(outputs)}Q").pack
        self._enqueue = None
        self._plans: dict = {}
        self._lock = threading.Lock()

    def __call__(self, tensors, given, allocate, absent, fields=(), size_fields=(), workspace=None,
                 stream=None):
        """Enqueue on ``tensors`` (None: an optional binding that is not given) and return the
        outputs: those ``given``, and ``allocate()``'s where that has None (None there as well:
        not wanted). ``absent(name)`` is the ``(dtype, shape)`` of a binding without a buffer.
        Outputs and workspace are allocated with the launch's stream as torch's current one."""
        device = torch.cuda.current_device()
        if stream is None:
            return self._launch(tensors, given, allocate, absent, fields, size_fields, workspace,
                                device, _current_stream(device))
        stream = _torch_stream(stream)
        if stream.device.index != device:
            # torch would make that device the current one for the launch.
            raise ValueError(f"stream is on {stream.device}, the current device is cuda:{device}")
        with torch.cuda.stream(stream):
            return self._launch(tensors, given, allocate, absent, fields, size_fields, workspace,
                                device, stream.cuda_stream)

    def _launch(self, tensors, given, allocate, absent, fields, size_fields, workspace, device,
                handle):
        grad, dual = torch.is_grad_enabled(), _dual()
        key, sources, i = [device, size_fields], [], 0
        for t in tensors:
            if t is None:
                sources.append(0)
                key.append(None)
            else:
                if (not isinstance(t, torch.Tensor) or t.get_device() != device
                        or not t.is_contiguous() or (grad and t.requires_grad)
                        or (dual and _has_tangent(t))):
                    _refuse(self.inputs[i], t, device, grad)
                sources.append(t.data_ptr())
                key.append(t.dtype)
                key.append(t.shape)
            i += 1
        i = 0
        for t in given:
            if t is None:
                key.append(None)
            else:
                if (not isinstance(t, torch.Tensor) or t.get_device() != device
                        or not t.is_contiguous() or (grad and t.requires_grad)
                        or (dual and _has_tangent(t))):
                    _refuse(self.outputs[i], t, device, grad)
                key.append(t.dtype)
                key.append(t.shape)
            i += 1
        outputs = allocate()
        targets = [0 if t is None else t.data_ptr() for t in outputs]
        key = tuple(key)
        plan = self._plans.get(key) or self._plan(key, tensors, outputs, absent, size_fields)
        size = plan.workspace
        address = None
        if size:
            if workspace is None:
                workspace = tensors[0].new_empty(size, dtype=torch.uint8)
            elif (not isinstance(workspace, torch.Tensor) or workspace.get_device() != device
                  or not workspace.is_contiguous()):
                raise ValueError("workspace must be a contiguous CUDA tensor on the current device")
            else:
                size = workspace.numel() * workspace.element_size()
            address = workspace.data_ptr()
        if self._enqueue is None:
            self._enqueue = _by_address(f"fga_{self.name}_enqueue")
        status = self._enqueue(plan.ins, plan.outs, self._pack_in(*sources),
                               self._pack_out(*targets), *fields, address, size, handle)
        if status:
            _check(status, self.name)
        return outputs

    def _plan(self, key, tensors, outputs, absent, size_fields):
        """Descriptors and workspace size of a call's shapes and types. The outputs' follow from
        the key: they are given, or shaped after an input."""
        def bindings(ts, names):
            return [absent(n) if t is None else (t.dtype, t.shape) for t, n in zip(ts, names)]

        ins, outs = descs(bindings(tensors, self.inputs)), descs(bindings(outputs, self.outputs))
        size = getattr(_lib.library(), f"fga_{self.name}_workspace_size")(
            ins, len(tensors), *size_fields)
        with self._lock:
            if len(self._plans) >= _MOST_PLANS:
                self._plans.clear()
            plan = self._plans[key] = _Plan(ins, outs, size)
        return plan
