"""The global norm of a set of gradients, and their clipping by it, on torch
CUDA tensors: what a training step does between its backward pass and its
update.  No counterpart in the reference, which only infers."""
from __future__ import annotations

import math
from array import array
from typing import Optional, Sequence

from . import _lib
from .device import Device
from .layers import _dtype_code, _on_stream, _stream_handle, _workspace


def _refs(name: str, tensors: Sequence, device: Device) -> array:
    """The af2_tensor_ref array of a set: (address, count, dtype) as three 64-bit words each."""
    words = array("q", bytes(24 * len(tensors)))
    for i, t in enumerate(tensors):
        if t.get_device() != device.ordinal or not t.is_contiguous():
            raise _lib.RangeError(f"{name} {i} must be a contiguous tensor on cuda:{device.ordinal}")
        words[3 * i] = t.data_ptr()
        words[3 * i + 1] = t.numel()
        words[3 * i + 2] = _dtype_code(t.dtype)
    return words


def gradient_norm_workspace_bytes(count: int) -> int:
    import ctypes
    out = ctypes.c_uint64()
    _lib.check(_lib.lib().af2_gradient_norm_workspace_bytes(count, ctypes.byref(out)))
    return int(out.value)


def _norm_out(device: Device):
    import torch
    return torch.empty((), dtype=torch.float32, device=torch.device("cuda", device.ordinal))


def encode_gradient_norm_tensors(device: Device, gradients: Sequence, *, stream: Optional[int] = None, workspace=None):
    """The square root of the sum of squares over all tensors, as an f32 scalar on the device."""
    gradients = list(gradients)
    refs = _refs("gradient", gradients, device)
    norm = _norm_out(device)
    ws = _workspace(workspace, lambda: gradient_norm_workspace_bytes(len(gradients)), device)
    status = _lib.lib().af2_gradient_norm(device.handle, refs.buffer_info()[0], len(gradients), norm.data_ptr(), ws,
                                          _stream_handle(device, stream))
    _lib.check(status, device.handle)
    _on_stream([norm], device, stream)
    return norm


def encode_clip_gradients_tensors(device: Device, gradients: Sequence, max_norm: float, *, out: Optional[Sequence] = None,
                                  stream: Optional[int] = None, workspace=None):
    """Scales every tensor by min(1, max_norm / (norm + 1e-6)), in place or into the tensors of
    `out` (same sizes and types), and returns the norm before clipping, an f32 scalar on the device."""
    gradients = list(gradients)
    max_norm = float(max_norm)
    if not (max_norm >= 0 and math.isfinite(max_norm)):
        raise _lib.RangeError(f"max_norm must be finite and not negative; received {max_norm}")
    refs = _refs("gradient", gradients, device)
    outs = None
    if out is not None:
        out = list(out)
        if len(out) != len(gradients):
            raise _lib.RangeError(f"out has {len(out)} tensors; expected {len(gradients)}")
        outs = _refs("out", out, device)
    norm = _norm_out(device)
    ws = _workspace(workspace, lambda: gradient_norm_workspace_bytes(len(gradients)), device)
    status = _lib.lib().af2_clip_gradients(device.handle, refs.buffer_info()[0],
                                           outs.buffer_info()[0] if outs is not None else None, len(gradients),
                                           max_norm, norm.data_ptr(), ws, _stream_handle(device, stream))
    _lib.check(status, device.handle)
    _on_stream([norm], device, stream)
    return norm
