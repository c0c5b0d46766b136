"""The global norm of a set of gradients, and their clipping by it, on torch
CUDA tensors: what a training step does between its backward pass and its
update.  No counterpart in the reference, which only infers."""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

from . import _lib
from .device import Device
from .layers import _native, _on_stream


def gradient_norm_workspace_bytes(count: int) -> int:
    out = ctypes.c_uint64()
    _lib.check(_lib.lib().af2_gradient_norm_workspace_bytes(count, ctypes.byref(out)))
    return int(out.value)


def encode_gradient_norm_tensors(device: Device, gradients: Sequence, *, stream: Optional[int] = None, workspace=None):
    """The square root of the sum of squares over all tensors, as an f32 scalar on the device."""
    norm = _native().gradients(device.handle.value, device.ordinal, list(gradients), None, None,
                               -1 if stream is None else stream, workspace)
    if stream is not None:
        _on_stream((norm,), device, stream)
    return norm


def encode_clip_gradients_tensors(device: Device, gradients: Sequence, max_norm: float, *, out: Optional[Sequence] = None,
                                  stream: Optional[int] = None, workspace=None):
    """Scales every tensor by min(1, max_norm / (norm + 1e-6)), in place or into the tensors of
    `out` (same sizes and types), and returns the norm before clipping, an f32 scalar on the device.
    Autograd does not record it.  Tensors that overlap where they are written are refused."""
    max_norm = float(max_norm)
    if not (max_norm >= 0 and math.isfinite(max_norm)):
        raise _lib.RangeError(f"max_norm must be finite and not negative; received {max_norm}")
    norm = _native().gradients(device.handle.value, device.ordinal, list(gradients), None if out is None else list(out),
                               max_norm, -1 if stream is None else stream, workspace)
    if stream is not None:
        _on_stream((norm,), device, stream)
    return norm
