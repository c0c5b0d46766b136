"""Layers with learned weights on torch CUDA tensors: the dense layer and the
gated transition, each with its backward pass.

    y, saved = encode_dense_tensors(device, x, weight, bias=b, activation="gelu", save=True)
    grads = encode_dense_backward_tensors(device, d_y, x, weight, saved=saved, bias=True, activation="gelu")

Every tensor of a call has one type (float32, float16 or bfloat16); weights
are [in, out] and used as they are stored, so they may change between calls.
Activations, residuals and outputs are [rows, width] with any row stride of at
least the width.  Calls run on torch's current stream unless ``stream`` names
another (a raw CUDA stream handle; 0 is the device context's own stream); a
named stream does not wait for the current one, so the inputs must be ready on it.
Autograd does not record the calls: results are detached, also from tensors that
require gradients, and the backward passes are called by hand.

No counterpart in the reference, whose weights are fixed and whose transition
is ReLU (src/evoformer/transition.ts); the weights' names follow its
firstWeight / firstBias style.
"""
from __future__ import annotations

import ctypes
from typing import Optional

from . import _lib
from .device import Device

_DTYPES = {"torch.float32": _lib.AF2_F32, "torch.float16": _lib.AF2_F16, "torch.bfloat16": _lib.AF2_BF16}
ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2, "silu": 3, "gelu": 4}
GATED_WEIGHTS = ("gateWeight", "gateBias", "valueWeight", "valueBias", "outputWeight", "outputBias")
_BOUND = ("af2_dense_saved_bytes", "af2_dense_workspace_bytes", "af2_dense", "af2_dense_backward",
          "af2_gated_transition_saved_bytes", "af2_gated_transition_workspace_bytes", "af2_gated_transition",
          "af2_gated_transition_backward", "af2_gradient_norm_workspace_bytes", "af2_gradient_norm",
          "af2_clip_gradients")
_BOTH = ("x", "weight")
_tensors = None


def _native():
    """The compiled torch glue (_tensors.cpp), bound to the loaded library's entry points."""
    global _tensors
    if _tensors is None:
        import torch  # noqa: F401  (its libraries are what the module links)
        try:
            from . import _tensors as module
        except ImportError as e:
            raise OSError("af2cuda/_tensors.so is missing or was built against another torch; build it with "
                          "`python alphafold2-webgpu_b200/build.py`") from e
        lib = _lib.lib()
        module.bind({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _BOUND},
                    _lib.RangeError, lambda status, ctx: _lib.check(status, ctypes.c_void_p(ctx)))
        _tensors = module
    return _tensors


def _dtype_code(dtype) -> int:
    code = _DTYPES.get(str(dtype))
    if code is None:
        raise _lib.RangeError(f"tensors must be float32, float16 or bfloat16; received {dtype}")
    return code


def _activation_code(activation: str) -> int:
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise _lib.RangeError(f"activation must be one of {', '.join(ACTIVATIONS)}; received {activation}")
    return code


def _needed(need, known) -> set:
    names = {need} if isinstance(need, str) else set(need)
    if not names <= set(known):
        raise _lib.RangeError(f"need names {', '.join(sorted(map(str, names - set(known))))}; "
                              f"expected some of {', '.join(known)}")
    return names


def _on_stream(tensors, device: Device, stream: int) -> None:
    """Keeps tensors that were written on a named stream from reuse until it, and torch's current stream,
    where the caller will read them, have passed.  (New ones were allocated on the named stream.)"""
    if stream == 0:  # the context's own stream: torch's allocator cannot follow it
        device.sync()
        return
    import torch
    where = torch.device("cuda", device.ordinal)
    streams = (torch.cuda.ExternalStream(stream, device=where), torch.cuda.current_stream(where))
    for t in tensors:
        for s in streams:
            t.record_stream(s)


def dense_saved_bytes(rows: int, inner: int, columns: int, dtype, activation: str = "none") -> int:
    out = ctypes.c_uint64()
    _lib.check(_lib.lib().af2_dense_saved_bytes(ctypes.byref(_lib.LinearShape(rows, inner, columns)),
                                                _dtype_code(dtype), _activation_code(activation), ctypes.byref(out)))
    return int(out.value)


def dense_workspace_bytes(rows: int, inner: int, columns: int, dtype, activation: str = "none",
                          backward: bool = False) -> int:
    out = ctypes.c_uint64()
    _lib.check(_lib.lib().af2_dense_workspace_bytes(ctypes.byref(_lib.LinearShape(rows, inner, columns)),
                                                    _dtype_code(dtype), _activation_code(activation),
                                                    1 if backward else 0, ctypes.byref(out)))
    return int(out.value)


def gated_transition_saved_bytes(rows: int, channels: int, hidden: int, dtype) -> int:
    out = ctypes.c_uint64()
    _lib.check(_lib.lib().af2_gated_transition_saved_bytes(ctypes.byref(_lib.TransitionShape(rows, channels, hidden)),
                                                           _dtype_code(dtype), ctypes.byref(out)))
    return int(out.value)


def gated_transition_workspace_bytes(rows: int, channels: int, hidden: int, dtype, backward: bool = False) -> int:
    out = ctypes.c_uint64()
    _lib.check(_lib.lib().af2_gated_transition_workspace_bytes(
        ctypes.byref(_lib.TransitionShape(rows, channels, hidden)), _dtype_code(dtype), 1 if backward else 0,
        ctypes.byref(out)))
    return int(out.value)


def encode_dense_tensors(device: Device, x, weight, *, bias=None, residual=None, activation: str = "none", out=None,
                         save: bool = False, stream: Optional[int] = None, workspace=None):
    """out = act(x weight + bias) (+ residual): x [rows, inner], weight [inner, columns], bias
    [columns], residual and out [rows, columns] (out may be the residual).  Returns out, or with
    save=True (out, saved), saved being what encode_dense_backward_tensors takes."""
    result = (_tensors or _native()).dense(device.handle.value, device.ordinal, x, weight, bias, residual,
                                           _activation_code(activation), out, save, -1 if stream is None else stream,
                                           workspace)
    if stream is not None:
        _on_stream(result if save else (result,), device, stream)
    return result


def encode_dense_backward_tensors(device: Device, d_out, x, weight, *, saved=None, bias: bool = False,
                                  activation: str = "none", need=_BOTH, stream: Optional[int] = None,
                                  workspace=None) -> dict:
    """Gradients of encode_dense_tensors for d_out [rows, columns]: {"x", "weight"}, those of them
    that `need` names, and "bias" with bias=True.  The residual's gradient is d_out itself."""
    if need is not _BOTH:
        need = _needed(need, ("x", "weight", "bias") if bias else _BOTH)
    grads = (_tensors or _native()).dense_backward(device.handle.value, device.ordinal, d_out, x, weight, saved, bias,
                                                   _activation_code(activation), "x" in need, "weight" in need,
                                                   -1 if stream is None else stream, workspace)
    if stream is not None:
        _on_stream(grads.values(), device, stream)
    return grads


def encode_gated_transition_tensors(device: Device, x, weights: dict, *, residual=None, activation: str = "silu",
                                    out=None, save: bool = False, stream: Optional[int] = None, workspace=None):
    """out = (act(x gateWeight + gateBias) * (x valueWeight + valueBias)) outputWeight + outputBias
    (+ residual): x, residual and out [rows, channels] (out may be the residual, and x), gateWeight and
    valueWeight [channels, hidden], outputWeight [hidden, channels]; the biases may be absent.
    Returns out, or with save=True (out, saved) for encode_gated_transition_backward_tensors."""
    result = (_tensors or _native()).gated(device.handle.value, device.ordinal, x, weights, residual,
                                           _activation_code(activation), out, save, -1 if stream is None else stream,
                                           workspace)
    if stream is not None:
        _on_stream(result if save else (result,), device, stream)
    return result


def encode_gated_transition_backward_tensors(device: Device, d_out, x, weights: dict, *, saved,
                                             activation: str = "silu", need=None, stream: Optional[int] = None,
                                             workspace=None) -> dict:
    """Gradients of encode_gated_transition_tensors for d_out [rows, channels]: "x" and every
    weight given, by its name, or those of them that `need` names.  The residual's gradient is d_out itself."""
    if need is not None:
        need = _needed(need, ("x", *GATED_WEIGHTS))
    grads = (_tensors or _native()).gated_backward(device.handle.value, device.ordinal, d_out, x, weights, saved,
                                                   _activation_code(activation), need,
                                                   -1 if stream is None else stream, workspace)
    if stream is not None:
        _on_stream(grads.values(), device, stream)
    return grads
