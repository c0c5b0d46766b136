"""Layers with learned weights on torch CUDA tensors: the dense layer and the
gated transition, each with its backward pass.

    y, saved = encode_dense_tensors(device, x, weight, bias=b, activation="gelu", save=True)
    grads = encode_dense_backward_tensors(device, d_y, x, weight, saved=saved, bias=True, activation="gelu")

Every tensor of a call has one type (float32, float16 or bfloat16); weights
are [in, out] and used as they are stored, so they may change between calls.
Activations, residuals and outputs are [rows, width] with any row stride of at
least the width.  Calls run on torch's current stream unless ``stream`` names
another (a raw CUDA stream handle; 0 is the device context's own stream).

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
_codes: dict = {}  # torch dtype -> af2_dtype, filled as types are met
_LEGACY_STREAM = 1  # cudaStreamLegacy: torch's default stream by its explicit handle


def _dtype_code(dtype) -> int:
    code = _codes.get(dtype)
    if code is None:
        code = _DTYPES.get(str(dtype))
        if code is None:
            raise _lib.RangeError(f"tensors must be float32, float16 or bfloat16; received {dtype}")
        _codes[dtype] = code
    return code


def _activation_code(activation: str) -> int:
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise _lib.RangeError(f"activation must be one of {', '.join(ACTIVATIONS)}; received {activation}")
    return code


def _stream_handle(device: Device, stream: Optional[int]):
    """The handle to pass: torch's current stream for None (its default stream is the null
    handle, which the library takes for the context's own), else the caller's."""
    if stream is None:
        import torch
        return torch._C._cuda_getCurrentRawStream(device.ordinal) or _LEGACY_STREAM
    return stream or None


def _rows(name: str, t, device: Device, dtype, rows: Optional[int], width: int) -> int:
    """Checks a [rows, width] tensor and returns its row stride."""
    if t.dim() != 2 or t.shape[1] != width or (rows is not None and t.shape[0] != rows):
        raise _lib.RangeError(f"{name} has shape {tuple(t.shape)}; expected ({'rows' if rows is None else rows}, {width})")
    if t.dtype != dtype or t.get_device() != device.ordinal:
        raise _lib.RangeError(f"{name} must be a {dtype} tensor on cuda:{device.ordinal}")
    if t.is_contiguous():
        return width
    if (t.stride(1) != 1 and width > 1) or (t.stride(0) < width and t.shape[0] > 1):
        raise _lib.RangeError(f"{name} must have contiguous rows a width or more apart; its strides are {t.stride()}")
    return max(t.stride(0), width)


def _whole(name: str, t, device: Device, dtype, shape: tuple) -> int:
    """Checks a contiguous tensor of the given shape and returns its address."""
    if tuple(t.shape) != shape:
        raise _lib.RangeError(f"{name} has shape {tuple(t.shape)}; expected {shape}")
    if t.dtype != dtype or t.get_device() != device.ordinal or not t.is_contiguous():
        raise _lib.RangeError(f"{name} must be a contiguous {dtype} tensor on cuda:{device.ordinal}")
    return t.data_ptr()


def _on_stream(tensors, device: Device, stream: Optional[int]) -> None:
    """New tensors written on a stream that is not torch's current one are kept from reuse until it has passed."""
    if stream is None:
        return
    import torch
    if stream == 0:  # the context's own stream has no torch object: the device's allocator cannot follow it
        device.sync()
        return
    for t in tensors:
        if t is not None:
            t.record_stream(torch.cuda.ExternalStream(stream, device=torch.device("cuda", device.ordinal)))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _saved(device: Device, nbytes: int):
    import torch
    return torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", device.ordinal))


def _check_saved(saved, nbytes: int, device: Device) -> int:
    if saved is None or saved.get_device() != device.ordinal or not saved.is_contiguous() \
            or saved.numel() * saved.element_size() < nbytes:
        raise _lib.RangeError(f"saved must be what the forward pass returned ({nbytes} bytes on cuda:{device.ordinal})")
    return saved.data_ptr()


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


def _workspace(workspace, need, device: Device):
    if workspace is None:
        return None
    nbytes = need()
    if workspace.get_device() != device.ordinal or not workspace.is_contiguous() \
            or workspace.numel() * workspace.element_size() < nbytes:
        raise _lib.RangeError(f"workspace must hold {nbytes} bytes on cuda:{device.ordinal}")
    return workspace.data_ptr()


def encode_dense_tensors(device: Device, x, weight, *, bias=None, residual=None, activation: str = "none", out=None,
                         save: bool = False, stream: Optional[int] = None, workspace=None):
    """out = act(x weight + bias) (+ residual): x [rows, inner], weight [inner, columns], bias
    [columns], residual and out [rows, columns] (out may be the residual).  Returns out, or with
    save=True (out, saved), saved being what encode_dense_backward_tensors takes."""
    import torch
    if weight.dim() != 2:
        raise _lib.RangeError(f"weight has shape {tuple(weight.shape)}; expected (inner, columns)")
    inner, columns = weight.shape
    dtype = x.dtype
    code, act = _dtype_code(dtype), _activation_code(activation)
    x_stride = _rows("x", x, device, dtype, None, inner)
    rows = x.shape[0]
    w = _whole("weight", weight, device, dtype, (inner, columns))
    b = None if bias is None else _whole("bias", bias, device, dtype, (columns,))
    r_stride = columns if residual is None else _rows("residual", residual, device, dtype, rows, columns)
    new = []
    if out is None:
        out, out_stride = torch.empty((rows, columns), dtype=dtype, device=x.device), columns
        new.append(out)
    else:
        out_stride = _rows("out", out, device, dtype, rows, columns)
    saved = None
    if save:
        saved = _saved(device, dense_saved_bytes(rows, inner, columns, dtype, activation))
        new.append(saved)
    ws = _workspace(workspace, lambda: dense_workspace_bytes(rows, inner, columns, dtype, activation), device)
    shape = _lib.LinearShape(rows, inner, columns)
    opts = _lib.LayerOptions(act, 0, x_stride, r_stride, out_stride, x_stride)
    status = _lib.lib().af2_dense(device.handle, ctypes.byref(shape), code, x.data_ptr(), w, b, _ptr(residual),
                                  ctypes.byref(opts), out.data_ptr(),
                                  saved.data_ptr() if saved is not None and saved.numel() else None, ws,
                                  _stream_handle(device, stream))
    _lib.check(status, device.handle)
    _on_stream(new, device, stream)
    return (out, saved) if save else out


def encode_dense_backward_tensors(device: Device, d_out, x, weight, *, saved=None, bias: bool = False,
                                  activation: str = "none", need=("x", "weight"), stream: Optional[int] = None,
                                  workspace=None) -> dict:
    """Gradients of encode_dense_tensors for d_out [rows, columns]: {"x", "weight"}, those of them
    that `need` names, and "bias" with bias=True.  The residual's gradient is d_out itself."""
    import torch
    if weight.dim() != 2:
        raise _lib.RangeError(f"weight has shape {tuple(weight.shape)}; expected (inner, columns)")
    inner, columns = weight.shape
    dtype = x.dtype
    code, act = _dtype_code(dtype), _activation_code(activation)
    x_stride = _rows("x", x, device, dtype, None, inner)
    rows = x.shape[0]
    d_stride = _rows("d_out", d_out, device, dtype, rows, columns)
    w = _whole("weight", weight, device, dtype, (inner, columns))
    kept = None
    if act:
        kept = _check_saved(saved, dense_saved_bytes(rows, inner, columns, dtype, activation), device)
    grads = {}
    if "x" in need:
        grads["x"] = torch.empty((rows, inner), dtype=dtype, device=x.device)
    if "weight" in need:
        grads["weight"] = torch.empty((inner, columns), dtype=dtype, device=x.device)
    if bias:
        grads["bias"] = torch.empty((columns,), dtype=dtype, device=x.device)
    ws = _workspace(workspace, lambda: dense_workspace_bytes(rows, inner, columns, dtype, activation, True), device)
    shape = _lib.LinearShape(rows, inner, columns)
    opts = _lib.LayerOptions(act, 0, x_stride, columns, d_stride, inner)
    status = _lib.lib().af2_dense_backward(device.handle, ctypes.byref(shape), code, d_out.data_ptr(), x.data_ptr(), w,
                                           kept, ctypes.byref(opts), _ptr(grads.get("x")), _ptr(grads.get("weight")),
                                           _ptr(grads.get("bias")), ws, _stream_handle(device, stream))
    _lib.check(status, device.handle)
    _on_stream(grads.values(), device, stream)
    return grads


def _gated_weights(weights: dict, device: Device, dtype):
    unknown = [k for k in weights if k not in GATED_WEIGHTS]
    if unknown:
        raise _lib.RangeError(f"unknown weights {unknown}; expected {', '.join(GATED_WEIGHTS)}")
    for k in ("gateWeight", "valueWeight", "outputWeight"):
        if weights.get(k) is None:
            raise _lib.RangeError(f"{k} is missing")
    if weights["gateWeight"].dim() != 2:
        raise _lib.RangeError(f"gateWeight has shape {tuple(weights['gateWeight'].shape)}; expected (channels, hidden)")
    c, h = weights["gateWeight"].shape
    shapes = {"gateWeight": (c, h), "gateBias": (h,), "valueWeight": (c, h), "valueBias": (h,),
              "outputWeight": (h, c), "outputBias": (c,)}
    ptrs = [None if weights.get(k) is None else _whole(k, weights[k], device, dtype, shapes[k]) for k in GATED_WEIGHTS]
    return c, h, shapes, _lib.GatedWeights(*ptrs)


def encode_gated_transition_tensors(device: Device, x, weights: dict, *, residual=None, activation: str = "silu",
                                    out=None, save: bool = False, stream: Optional[int] = None, workspace=None):
    """out = (act(x gateWeight + gateBias) * (x valueWeight + valueBias)) outputWeight + outputBias
    (+ residual): x, residual and out [rows, channels] (out may be the residual), gateWeight and
    valueWeight [channels, hidden], outputWeight [hidden, channels]; the biases may be absent.
    Returns out, or with save=True (out, saved) for encode_gated_transition_backward_tensors."""
    import torch
    dtype = x.dtype
    code, act = _dtype_code(dtype), _activation_code(activation)
    c, h, _, cw = _gated_weights(weights, device, dtype)
    x_stride = _rows("x", x, device, dtype, None, c)
    rows = x.shape[0]
    r_stride = c if residual is None else _rows("residual", residual, device, dtype, rows, c)
    new = []
    if out is None:
        out, out_stride = torch.empty((rows, c), dtype=dtype, device=x.device), c
        new.append(out)
    else:
        out_stride = _rows("out", out, device, dtype, rows, c)
    saved = None
    if save:
        saved = _saved(device, gated_transition_saved_bytes(rows, c, h, dtype))
        new.append(saved)
    ws = _workspace(workspace, lambda: gated_transition_workspace_bytes(rows, c, h, dtype), device)
    shape = _lib.TransitionShape(rows, c, h)
    opts = _lib.LayerOptions(act, 0, x_stride, r_stride, out_stride, x_stride)
    status = _lib.lib().af2_gated_transition(device.handle, ctypes.byref(shape), code, x.data_ptr(), ctypes.byref(cw),
                                             _ptr(residual), ctypes.byref(opts), out.data_ptr(),
                                             saved.data_ptr() if saved is not None and saved.numel() else None, ws,
                                             _stream_handle(device, stream))
    _lib.check(status, device.handle)
    _on_stream(new, device, stream)
    return (out, saved) if save else out


def encode_gated_transition_backward_tensors(device: Device, d_out, x, weights: dict, *, saved,
                                             activation: str = "silu", need=None, stream: Optional[int] = None,
                                             workspace=None) -> dict:
    """Gradients of encode_gated_transition_tensors for d_out [rows, channels]: "x" and every
    weight given, by its name, or those that `need` names.  The residual's gradient is d_out itself."""
    import torch
    dtype = x.dtype
    code, act = _dtype_code(dtype), _activation_code(activation)
    c, h, shapes, cw = _gated_weights(weights, device, dtype)
    x_stride = _rows("x", x, device, dtype, None, c)
    rows = x.shape[0]
    d_stride = _rows("d_out", d_out, device, dtype, rows, c)
    kept = _check_saved(saved, gated_transition_saved_bytes(rows, c, h, dtype), device)
    names = ["x"] + [k for k in GATED_WEIGHTS if weights.get(k) is not None]
    if need is not None:
        names = [k for k in names if k in need]
    grads = {k: torch.empty((rows, c) if k == "x" else shapes[k], dtype=dtype, device=x.device) for k in names}
    ws = _workspace(workspace, lambda: gated_transition_workspace_bytes(rows, c, h, dtype, True), device)
    shape = _lib.TransitionShape(rows, c, h)
    opts = _lib.LayerOptions(act, 0, x_stride, c, d_stride, c)
    cg = _lib.GatedGradients(_ptr(grads.get("x")), *(_ptr(grads.get(k)) for k in GATED_WEIGHTS))
    status = _lib.lib().af2_gated_transition_backward(device.handle, ctypes.byref(shape), code, d_out.data_ptr(),
                                                      x.data_ptr(), ctypes.byref(cw), kept, ctypes.byref(opts),
                                                      ctypes.byref(cg), ws, _stream_handle(device, stream))
    _lib.check(status, device.handle)
    _on_stream(grads.values(), device, stream)
    return grads
