"""CPU tests of the learned layers' C entry points: sizes and the checks that need no device."""
import ctypes

import pytest

import af2cuda
from af2cuda import _lib


def _bytes(fn, *args):
    out = ctypes.c_uint64()
    return fn(*args, ctypes.byref(out)), int(out.value)


@pytest.mark.parametrize("dtype", [_lib.AF2_F32, _lib.AF2_F16, _lib.AF2_BF16])
def test_sizes_of_saved_and_scratch(dtype):
    lib = _lib.lib()
    shape = _lib.LinearShape(1000, 256, 1024)
    assert _bytes(lib.af2_dense_saved_bytes, ctypes.byref(shape), dtype, 0) == (0, 0)
    st, saved = _bytes(lib.af2_dense_saved_bytes, ctypes.byref(shape), dtype, 3)
    assert st == 0 and 2 * 1000 * 1024 <= saved <= 5 * 1000 * 1024
    for backward in (0, 1):
        assert _bytes(lib.af2_dense_workspace_bytes, ctypes.byref(shape), dtype, 3, backward)[0] == 0
    gated = _lib.TransitionShape(1000, 256, 1024)
    st, saved = _bytes(lib.af2_gated_transition_saved_bytes, ctypes.byref(gated), dtype)
    assert st == 0 and saved >= 4 * 1000 * 1024
    for backward in (0, 1):
        assert _bytes(lib.af2_gated_transition_workspace_bytes, ctypes.byref(gated), dtype, backward)[0] == 0
    assert _bytes(lib.af2_gated_transition_saved_bytes, ctypes.byref(_lib.TransitionShape(0, 8, 8)), dtype) == (0, 0)


def test_sizes_past_32_bits():
    shape = _lib.TransitionShape(2**31 - 2048, 256, 1024)
    st, saved = _bytes(_lib.lib().af2_gated_transition_saved_bytes, ctypes.byref(shape), _lib.AF2_BF16)
    assert st == 0 and saved >= 4 * (2**31 - 2048) * 1024


@pytest.mark.parametrize("rows,inner,columns,dtype,act,status", [
    (-1, 8, 8, 0, 0, _lib.AF2_ERR_INVALID_ARGUMENT), (1, 0, 8, 0, 0, _lib.AF2_ERR_INVALID_ARGUMENT),
    (1, 8, -8, 0, 0, _lib.AF2_ERR_INVALID_ARGUMENT), (1, 8, 8, 3, 0, _lib.AF2_ERR_INVALID_ARGUMENT),
    (1, 8, 8, 0, 5, _lib.AF2_ERR_INVALID_ARGUMENT), (1, 8, 8, 0, -1, _lib.AF2_ERR_INVALID_ARGUMENT),
    (1, 65537, 8, 0, 0, _lib.AF2_ERR_UNSUPPORTED), (2**31, 8, 8, 0, 0, _lib.AF2_ERR_UNSUPPORTED)])
def test_sizes_that_are_refused(rows, inner, columns, dtype, act, status):
    lib, shape = _lib.lib(), _lib.LinearShape(rows, inner, columns)
    assert _bytes(lib.af2_dense_saved_bytes, ctypes.byref(shape), dtype, act)[0] == status
    assert _bytes(lib.af2_dense_workspace_bytes, ctypes.byref(shape), dtype, act, 0)[0] == status


def test_calls_without_a_context_or_sizes():
    lib = _lib.lib()
    null = None
    assert lib.af2_dense(null, null, 0, null, null, null, null, null, null, null, null, null) != 0
    assert lib.af2_gated_transition_backward(null, null, 0, null, null, null, null, null, null, null, null) != 0
    assert lib.af2_gradient_norm(null, null, 0, null, null, null) != 0
    assert lib.af2_clip_gradients(null, null, null, 0, 1.0, null, null, null) != 0
    assert lib.af2_dense_saved_bytes(null, 0, 0, null) == _lib.AF2_ERR_INVALID_ARGUMENT
    assert lib.af2_gradient_norm_workspace_bytes(-1, ctypes.byref(ctypes.c_uint64())) == _lib.AF2_ERR_INVALID_ARGUMENT


def test_python_sizes():
    torch = pytest.importorskip("torch")
    assert af2cuda.dense_saved_bytes(10, 8, 8, torch.bfloat16) == 0
    assert af2cuda.gated_transition_saved_bytes(10, 8, 16, torch.float32) >= 2 * 4 * 10 * 16
    with pytest.raises(af2cuda.RangeError, match="activation"):
        af2cuda.dense_saved_bytes(10, 8, 8, torch.bfloat16, "tanh")
    with pytest.raises(af2cuda.RangeError, match="float32, float16 or bfloat16"):
        af2cuda.dense_saved_bytes(10, 8, 8, torch.float64)
    assert af2cuda.gradient_norm_workspace_bytes(1000) > 1000
