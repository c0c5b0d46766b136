"""The learned layers at their edges: the caller's scratch, streams and captures, values far from one.
Tolerances as in test_layers_gpu.py, but where a test states its own."""
import pytest
import torch

import af2cuda
import layer_reference as ref
from test_layers_gpu import BF16, DTYPES, F16, F32, close, dense_case, gated_case

pytestmark = pytest.mark.gpu


# ---- the caller's scratch -------------------------------------------------------------------------


def guarded(size):
    """`size` bytes of scratch with a pattern behind them: (scratch, whether the pattern is as it was)."""
    whole = torch.full((size + (32 << 20),), 77, dtype=torch.uint8, device="cuda")
    return whole[:size], lambda: bool((whole[size:] == 77).all())


@pytest.mark.parametrize("rows,inner,columns,dtype,act", [
    (2048, 768, 3000, F32, "silu"), (2048, 512, 512, BF16, "none"), (6000, 293, 1909, F32, "gelu"),
    (3001, 259, 387, F16, "silu")])
def test_dense_backward_in_the_callers_scratch(device, rows, inner, columns, dtype, act):
    """One gradient alone is cut deeper than both together: the query has to cover it."""
    s = dense_case(rows, inner, columns, dtype, seed=1000)
    _, saved = af2cuda.encode_dense_tensors(device, s["x"], s["weight"], bias=s["bias"], activation=act, save=True)
    want = ref.dense(s["x"], s["weight"], s["bias"], None, act, s["d_out"])
    size = af2cuda.dense_workspace_bytes(rows, inner, columns, dtype, act, backward=True)
    for need in (("x",), ("weight",), ("x", "weight"), ()):
        for bias in (True, False):
            scratch, intact = guarded(size)
            got = af2cuda.encode_dense_backward_tensors(device, s["d_out"], s["x"], s["weight"], saved=saved, bias=bias,
                                                        activation=act, need=need, workspace=scratch)
            assert sorted(got) == sorted(need + (("bias",) if bias else ()))
            for k in got:
                close(k, got[k], want[k], dtype)
            assert intact(), (need, bias)


@pytest.mark.parametrize("rows,channels,hidden,dtype", [(2048, 1024, 4096, BF16), (700, 130, 390, F32), (1500, 264, 1032, F16)])
def test_gated_backward_in_the_callers_scratch(device, rows, channels, hidden, dtype):
    s = gated_case(rows, channels, hidden, dtype, seed=1010)
    _, saved = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], save=True)
    want = ref.gated(s["x"], s["weights"], None, "silu", s["d_out"])
    size = af2cuda.gated_transition_workspace_bytes(rows, channels, hidden, dtype, backward=True)
    for need in (["x"], ["gateWeight"], ["gateWeight", "valueWeight"], ["outputWeight"], ["x", "outputWeight"],
                 ["x", "valueWeight", "valueBias"], ["gateBias", "outputBias"], None):
        scratch, intact = guarded(size)
        got = af2cuda.encode_gated_transition_backward_tensors(device, s["d_out"], s["x"], s["weights"], saved=saved,
                                                               need=need, workspace=scratch)
        assert need is None or sorted(got) == sorted(need)
        for k in got:
            close(k, got[k], want[k], dtype)
        assert intact(), need


# ---- blocks that add up through one another's shared memory ------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inner,columns", [(256, 32), (512, 64), (1024, 200), (4096, 96), (4096, 1000)])
def test_few_rows_whose_depth_is_shared(device, inner, columns, dtype):
    """Clusters of two to eight blocks, launch upon launch: the same bits each time."""
    s = dense_case(3, inner, columns, dtype, seed=1020)
    want = ref.dense(s["x"], s["weight"], s["bias"], s["residual"], "silu")["y"]
    outs = [af2cuda.encode_dense_tensors(device, s["x"], s["weight"], bias=s["bias"], residual=s["residual"],
                                         activation="silu") for _ in range(100)]
    close("y", outs[0], want, dtype)
    assert all(torch.equal(y, outs[0]) for y in outs)
