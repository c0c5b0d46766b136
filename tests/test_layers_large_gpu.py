"""The layers where launches are long or change form: products whose last rows are cut in depth, tiles of
several lengths dealt out, rows that TMA cannot address beside kept slopes, bias sums over many rows, and
the row counts at which a forward pass changes kernels.  Tolerances as in test_layers_gpu.py.

relu has no slope at 0: where rounding in f32 can decide a pre-activation's sign (it is below 2^-22 of the
size of its terms, a few in ten million), 0 and 1 are both right, and what such an element enters (its row
of dx, its column of the gate's gradients) has no one reference value: these are left out there."""
import pytest
import torch

import af2cuda
import layer_reference as ref
from test_layers_gpu import BF16, DTYPES, F16, F32, close, dense_case, gated_case, run_dense, run_gated

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,channels,hidden,dtype,act", [
    (8192, 1024, 4096, BF16, "silu"),   # the gradients' tiles fill the SMs 4.3 times
    (8000, 1000, 3000, F16, "relu"),    # the same with ragged tiles
    (20000, 264, 1032, F32, "gelu"),
    (5000, 1025, 2049, BF16, "sigmoid"),  # nothing that TMA reads in place
])
def test_long_gated_training_steps(device, rows, channels, hidden, dtype, act):
    s = gated_case(rows, channels, hidden, dtype, seed=500)
    got, want = run_gated(device, s, act)
    if act == "relu":
        x, w = s["x"].double(), s["weights"]["gateWeight"].double()
        g, size = x @ w + s["weights"]["gateBias"].double(), x.abs() @ w.abs()
        unsure = g.abs() < 2.0**-22 * size
        rows_in, columns_in = ~unsure.any(1), ~unsure.any(0)
        assert rows_in.float().mean() > 0.9 and columns_in.float().mean() > 0.9
        for k, index in (("x", (rows_in,)), ("gateWeight", (slice(None), columns_in)), ("gateBias", (columns_in,))):
            got[k], want[k] = got[k][index], want[k][index]
    for k in got:
        close(k, got[k], want[k], dtype)


@pytest.mark.parametrize("rows,inner,columns,dtype,act", [
    (16384, 1024, 4096, BF16, "gelu"),  # tiles of 64 and of 256 steps
    (30000, 700, 1500, F16, "silu"),
    (16000, 1303, 346, F32, "relu"),
    (30000, 40, 64, BF16, "none"),      # bias sums of a tensor used as it is
])
def test_long_dense_training_steps(device, rows, inner, columns, dtype, act):
    got, want = run_dense(device, dense_case(rows, inner, columns, dtype, seed=600), act)
    for k in got:
        close(k, got[k], want[k], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("columns", [736, 737, 738, 740])
@pytest.mark.parametrize("act,residual", [("none", True), ("silu", True), ("silu", False)])
def test_rows_of_every_alignment(device, columns, act, residual, dtype):
    got, want = run_dense(device, dense_case(2999, 264, columns, dtype, seed=700), act, residual=residual)
    for k in got:
        close(k, got[k], want[k], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels,hidden", [(128, 512), (120, 333), (293, 893), (512, 2048)])
@pytest.mark.parametrize("rows", [4, 5, 20, 40, 64, 100, 256, 257])
def test_row_counts_between_kernels(device, rows, channels, hidden, dtype):
    s = gated_case(rows, channels, hidden, dtype, seed=800)
    want = ref.gated(s["x"], s["weights"], s["residual"], "silu")["y"]
    y = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], residual=s["residual"])
    close("y", y, want, dtype)
    # the caller's scratch has to do for whichever kernel runs
    size = af2cuda.gated_transition_workspace_bytes(rows, channels, hidden, dtype)
    scratch = torch.full((size + 4096,), 77, dtype=torch.uint8, device="cuda")
    y = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], residual=s["residual"],
                                                workspace=scratch[:size])
    close("y in the caller's scratch", y, want, dtype)
    assert bool((scratch[size:] == 77).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1023, 1024, 1025, 4097])
def test_bias_sums(device, rows, dtype):
    got, want = run_dense(device, dense_case(rows, 24, 72, dtype, seed=900), "none")
    close("bias", got["bias"], want["bias"], dtype)
    got, want = run_gated(device, gated_case(rows, 72, 40, dtype, seed=910), "relu")
    for k in ("gateBias", "valueBias", "outputBias"):
        close(k, got[k], want[k], dtype)


def test_same_bits_again(device):
    """Split sums, dealt tiles and bias sums join in a fixed order."""
    s = gated_case(8192, 512, 1032, BF16, seed=950)
    first, _ = run_gated(device, s, "silu")
    again, _ = run_gated(device, s, "silu")
    for k in first:
        assert torch.equal(first[k], again[k]), k
