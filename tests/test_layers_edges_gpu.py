"""The learned layers at their edges: the caller's scratch, streams and captures, values far from one.
Tolerances as in test_layers_gpu.py, but where a test states its own."""
import ctypes

import pytest
import torch

import af2cuda
from af2cuda import _lib
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


# ---- streams and captures ---------------------------------------------------------------------------


def test_captured_without_a_workspace(device):
    """What a graph holds stays its own: neither a larger call, which replaces the context's scratch, nor
    calls on another stream between the replays touch it."""
    s = gated_case(700, 130, 390, F32, seed=1100)
    want = ref.gated(s["x"], s["weights"], None, "gelu", s["d_out"])

    def step():
        y, saved = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], activation="gelu", save=True)
        grads = af2cuda.encode_gated_transition_backward_tensors(device, s["d_out"], s["x"], s["weights"], saved=saved,
                                                                 activation="gelu")
        norm = af2cuda.encode_gradient_norm_tensors(device, list(grads.values()))
        return {"y": y, **grads}, norm

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, norm = step()
    large = gated_case(9000, 264, 1032, F32, seed=1110)
    side = torch.cuda.Stream()
    for _ in range(4):
        for t in (*got.values(), norm):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            y = af2cuda.encode_gated_transition_tensors(device, large["x"], large["weights"])
        torch.cuda.synchronize()
        for k in got:
            close(k, got[k], want[k], F32)
        exact = sum(got[k].double().square().sum().item() for k in got if k != "y") ** 0.5
        assert abs(norm.item() - exact) <= 2.0**-23 * exact
    close("y", y, ref.gated(large["x"], large["weights"], None, "silu")["y"], F32)


def test_the_contexts_scratch_is_refused_in_a_capture(device):
    s = dense_case(700, 130, 390, F32, seed=1120)
    out = torch.empty_like(s["residual"])
    shape = _lib.LinearShape(700, 130, 390)

    def call(stream):
        return _lib.lib().af2_dense(device.handle, ctypes.byref(shape), _lib.AF2_F32, s["x"].data_ptr(),
                                    s["weight"].data_ptr(), None, None, None, out.data_ptr(), None, None, stream)

    assert call(1) == _lib.AF2_OK
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        status = call(torch.cuda.current_stream().cuda_stream)
        out.add_(1)
    assert status == _lib.AF2_ERR_UNSUPPORTED
    assert "workspace" in _lib.lib().af2_last_error(device.handle).decode()
    graph.replay()
    torch.cuda.synchronize()
    close("y", out, ref.dense(s["x"], s["weight"], None, None, "none")["y"] + 1, F32)


def test_a_named_streams_outputs_do_not_reuse_what_is_still_read(device):
    """Memory freed on torch's current stream, whose last reader there is still queued, is not what a call
    on another stream writes its outputs to."""
    s = dense_case(4096, 64, 1024, F32, seed=1130)
    want = ref.dense(s["x"], s["weight"], None, None, "none")["y"]
    side = torch.cuda.Stream()
    for stream in (side.cuda_stream, 0):
        kept = torch.zeros(4096, 1024, device="cuda")
        freed = torch.full((4096, 1024), 3.0, device="cuda")
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)
        kept.copy_(freed)
        del freed
        y = af2cuda.encode_dense_tensors(device, s["x"], s["weight"], stream=stream)
        torch.cuda.synchronize()
        assert bool((kept == 3.0).all()), stream
        close("y", y, want, F32)


def test_a_named_streams_outputs_live_until_the_current_stream_has_read_them(device):
    s = dense_case(4096, 64, 1024, F32, seed=1140)
    side, current = torch.cuda.Stream(), torch.cuda.current_stream()
    kept, other = torch.zeros(4096, 1024, device="cuda"), torch.full_like(s["weight"], 9.0)
    torch.cuda.synchronize()
    y = af2cuda.encode_dense_tensors(device, s["x"], s["weight"], stream=side.cuda_stream)
    want = ref.dense(s["x"], s["weight"], None, None, "none")["y"]
    current.wait_stream(side)
    torch.cuda._sleep(100_000_000)
    kept.copy_(y)
    del y
    for _ in range(3):
        af2cuda.encode_dense_tensors(device, s["x"], other, stream=side.cuda_stream)
    torch.cuda.synchronize()
    close("y", kept, want, F32)


def test_streams_that_come_and_go_share_the_scratch_safely(device):
    """Each call on a new stream, destroyed with the work pending: handles come back, streams do not."""
    runtime = ctypes.CDLL("libcudart.so.12")  # the one that torch has loaded
    runtime.cudaStreamDestroy.argtypes = [ctypes.c_size_t]
    cases = [gated_case(700, 130, 260, F32, seed=1150 + i) for i in range(2)]
    want = [ref.gated(s["x"], s["weights"], None, "silu")["y"] for s in cases]
    outs = [torch.empty_like(cases[0]["x"]) for _ in range(16)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        stream = ctypes.c_size_t()
        assert runtime.cudaStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
        s = cases[i % 2]
        shape = _lib.TransitionShape(700, 130, 260)
        w = _lib.GatedWeights(*[s["weights"][k].data_ptr() for k in ("gateWeight", "gateBias", "valueWeight", "valueBias",
                                                                     "outputWeight", "outputBias")])
        o = _lib.LayerOptions(3, 0, 130, 130, 130, 130)
        _lib.check(_lib.lib().af2_gated_transition(device.handle, ctypes.byref(shape), _lib.AF2_F32, s["x"].data_ptr(),
                                                   ctypes.byref(w), None, ctypes.byref(o), out.data_ptr(), None, None,
                                                   stream.value), device.handle)
        assert runtime.cudaStreamDestroy(stream.value) == 0
    torch.cuda.synchronize()
    for i, y in enumerate(outs):
        close("y", y, want[i % 2], F32)


# ---- values far from one ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["relu", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("rows", [3, 40, 600])
def test_gates_shut_by_the_lowest_value(device, rows, act, dtype):
    """A bias of the type's lowest value shuts some hidden channels: their activation is 0, and what
    stands beside them is as it would be alone."""
    lowest = torch.finfo(dtype).min
    for channels in (64, 200):
        s = gated_case(rows, channels, 264, dtype, seed=1200)
        s["weights"]["gateBias"][::3] = lowest
        w = s["weights"]
        want = ref.gated(s["x"], w, None, act, s["d_out"])
        y = af2cuda.encode_gated_transition_tensors(device, s["x"], w, activation=act)
        close("y alone", y, want["y"], dtype)
        y, saved = af2cuda.encode_gated_transition_tensors(device, s["x"], w, activation=act, save=True)
        grads = af2cuda.encode_gated_transition_backward_tensors(device, s["d_out"], s["x"], w, saved=saved, activation=act)
        for k, v in {"y": y, **grads}.items():
            close(k, v, want[k], dtype)
            if k in ("gateBias", "valueBias", "gateWeight", "valueWeight"):
                assert not v[..., ::3].any(), k
    d = dense_case(rows, 96, 136, dtype, seed=1210)
    d["bias"][::3] = lowest
    want = ref.dense(d["x"], d["weight"], d["bias"], None, act, d["d_out"])
    y = af2cuda.encode_dense_tensors(device, d["x"], d["weight"], bias=d["bias"], activation=act)
    close("y alone", y, want["y"], dtype)
    y, saved = af2cuda.encode_dense_tensors(device, d["x"], d["weight"], bias=d["bias"], activation=act, save=True)
    grads = af2cuda.encode_dense_backward_tensors(device, d["d_out"], d["x"], d["weight"], saved=saved, bias=True, activation=act)
    for k, v in {"y": y, **grads}.items():
        close(k, v, want[k], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
def test_infinite_and_nan_pre_activations(device, act, dtype):
    """Through biases: each column is what the formula makes of it, the columns beside it what they were."""
    for rows in (4, 500):
        d = dense_case(rows, 64, 80, dtype, seed=1220)
        clean = af2cuda.encode_dense_tensors(device, d["x"], d["weight"], bias=d["bias"], activation=act)
        for value in (float("inf"), float("-inf"), float("nan")):
            bias = d["bias"].clone()
            bias[[0, 17, 33]] = value
            limit = ref.act(act, torch.tensor(value, dtype=torch.float64)).item()
            for save in (False, True):
                y = af2cuda.encode_dense_tensors(device, d["x"], d["weight"], bias=bias, activation=act, save=save)
                y = y[0] if save else y
                other = [c for c in range(80) if c not in (0, 17, 33)]
                close("the others", y[:, other], clean[:, other].double(), dtype)
                got = y[:, [0, 17, 33]]
                assert bool(torch.isnan(got).all() if limit != limit else (got == limit).all()), (value, save)


def bare_gate(rows, width, dtype, low, high):
    """A gated transition whose hidden activations are act(x), one by one: the gate and output weights are
    identities, the value is 1, and x goes from low to high."""
    x = torch.linspace(low, high, rows * width, device="cuda").to(dtype).view(rows, width)
    one = torch.eye(width, device="cuda").to(dtype)
    return x, {"gateWeight": one, "valueWeight": torch.zeros_like(one), "valueBias": torch.ones_like(one[0]),
               "outputWeight": one}


def exact_act(kind, z):
    """ref.act in f64 with its last places on the negative side: Phi(z) from erfc, since 1 + erf cancels."""
    return z * torch.erfc(-z * 0.5**0.5) / 2 if kind == "gelu" else ref.act(kind, z)


def elements_close(name, got, want, relative, dtype):
    """Within `relative` of each element, and half of f16's smallest step."""
    err = (got.double() - want).abs() - (2.0**-25 if dtype == F16 else 0.0)
    worst = (err / want.abs().clamp(min=1e-300)).max().item()
    assert worst <= relative, f"{name}: an element is off by {worst:.3e} of its size"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act,low", [("sigmoid", -30.0), ("silu", -30.0), ("gelu", -10.0)])
@pytest.mark.parametrize("rows,width", [(4, 64), (700, 64), (5000, 128), (700, 200)])
def test_activations_element_by_element(device, rows, width, act, low, dtype):
    """No positive gate hides the error of a negative one.  Each element is rounded once (the output's
    product copies it), and the activations of 16-bit tensors are within 2^-16."""
    x, w = bare_gate(rows, width, dtype, low, 12.0)
    want = exact_act(act, x.double())
    alone = af2cuda.encode_gated_transition_tensors(device, x, w, activation=act)
    elements_close("y alone", alone, want, ref.ROUNDOFF[dtype] + 2.0**-16, dtype)
    kept, _ = af2cuda.encode_gated_transition_tensors(device, x, w, activation=act, save=True)
    elements_close("y", kept, want, ref.ROUNDOFF[dtype] + 2.0**-16, dtype)
    d = af2cuda.encode_dense_tensors(device, x, w["gateWeight"], activation=act)
    elements_close("dense", d, want, ref.ROUNDOFF[dtype] + 2.0**-16, dtype)


def exact_slope(kind, z):
    """The slope, and the size of the terms that it is a sum of."""
    s = torch.sigmoid(z)
    if kind == "sigmoid":
        return s * torch.sigmoid(-z), s
    if kind == "silu":
        return s + z * s * torch.sigmoid(-z), s + z.abs() * s * torch.sigmoid(-z)
    phi, pdf = torch.erfc(-z * 0.5**0.5) / 2, torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    return phi + z * pdf, phi + z.abs() * pdf


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act,low,high", [("sigmoid", -24.0, 4.0), ("silu", -24.0, 8.0), ("gelu", -6.0, 6.0)])
@pytest.mark.parametrize("rows,width,scale", [(700, 64, 1.0), (700, 64, 2.0**14), (4, 128, 2.0**14), (3000, 77, 2.0**14)])
def test_slopes_element_by_element(device, rows, width, scale, act, low, high, dtype):
    """The gradient at each pre-activation of a dense layer, saturated ones too: through an identity weight
    it is dx itself.  Its product with the slope is rounded once, the activations' arithmetic is within 2^-16
    of the slope's terms, and bf16 keeps a slope to 2^-11 (to 2^-39 where it is below 2^-28)."""
    x, w = bare_gate(rows, width, dtype, low, high)
    d_out = torch.full_like(x, scale)
    _, saved = af2cuda.encode_dense_tensors(device, x, w["gateWeight"], activation=act, save=True)
    got = af2cuda.encode_dense_backward_tensors(device, d_out, x, w["gateWeight"], saved=saved, activation=act)
    slope, terms = exact_slope(act, x.double())
    err = (got["x"].double() - scale * slope).abs()
    kept, least = (2.0**-11, 2.0**-39) if dtype == BF16 else (0.0, 0.0)
    allowed = (ref.ROUNDOFF[dtype] + kept + 2.0**-18) * slope.abs() + 2.0**-16 * terms
    allowed = scale * (allowed + least) + (2.0**-25 if dtype == F16 else 0.0)
    assert bool((err <= allowed).all()), (err / allowed).max().item()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,width", [(4, 64), (700, 64), (3000, 77), (1000, 264)])
@pytest.mark.parametrize("outlier", [1.0, 300.0, 4096.0])
def test_factors_beside_outliers_element_by_element(device, rows, width, outlier, dtype):
    """The gated transition's two factors in every column, one of which in eight is `outlier` times the
    others: through identity weights dx is dg, or dv.  Their products are rounded once, the activations'
    arithmetic is within 2^-16 of the terms, and bf16 keeps a factor to 2^-11."""
    rounded = ref.ROUNDOFF[dtype] + 2.0**-18 + (2.0**-11 if dtype == BF16 else 0.0)
    tiny = 2.0**-25 if dtype == F16 else 0.0
    x, w = bare_gate(rows, width, dtype, -8.0, 5.0)
    d_out = torch.full_like(x, 0.75)
    size = torch.ones(width, device="cuda").to(dtype)
    size[::8] = outlier
    w["valueBias"] = size  # v
    _, saved = af2cuda.encode_gated_transition_tensors(device, x, w, save=True)
    got = af2cuda.encode_gated_transition_backward_tensors(device, d_out, x, w, saved=saved)["x"]
    slope, terms = exact_slope("silu", x.double())
    want = 0.75 * size.double() * slope
    allowed = rounded * want.abs() + 2.0**-16 * 0.75 * size.double() * terms + tiny
    assert bool(((got.double() - want).abs() <= allowed).all()), "dg"
    # a = the gate's bias, v = x
    w = {"gateWeight": torch.zeros_like(w["gateWeight"]), "gateBias": size / 3, "valueWeight": w["gateWeight"],
         "outputWeight": w["outputWeight"]}
    _, saved = af2cuda.encode_gated_transition_tensors(device, x, w, activation="none", save=True)
    got = af2cuda.encode_gated_transition_backward_tensors(device, d_out, x, w, saved=saved, activation="none")["x"]
    want = 0.75 * (size / 3).double().expand_as(got)
    assert bool(((got.double() - want).abs() <= rounded * want.abs() + tiny).all()), "dv"


@pytest.mark.parametrize("act,low,units", [("sigmoid", -60.0, 12), ("silu", -60.0, 13), ("gelu", -12.0, 22)])
@pytest.mark.parametrize("rows,width", [(4, 64), (700, 64), (3000, 77), (700, 200)])
def test_f32_activations_element_by_element(device, rows, width, act, low, units):
    """In units of 2^-24 of the element: the hardware's exponential 4 and reciprocal 2, one for each
    operation beside them (gelu's polynomial has nine), two for the copies through identity weights."""
    x, w = bare_gate(rows, width, F32, low, 12.0)
    want = exact_act(act, x.double())
    alone = af2cuda.encode_gated_transition_tensors(device, x, w, activation=act)
    elements_close("y alone", alone, want, units * 2.0**-24, F32)
    kept, _ = af2cuda.encode_gated_transition_tensors(device, x, w, activation=act, save=True)
    elements_close("y", kept, want, units * 2.0**-24, F32)
    d = af2cuda.encode_dense_tensors(device, x, w["gateWeight"], activation=act)
    elements_close("dense", d, want, units * 2.0**-24, F32)


# ---- sets of tensors ---------------------------------------------------------------------------------


def test_overlapping_tensors_are_refused_where_they_are_written(device):
    """Blocks scale their parts of a set in no order: what two of them would write is refused."""
    flat = torch.randn(4000, device="cuda")
    a, b, c = flat[:1000], flat[1000:2500], flat[2500:]
    clip = af2cuda.encode_clip_gradients_tensors
    before = flat.clone()
    for bad in ([a, a], [a, b, a], [flat, c], [c, flat], [a, flat[999:1001]], [b, a, flat[2400:2600]]):
        with pytest.raises(af2cuda.RangeError, match="overlap"):
            clip(device, bad, 1.0)
    with pytest.raises(af2cuda.RangeError, match="overlap"):
        clip(device, [a, torch.randn(1000, device="cuda")], 1.0, out=[flat[:1000], flat[500:1500]])
    with pytest.raises(af2cuda.RangeError, match="output 1 overlaps tensor 0"):
        clip(device, [a, torch.randn(1000, device="cuda")], 1.0, out=[torch.empty(1000, device="cuda"), a])
    with pytest.raises(af2cuda.RangeError, match="output 0 overlaps tensor 0"):
        clip(device, [a], 1.0, out=[flat[1:1001]])
    assert torch.equal(flat, before)
    # read twice and written apart; in any order; in place by name; nothing at all
    outs = [torch.empty(1000, device="cuda") for _ in range(2)]
    norm = clip(device, [a, a], 1.0, out=outs)
    assert abs(norm.item() - 2**0.5 * before[:1000].double().norm().item()) <= 1e-5 * norm.item()
    assert torch.equal(outs[0], outs[1])
    empty = flat[:0]
    norm = clip(device, [c, empty, a, b, empty], 1.0, out=[c, empty, a, b, empty])
    assert abs(norm.item() - before.double().norm().item()) <= 1e-5 * norm.item()
    assert torch.allclose(flat, before / norm, rtol=1e-5)
    assert abs(af2cuda.encode_gradient_norm_tensors(device, [a, a]).item() - 2**0.5 * a.norm().item()) <= 1e-5


# ---- arguments -----------------------------------------------------------------------------------------


def test_options_without_a_truth_value_are_errors(device):
    """The bias itself where the backward pass asks whether there is one."""
    d = dense_case(20, 16, 24, BF16, seed=1300)
    with pytest.raises(RuntimeError, match="[Aa]mbiguous"):
        af2cuda.encode_dense_backward_tensors(device, d["d_out"], d["x"], d["weight"], bias=d["bias"])
    with pytest.raises(RuntimeError, match="[Aa]mbiguous"):
        af2cuda.encode_dense_tensors(device, d["x"], d["weight"], save=d["bias"])
    got = af2cuda.encode_dense_backward_tensors(device, d["d_out"], d["x"], d["weight"], bias=True)
    close("bias", got["bias"], d["d_out"].double().sum(0), BF16)


def test_one_need_by_its_name(device):
    d = dense_case(20, 16, 24, BF16, seed=1310)
    assert list(af2cuda.encode_dense_backward_tensors(device, d["d_out"], d["x"], d["weight"], need="weight")) == ["weight"]
    got = af2cuda.encode_dense_backward_tensors(device, d["d_out"], d["x"], d["weight"], bias=True, need=["bias", "x"])
    assert sorted(got) == ["bias", "x"]
    s = gated_case(20, 16, 24, BF16, seed=1320)
    _, saved = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], save=True)
    for need in ("x", "gateBias", ["valueWeight", "outputBias"], iter(["x", "outputWeight"])):
        names = [need] if isinstance(need, str) else need if isinstance(need, list) else ["x", "outputWeight"]
        got = af2cuda.encode_gated_transition_backward_tensors(device, s["d_out"], s["x"], s["weights"], saved=saved, need=need)
        assert sorted(got) == sorted(names)


def test_written_tensors_show_it_to_autograd(device):
    """What a call writes counts as written in place: a backward pass of torch's that saved it refuses."""
    d = dense_case(20, 16, 24, F32, seed=1330)
    out = torch.ones(20, 24, device="cuda")
    factor = torch.ones(20, 24, device="cuda", requires_grad=True)
    product = (out * factor).sum()
    af2cuda.encode_dense_tensors(device, d["x"], d["weight"], out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    s = gated_case(20, 16, 24, F32, seed=1340)
    residual = s["residual"].clone()
    version = residual._version
    af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], residual=residual, out=residual)
    assert residual._version > version
    a, b, c = (torch.ones(50, device="cuda") for _ in range(3))
    versions = [t._version for t in (a, b, c)]
    af2cuda.encode_clip_gradients_tensors(device, [a], 1.0, out=[b])
    af2cuda.encode_clip_gradients_tensors(device, [c], 1.0)
    assert [t._version for t in (a, b, c)] == [versions[0], versions[1] + 1, versions[2] + 1]
    with torch.inference_mode():
        t = torch.ones(20, 24, device="cuda")
        af2cuda.encode_dense_tensors(device, d["x"], d["weight"], out=t)
    af2cuda.encode_dense_tensors(device, d["x"], d["weight"], out=t)
    close("y", t, ref.dense(d["x"], d["weight"], None, None, "none")["y"], F32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,inner,columns", [(2, 8192, 512), (16, 4096, 1024), (16, 1024, 1024), (40, 20001, 33),
                                                (200, 16384, 32), (256, 256, 32), (5, 40, 5000)])
def test_dense_layers_deep_and_wide_for_few_rows(device, rows, inner, columns, dtype):
    """On both sides of the choice between the kernels."""
    d = dense_case(rows, inner, columns, dtype, seed=1350)
    y = af2cuda.encode_dense_tensors(device, d["x"], d["weight"], bias=d["bias"], residual=d["residual"], activation="silu")
    close("y", y, ref.dense(d["x"], d["weight"], d["bias"], d["residual"], "silu")["y"], dtype)
    size = af2cuda.dense_workspace_bytes(rows, inner, columns, dtype, "silu")
    scratch, intact = guarded(size)
    y = af2cuda.encode_dense_tensors(device, d["x"], d["weight"], activation="silu", workspace=scratch)
    close("y", y, ref.dense(d["x"], d["weight"], None, None, "silu")["y"], dtype)
    assert intact()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,low,high", [("sigmoid", 0.0, 24.0), ("sigmoid", -24.0, 0.0), ("silu", -24.0, 24.0),
                                          ("gelu", -6.0, 6.0)])
@pytest.mark.parametrize("rows,width", [(700, 64), (3000, 77)])
def test_slopes_at_both_ends(device, rows, width, act, low, high, dtype):
    """As test_slopes_element_by_element, for sigmoid's positive side and for f32 too: there the slope's
    terms are within 24 units of 2^-24."""
    x, w = bare_gate(rows, width, dtype, low, high)
    scale = 2.0**14
    _, saved = af2cuda.encode_dense_tensors(device, x, w["gateWeight"], activation=act, save=True)
    got = af2cuda.encode_dense_backward_tensors(device, torch.full_like(x, scale), x, w["gateWeight"], saved=saved,
                                                activation=act)["x"]
    slope, terms = exact_slope(act, x.double())
    if act == "sigmoid":
        terms = slope
    kept, least = (2.0**-11, 2.0**-39) if dtype == BF16 else (0.0, 0.0)
    rounded = ref.ROUNDOFF[dtype] + kept + 2.0**-18 if dtype != F32 else 0.0
    allowed = rounded * slope.abs() + (24 * 2.0**-24 if dtype == F32 else 2.0**-16) * terms + least
    allowed = scale * allowed + (2.0**-25 if dtype == F16 else 0.0)
    err = (got.double() - scale * slope).abs()
    assert bool((err <= allowed).all()), (err / allowed).max().item()


def test_outputs_that_overlap_inputs_are_refused(device):
    """Blocks write an output while others read: in place works where each row is read before it is written."""
    dense, gated = af2cuda.encode_dense_tensors, af2cuda.encode_gated_transition_tensors
    flat = torch.randn(4000, device="cuda").to(BF16)
    x, w = flat[:1600].view(100, 16), torch.randn(16, 16, device="cuda").to(BF16)
    for bad in (x, flat[1500:3100].view(100, 16), flat[1:1601].view(100, 16)):
        with pytest.raises(af2cuda.RangeError, match="out overlaps"):
            dense(device, x, w, out=bad)
    with pytest.raises(af2cuda.RangeError, match="out overlaps"):
        dense(device, flat[2000:3600].view(100, 16), x[:16], out=x)
    with pytest.raises(af2cuda.RangeError, match="out overlaps"):
        dense(device, flat[2000:3600].view(100, 16), w, bias=x[99], out=x)
    with pytest.raises(af2cuda.RangeError, match="without being it"):
        dense(device, flat[2000:3600].view(100, 16), w, residual=flat[16:1616].view(100, 16), out=x)
    # the halves of one buffer's rows, rows between rows, and what only touches
    both = torch.randn(100, 32, device="cuda").to(BF16)
    want = ref.dense(both[:, :16], w, None, None, "none")["y"]
    close("halves", dense(device, both[:, :16], w, out=both[:, 16:]), want, BF16)
    with pytest.raises(af2cuda.RangeError, match="out overlaps"):
        dense(device, both[:, :16], w, out=both[:, 15:31])
    with pytest.raises(af2cuda.RangeError, match="out overlaps"):
        dense(device, both[:99, 16:], w, out=both[1:, 10:26])
    close("rows", dense(device, both[::2, :16], w, out=both[1::2, :16]),
          ref.dense(both[::2, :16], w, None, None, "none")["y"], BF16)
    close("next to it", dense(device, x, w, out=flat[1600:3200].view(100, 16)),
          ref.dense(x, w, None, None, "none")["y"], BF16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,channels,hidden", [(3, 64, 128), (700, 64, 128), (20000, 128, 512), (700, 200, 264),
                                                  (700, 77, 130)])
def test_gated_transition_in_place(device, rows, channels, hidden, dtype):
    s = gated_case(rows, channels, hidden, dtype, seed=1360)
    want = ref.gated(s["x"], s["weights"], s["x"], "silu")["y"]
    alone = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], residual=s["x"])
    x = s["x"].clone()
    af2cuda.encode_gated_transition_tensors(device, x, s["weights"], residual=x, out=x)
    close("y", x, want, dtype)
    assert torch.equal(x, alone)
