"""The dense layer and the gated transition against the formulas in 64 bits,
against differences, and at the sizes and strides where tiles end.

Tolerances.  One rounding to a type changes a tensor by at most u of its
2-norm, u being half the type's unit roundoff (layer_reference.UNIT).  An output has at most three on its way: the saved
pre-activation's (where the type has one), the operand's (the hidden
activation, or the gradient at a pre-activation) and its own.  For random
operands they add as squares, so 3 u bounds all of them with room; f32
products carry a relative error that grows with the depth, below 2^-24 times
the square root of the terms each, and 1e-5 bounds two of them in a row for
every depth here."""
import pytest
import torch

import af2cuda
import layer_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = [BF16, F16, F32]
ACTS = ["none", "relu", "sigmoid", "silu", "gelu"]
# (rows, inner, columns): below, at and past tiles; odd widths; one of each; deep and wide
SHAPES = [(1, 1, 1), (1, 1024, 512), (2, 3, 5), (5, 8, 8), (7, 64, 72), (16, 256, 264), (33, 130, 390), (128, 128, 512),
          (129, 257, 129), (255, 72, 320), (256, 512, 256), (300, 1000, 1032), (1000, 136, 24), (2500, 264, 136)]


def tolerance(dtype) -> float:
    return 1e-5 if dtype == F32 else 3 * ref.UNIT[dtype]


def normal(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def close(name, got, want, dtype):
    assert got.dtype == dtype and tuple(got.shape) == tuple(want.shape), name
    tol = tolerance(dtype)
    err = ref.relative(got, want)
    assert err <= tol, f"{name}: relative error {err:.3e} > {tol:.3e}"
    if want.numel():
        rms = want.square().mean().sqrt().clamp(min=1e-30)
        worst = ((got.double() - want).abs() / torch.maximum(want.abs(), rms)).max().item()
        assert worst <= 16 * tol, f"{name}: an element is off by {worst:.3e} of its size"


def dense_case(rows, inner, columns, dtype, seed=0):
    return {"x": normal(seed, rows, inner, dtype=dtype), "weight": normal(seed + 1, inner, columns, dtype=dtype,
                                                                          scale=inner**-0.5),
            "bias": normal(seed + 2, columns, dtype=dtype, scale=0.3),
            "residual": normal(seed + 3, rows, columns, dtype=dtype),
            "d_out": normal(seed + 4, rows, columns, dtype=dtype, scale=1 / 16)}


def gated_case(rows, c, h, dtype, seed=0):
    w = {"gateWeight": normal(seed + 1, c, h, dtype=dtype, scale=c**-0.5),
         "gateBias": normal(seed + 2, h, dtype=dtype, scale=0.3),
         "valueWeight": normal(seed + 3, c, h, dtype=dtype, scale=c**-0.5),
         "valueBias": normal(seed + 4, h, dtype=dtype, scale=0.3),
         "outputWeight": normal(seed + 5, h, c, dtype=dtype, scale=h**-0.5),
         "outputBias": normal(seed + 6, c, dtype=dtype, scale=0.3)}
    return {"x": normal(seed, rows, c, dtype=dtype), "weights": w, "residual": normal(seed + 7, rows, c, dtype=dtype),
            "d_out": normal(seed + 8, rows, c, dtype=dtype, scale=1 / 16)}


def run_dense(device, s, act, bias=True, residual=True):
    b, r = (s["bias"] if bias else None), (s["residual"] if residual else None)
    y, saved = af2cuda.encode_dense_tensors(device, s["x"], s["weight"], bias=b, residual=r, activation=act, save=True)
    grads = af2cuda.encode_dense_backward_tensors(device, s["d_out"], s["x"], s["weight"], saved=saved, bias=bias,
                                                  activation=act)
    want = ref.dense(s["x"], s["weight"], b, r, act, s["d_out"])
    device.sync(1)
    return {"y": y, **grads}, want


def run_gated(device, s, act, residual=True, weights=None):
    w, r = weights or s["weights"], (s["residual"] if residual else None)
    y, saved = af2cuda.encode_gated_transition_tensors(device, s["x"], w, residual=r, activation=act, save=True)
    grads = af2cuda.encode_gated_transition_backward_tensors(device, s["d_out"], s["x"], w, saved=saved,
                                                             activation=act)
    want = ref.gated(s["x"], w, r, act, s["d_out"])
    device.sync(1)
    return {"y": y, **grads}, want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_dense_forward_and_backward(device, shape, dtype):
    act = ACTS[(shape[0] + shape[1]) % 5]
    got, want = run_dense(device, dense_case(*shape, dtype), act)
    for k in got:
        close(k, got[k], want[k], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(True, True), (True, False), (False, True), (False, False)])
def test_dense_options(device, act, bias, residual, dtype):
    got, want = run_dense(device, dense_case(150, 96, 200, dtype, seed=20), act, bias, residual)
    for k in got:
        close(k, got[k], want[k], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gated_forward_and_backward(device, shape, dtype):
    act = ACTS[(shape[0] + 2 * shape[1]) % 5]
    got, want = run_gated(device, gated_case(*shape, dtype), act)
    assert set(got) == set(want)
    for k in got:
        close(k, got[k], want[k], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_gated_options(device, act, dtype):
    s = gated_case(140, 96, 200, dtype, seed=40)
    bare = {k: v for k, v in s["weights"].items() if k.endswith("Weight")}
    got, want = run_gated(device, s, act, residual=False, weights=bare)
    assert set(got) == {"y", "x", *bare}
    for k in got:
        close(k, got[k], want[k], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 8, 9, 17, 31, 64, 65, 127])
def test_few_rows(device, rows, dtype):
    """The serving sizes: one token to a small batch, forward only."""
    s = gated_case(rows, 512, 1024, dtype, seed=60)
    y = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], residual=s["residual"])
    close("gated", y, ref.gated(s["x"], s["weights"], s["residual"], "silu")["y"], dtype)
    d = dense_case(rows, 1024, 520, dtype, seed=70)
    y = af2cuda.encode_dense_tensors(device, d["x"], d["weight"], bias=d["bias"], activation="gelu")
    close("dense", y, ref.dense(d["x"], d["weight"], d["bias"], None, "gelu")["y"], dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,inner,columns", [(1, 40, 24), (64, 64, 64), (130, 200, 72), (520, 128, 264), (300, 77, 51)])
def test_integer_products_are_exact(device, rows, inner, columns, dtype):
    """Small whole numbers: every product and sum is exact in f32, and the results, below 2^8, in
    either type, so any element taken from a wrong place shows."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randint(-1, 2, (rows, inner), generator=g, device="cuda").to(dtype)
    w = torch.randint(-1, 2, (inner, columns), generator=g, device="cuda").to(dtype)
    d = torch.randint(-1, 2, (rows, columns), generator=g, device="cuda").to(dtype)
    r = torch.randint(-3, 4, (rows, columns), generator=g, device="cuda").to(dtype)
    y = af2cuda.encode_dense_tensors(device, x, w, residual=r)
    grads = af2cuda.encode_dense_backward_tensors(device, d, x, w, bias=True)
    want = ref.dense(x, w, None, r, "none", d)
    for k, v in {"y": y, **grads}.items():
        assert want[k].abs().max().item() <= 256
        assert torch.equal(v.double(), want[k]), k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [8, 3])
def test_row_strides_and_untouched_surroundings(device, dtype, pad):
    """Rows further apart than they are wide, at 16-byte and at odd distances; what lies between
    the rows of an output and past its end stays as it was."""
    rows, c, h = 133, 72, 136
    s = gated_case(rows, c, h, dtype, seed=80)

    def spread(t):
        big = torch.full((t.shape[0] + 2, t.shape[1] + pad), 7.0, dtype=dtype, device="cuda")
        view = big[1:-1, :t.shape[1]]
        view.copy_(t)
        return big, view

    (_, x), (_, r), (_, d) = spread(s["x"]), spread(s["residual"]), spread(s["d_out"])
    big, out = spread(torch.zeros_like(s["x"]))
    y, saved = af2cuda.encode_gated_transition_tensors(device, x, s["weights"], residual=r, out=out, save=True)
    assert y is out
    grads = af2cuda.encode_gated_transition_backward_tensors(device, d, x, s["weights"], saved=saved)
    want = ref.gated(s["x"], s["weights"], s["residual"], "silu", s["d_out"])
    for k, v in {"y": out, **grads}.items():
        close(k, v, want[k], dtype)
    edge = big.clone()
    edge[1:-1, :c] = 7.0
    assert (edge == 7.0).all()
    dn = dense_case(rows, c, h, dtype, seed=90)
    (_, x), (_, d) = spread(dn["x"]), spread(dn["d_out"])
    big, out = spread(dn["residual"])
    _, saved = af2cuda.encode_dense_tensors(device, x, dn["weight"], bias=dn["bias"], residual=out, activation="silu",
                                            out=out, save=True)
    grads = af2cuda.encode_dense_backward_tensors(device, d, x, dn["weight"], saved=saved, bias=True, activation="silu")
    want = ref.dense(dn["x"], dn["weight"], dn["bias"], dn["residual"], "silu", dn["d_out"])
    for k, v in {"y": out, **grads}.items():
        close(k, v, want[k], dtype)
    edge = big.clone()
    edge[1:-1, :h] = 7.0
    assert (edge == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_at_odd_addresses(device, dtype):
    """Weights that are slices of one flat buffer, at addresses of their element size only."""
    c, h, rows = 48, 80, 70
    s = gated_case(rows, c, h, dtype, seed=100)
    flat = torch.zeros(sum(v.numel() for v in s["weights"].values()) + 8, dtype=dtype, device="cuda")
    views, at = {}, 1
    for k, v in s["weights"].items():
        views[k] = flat[at:at + v.numel()].view(v.shape)
        views[k].copy_(v)
        at += v.numel()
    got, want = run_gated(device, s, "gelu", weights=views)
    for k in got:
        close(k, got[k], want[k], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(device, dtype):
    s = gated_case(0, 24, 40, dtype)
    got, _ = run_gated(device, s, "silu")
    assert got["y"].shape == (0, 24) and got["x"].shape == (0, 24)
    for k, v in s["weights"].items():
        assert got[k].shape == v.shape and not got[k].any(), k
    d = dense_case(0, 24, 40, dtype)
    got, _ = run_dense(device, d, "relu")
    assert not got["weight"].any() and not got["bias"].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_bad_row_stays_in_its_row(device, dtype, value):
    s = gated_case(200, 64, 128, dtype, seed=110)
    clean = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"])
    x = s["x"].clone()
    x[137, 5] = value
    y = af2cuda.encode_gated_transition_tensors(device, x, s["weights"])
    assert not torch.isfinite(y[137]).any()
    keep = torch.arange(200, device="cuda") != 137
    assert torch.equal(y[keep], clean[keep])


def test_f32_gradients_against_differences(device):
    """Central differences of sum(y * d_out) in f32, eps 2^-6: the truncation is eps^2 times third
    derivatives (below 1e-3 of the gradient here), the rounding 2^-24 |loss| / eps."""
    rows, c, h, eps = 6, 10, 14, 2.0**-6
    s = gated_case(rows, c, h, F32, seed=120)
    got, _ = run_gated(device, s, "gelu")

    def loss(x, w):
        y = af2cuda.encode_gated_transition_tensors(device, x, w, residual=s["residual"], activation="gelu")
        return (y.double() * s["d_out"].double()).sum().item()

    tensors = {"x": s["x"], **s["weights"]}
    for name, t in tensors.items():
        for at in [(0,) * t.dim(), tuple(n - 1 for n in t.shape), tuple(n // 2 for n in t.shape)]:
            ends = []
            for sign in (1, -1):
                moved = {k: v.clone() for k, v in tensors.items()}
                moved[name][at] += sign * eps
                ends.append(loss(moved["x"], {k: moved[k] for k in s["weights"]}))
            diff = (ends[0] - ends[1]) / (2 * eps)
            scale = got[name].abs().max().item()
            assert abs(diff - got[name][at].item()) <= 2e-3 * scale, (name, at)


@pytest.mark.parametrize("dtype", DTYPES)
def test_results_do_not_change_from_call_to_call(device, dtype):
    """No order of sums depends on timing: the same inputs give the same bits."""
    s = gated_case(1500, 136, 264, dtype, seed=130)
    first, _ = run_gated(device, s, "silu")
    first = {k: v.clone() for k, v in first.items()}
    for _ in range(3):
        again, _ = run_gated(device, s, "silu")
        for k in first:
            assert torch.equal(first[k], again[k]), k


def test_weights_may_change_between_calls(device):
    s = dense_case(64, 128, 128, BF16, seed=140)
    a = af2cuda.encode_dense_tensors(device, s["x"], s["weight"]).clone()
    s["weight"].mul_(2)
    b = af2cuda.encode_dense_tensors(device, s["x"], s["weight"])
    assert torch.equal(2 * a, b)


def test_calls_on_two_streams_share_the_scratch_safely(device):
    """The context's scratch is one buffer: calls on two streams, without the host waiting, keep apart."""
    cases = [gated_case(700, 130, 260, F32, seed=150 + i) for i in range(2)]
    want = [ref.gated(s["x"], s["weights"], None, "silu")["y"] for s in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(af2cuda.encode_gated_transition_tensors(device, cases[i % 2]["x"], cases[i % 2]["weights"]))
    torch.cuda.synchronize()
    for i, y in enumerate(outs):
        close("y", y, want[i % 2], F32)


def test_an_explicit_stream_and_workspace(device):
    s = gated_case(300, 64, 128, BF16, seed=160)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    nbytes = af2cuda.gated_transition_workspace_bytes(300, 64, 128, BF16)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device="cuda")
    y = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], stream=side.cuda_stream, workspace=ws)
    side.synchronize()
    close("y", y, ref.gated(s["x"], s["weights"], None, "silu")["y"], BF16)


def test_captured_in_a_graph(device):
    s = gated_case(256, 64, 128, BF16, seed=170)
    out = torch.empty_like(s["x"])
    nbytes = af2cuda.gated_transition_workspace_bytes(256, 64, 128, BF16)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device="cuda")
    run = lambda: af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], out=out, workspace=ws)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    s["x"].mul_(-0.5)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    close("y", out, ref.gated(s["x"], s["weights"], None, "silu")["y"], BF16)


def test_parts_of_the_gradients(device):
    s = gated_case(200, 64, 96, BF16, seed=180)
    _, saved = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], save=True)
    want = ref.gated(s["x"], s["weights"], None, "silu", s["d_out"])
    for need in (["x"], ["outputWeight"], ["gateWeight"], ["valueWeight", "gateBias"], ["valueBias", "outputBias"]):
        got = af2cuda.encode_gated_transition_backward_tensors(device, s["d_out"], s["x"], s["weights"], saved=saved,
                                                               need=need)
        assert sorted(got) == sorted(need)
        for k in got:
            close(k, got[k], want[k], BF16)
    d = dense_case(200, 64, 96, F16, seed=190)
    for need in (["x"], ["weight"]):
        got = af2cuda.encode_dense_backward_tensors(device, d["d_out"], d["x"], d["weight"], need=need)
        assert list(got) == need


def test_refusals(device):
    s = gated_case(20, 16, 24, BF16)
    d = dense_case(20, 16, 24, BF16)
    dense, gated = af2cuda.encode_dense_tensors, af2cuda.encode_gated_transition_tensors
    with pytest.raises(af2cuda.RangeError, match="activation"):
        dense(device, d["x"], d["weight"], activation="tanh")
    with pytest.raises(af2cuda.RangeError, match="x has shape"):
        dense(device, d["x"], d["weight"].t())
    with pytest.raises(af2cuda.RangeError, match="weight"):
        dense(device, d["x"], d["weight"].float())
    with pytest.raises(af2cuda.RangeError, match="float32, float16 or bfloat16"):
        dense(device, d["x"].double(), d["weight"].double())
    with pytest.raises(af2cuda.RangeError, match="bias"):
        dense(device, d["x"], d["weight"], bias=d["bias"][:-1])
    with pytest.raises(af2cuda.RangeError, match="residual"):
        dense(device, d["x"], d["weight"], residual=d["residual"][:-1])
    with pytest.raises(af2cuda.RangeError, match="x must have contiguous rows"):
        dense(device, d["x"].t().contiguous().t(), d["weight"])
    with pytest.raises(af2cuda.RangeError, match="d_out must have contiguous rows"):
        af2cuda.encode_dense_backward_tensors(device, d["d_out"][:1].expand(20, 24), d["x"], d["weight"])
    with pytest.raises(af2cuda.RangeError, match="cuda:0"):
        dense(device, d["x"].cpu(), d["weight"].cpu())
    with pytest.raises(af2cuda.RangeError, match="saved"):
        af2cuda.encode_dense_backward_tensors(device, d["d_out"], d["x"], d["weight"], activation="silu")
    with pytest.raises(af2cuda.RangeError, match="gateWeight is missing"):
        gated(device, s["x"], {k: v for k, v in s["weights"].items() if k != "gateWeight"})
    with pytest.raises(af2cuda.RangeError, match="unknown weights"):
        gated(device, s["x"], {**s["weights"], "firstWeight": s["x"]})
    with pytest.raises(af2cuda.RangeError, match="outputWeight"):
        gated(device, s["x"], {**s["weights"], "outputWeight": s["weights"]["gateWeight"]})
    with pytest.raises(af2cuda.RangeError, match="workspace"):
        gated(device, s["x"], s["weights"], workspace=torch.empty(0, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,c,h", [(257, 128, 512), (300, 8, 24), (1000, 72, 200), (5000, 64, 64), (20000, 128, 136),
                                      (40001, 104, 1000), (513, 40, 2056), (700, 100, 300)])
def test_forward_of_narrow_transitions(device, rows, c, h, act, dtype):
    """Inference with up to 128 channels, past the few-row sizes: one tile to several per SM, hidden
    widths inside a chunk and past many, with and without the residual and the biases."""
    s = gated_case(rows, c, h, dtype, seed=200)
    y = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], residual=s["residual"], activation=act)
    close("y", y, ref.gated(s["x"], s["weights"], s["residual"], act)["y"], dtype)
    bare = {k: v for k, v in s["weights"].items() if k.endswith("Weight")}
    y = af2cuda.encode_gated_transition_tensors(device, s["x"], bare, activation=act)
    close("y", y, ref.gated(s["x"], bare, None, act)["y"], dtype)
    device.sync(1)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_saturated_gates(device, dtype):
    """Pre-activations far out on both sides: no overflow in the gate's exponentials."""
    s = gated_case(600, 64, 128, dtype, seed=210)
    s["x"].mul_(30)
    for act in ACTS:
        y = af2cuda.encode_gated_transition_tensors(device, s["x"], s["weights"], activation=act)
        want = ref.gated(s["x"], s["weights"], None, act)["y"]
        if dtype == BF16 or want.abs().max() < 6e4:
            close(act, y, want, dtype)
