"""The norm of a set of gradients and their clipping, against 64 bits.

The squares are summed in 64 bits and the norm rounded once to f32: 2^-23
relative bounds it.  A clipped element carries the factor's roundings (the sum,
the quotient) and its own: 2^-22 in f32, the type's unit roundoff more in a 16-bit one."""
import math

import pytest
import torch

import af2cuda
import layer_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def tensors(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * scale).to(dtypes[i % len(dtypes)])
            for i, n in enumerate(sizes)]


def exact_norm(ts) -> float:
    return math.sqrt(sum(t.double().square().sum().item() for t in ts))


SETS = {
    "one element": ([1], [F32]),
    "one": ([1000], [BF16]),
    "odd": ([1, 3, 7, 8191, 8192, 8193, 16385], [F32, BF16, F16]),
    "empty among others": ([0, 5, 0, 100000, 0], [BF16]),
    "many small": ([17 + i % 90 for i in range(1500)], [F32, BF16]),
    "large": ([3_000_001, 12, 5_000_000], [BF16, F32]),
    "table boundaries": ([33] * 64, [F16]),
    "past the table": ([33] * 65, [F16]),
}


@pytest.mark.parametrize("name", list(SETS))
def test_norm_and_clipping(device, name):
    sizes, dtypes = SETS[name]
    ts = tensors(sizes, dtypes, seed=len(name))
    want = exact_norm(ts)
    norm = af2cuda.encode_gradient_norm_tensors(device, ts)
    assert norm.dtype == F32 and norm.shape == ()
    assert abs(norm.item() - want) <= 2.0**-23 * want
    for limit in (0.3 * want, 4 * want):
        factor = min(1.0, limit / (want + 1e-6))
        before = [t.clone() for t in ts]
        outs = [torch.full_like(t, 9.0) for t in ts]
        got = af2cuda.encode_clip_gradients_tensors(device, ts, limit, out=outs)
        assert abs(got.item() - want) <= 2.0**-23 * want
        inplace = [t.clone() for t in ts]
        af2cuda.encode_clip_gradients_tensors(device, inplace, limit)
        for t, b, o, i in zip(ts, before, outs, inplace):
            assert torch.equal(t, b)
            assert torch.equal(o, i)
            tol = 2.0**-22 + (0 if t.dtype == F32 else ref.ROUNDOFF[t.dtype])
            tiny = 2.0**-24 if t.dtype == F16 else 0.0  # half the smallest step of f16 near zero, doubled
            assert ((o.double() - b.double() * factor).abs() <= tol * b.double().abs() * factor + tiny).all()


def test_views_at_odd_addresses(device):
    flat = tensors([10000], [BF16])[0]
    views, at = [], 1
    for n in (5, 1, 100, 4097, 33, 2048):
        views.append(flat[at:at + n])
        at += n + 1
    want = exact_norm(views)
    before = flat.clone()
    norm = af2cuda.encode_clip_gradients_tensors(device, views, want / 3)
    assert abs(norm.item() - want) <= 2.0**-23 * want
    touched = torch.zeros_like(flat, dtype=torch.bool)
    at = 1
    for n in (5, 1, 100, 4097, 33, 2048):
        touched[at:at + n] = True
        at += n + 1
    assert torch.equal(flat[~touched], before[~touched])
    err = (flat[touched].double() - before[touched].double() / 3).abs()
    assert (err <= (ref.ROUNDOFF[BF16] + 2e-6) * before[touched].double().abs()).all()


def test_outputs_at_other_alignments(device):
    src = tensors([5001], [F32])[0]
    buf = torch.zeros(5010, device="cuda")
    for shift in (0, 1, 2, 3):
        out = buf[shift:shift + 5000]
        af2cuda.encode_clip_gradients_tensors(device, [src[1:]], 1.0, out=[out])
        want = src[1:].double() / (exact_norm([src[1:]]) + 1e-6)
        assert ((out.double() - want).abs() <= 2.0**-22 * want.abs()).all()


def test_no_tensors(device):
    assert af2cuda.encode_gradient_norm_tensors(device, []).item() == 0.0
    assert af2cuda.encode_clip_gradients_tensors(device, [], 1.0).item() == 0.0
    empty = torch.empty(0, device="cuda")
    assert af2cuda.encode_clip_gradients_tensors(device, [empty], 1.0).item() == 0.0


def test_zero_gradients_and_a_zero_limit(device):
    z = torch.zeros(1000, device="cuda")
    assert af2cuda.encode_clip_gradients_tensors(device, [z], 1.0).item() == 0.0
    assert not z.any()
    t = tensors([1000], [F32])[0]
    af2cuda.encode_clip_gradients_tensors(device, [t], 0.0)
    assert not t.any()


@pytest.mark.parametrize("dtype,value", [(F32, 1e30), (F32, 3e38), (F32, 1e-30), (BF16, 1e38), (F16, 60000.0)])
def test_squares_do_not_overflow_or_vanish(device, dtype, value):
    t = torch.full((100,), value, dtype=dtype, device="cuda")
    want = exact_norm([t])
    got = af2cuda.encode_gradient_norm_tensors(device, [t]).item()
    if want < 3.4e38:
        assert abs(got - want) <= 2.0**-23 * want
    else:
        assert math.isinf(got)


def test_infinite_and_nan_elements(device):
    t = tensors([5000], [F32])[0]
    t[77] = float("inf")
    norm = af2cuda.encode_clip_gradients_tensors(device, [t], 1.0)
    assert math.isinf(norm.item())
    assert torch.isnan(t[77]) and not t[torch.arange(5000, device="cuda") != 77].any()
    t = tensors([5000], [BF16])[0]
    t[4999] = float("nan")
    norm = af2cuda.encode_clip_gradients_tensors(device, [t, torch.ones(10, device="cuda")], 1.0)
    assert math.isnan(norm.item()) and torch.isnan(t).all()


def test_the_sum_has_one_order(device):
    ts = tensors([100003, 7, 65536, 999], [F32, BF16])
    first = af2cuda.encode_gradient_norm_tensors(device, ts).item()
    for _ in range(5):
        assert af2cuda.encode_gradient_norm_tensors(device, ts).item() == first


def test_on_another_stream(device):
    ts = tensors([300000, 11], [F32])
    want = exact_norm(ts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm = af2cuda.encode_clip_gradients_tensors(device, ts, want / 3)
    side.synchronize()
    assert abs(norm.item() - want) <= 2.0**-23 * want
    assert abs(exact_norm(ts) - want / 3) <= 1e-5 * want


def test_refusals(device):
    t = tensors([100], [F32])[0]
    with pytest.raises(af2cuda.RangeError, match="contiguous"):
        af2cuda.encode_gradient_norm_tensors(device, [t.view(10, 10).t()])
    with pytest.raises(af2cuda.RangeError, match="cuda:0"):
        af2cuda.encode_gradient_norm_tensors(device, [t.cpu()])
    with pytest.raises(af2cuda.RangeError, match="float32, float16 or bfloat16"):
        af2cuda.encode_gradient_norm_tensors(device, [t.double()])
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(af2cuda.RangeError, match="max_norm"):
            af2cuda.encode_clip_gradients_tensors(device, [t], bad)
    with pytest.raises(af2cuda.RangeError, match="expected 1"):
        af2cuda.encode_clip_gradients_tensors(device, [t], 1.0, out=[t, t])
    with pytest.raises(af2cuda.RangeError, match="size or type"):
        af2cuda.encode_clip_gradients_tensors(device, [t], 1.0, out=[t[:50]])
    with pytest.raises(af2cuda.RangeError, match="size or type"):
        af2cuda.encode_clip_gradients_tensors(device, [t], 1.0, out=[torch.empty(100, dtype=BF16, device="cuda")])
