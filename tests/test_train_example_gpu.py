"""The training example: its gradients against autograd in 64 bits, and that it learns."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

# f32 products keep 24 bits, and a sum of k of them is within about sqrt(k) of f32's half roundoff
# (2^-24) of its terms' size; the longest here is 300 rows, a gradient passes some ten of them one after
# the other, and cancellation may cost a factor of 100 more: 10 * sqrt(300) * 100 * 2^-24 = 1.1e-3.
TOLERANCE = 1.1e-3


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "train_transitions.py"
    spec = importlib.util.spec_from_file_location("train_transitions", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _plain_loss(p, x, target):
    for w in p["blocks"]:
        gate = torch.nn.functional.silu(x @ w["gateWeight"] + w["gateBias"])
        x = x + (gate * (x @ w["valueWeight"] + w["valueBias"])) @ w["outputWeight"] + w["outputBias"]
    return (x @ p["head"]["weight"] + p["head"]["bias"] - target).square().mean(), x


@pytest.mark.parametrize("rows,channels,hidden,bins", [(300, 48, 100, 17), (1, 64, 128, 8)])
def test_gradients_and_clipping(rows, channels, hidden, bins):
    import af2cuda
    m = _example()
    device = af2cuda.Device(0)
    p = m.parameters(channels, hidden, 2, bins, torch.float32, seed=3)
    x = torch.randn(rows, channels, device="cuda")
    target = torch.randn(rows, bins, device="cuda")
    exact = {"blocks": [{k: v.double().requires_grad_() for k, v in w.items()} for w in p["blocks"]],
             "head": {k: v.double().requires_grad_() for k, v in p["head"].items()}}
    want, _ = _plain_loss(exact, x.double(), target.double())
    want.backward()
    want = want.detach()
    want_grads = [v.grad for v in m.flat(exact)]
    loss, grads = m.loss_and_gradients(device, p, x, target)
    grads = m.flat(grads)
    assert abs(float(loss) - float(want)) <= TOLERANCE * float(want)
    for got, exact_grad in zip(grads, want_grads):
        scale = float(exact_grad.norm()) + 1e-30
        assert float((got.double() - exact_grad).norm()) <= TOLERANCE * scale
    want_norm = float(torch.stack([g.norm() for g in want_grads]).norm())
    norm = af2cuda.encode_clip_gradients_tensors(device, grads, 0.25 * want_norm)
    assert abs(float(norm) - want_norm) <= TOLERANCE * want_norm
    clipped = float(torch.stack([g.double().norm() for g in grads]).norm())
    assert abs(clipped - 0.25 * want_norm) <= 2 * TOLERANCE * want_norm


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_it_learns(dtype):
    losses = _example().main(["--length", "24", "--channels", "64", "--hidden", "128", "--blocks", "2", "--bins", "16",
                              "--steps", "30", "--dtype", dtype])
    assert losses[-1] < 0.5 * losses[0]


def test_answer_matches_the_training_pass():
    import af2cuda
    m = _example()
    device = af2cuda.Device(0)
    p = m.parameters(64, 128, 2, 16, torch.float32)
    x = torch.randn(200, 64, device="cuda")
    exact = {"blocks": [{k: v.double() for k, v in w.items()} for w in p["blocks"]],
             "head": {k: v.double() for k, v in p["head"].items()}}
    _, hidden = _plain_loss(exact, x.double(), torch.zeros(200, 16, device="cuda", dtype=torch.float64))
    want = hidden @ exact["head"]["weight"] + exact["head"]["bias"]
    got = m.answer(device, p, x)
    assert float((got.double() - want).norm()) <= TOLERANCE * float(want.norm())
