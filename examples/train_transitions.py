"""Trains a stack of gated transitions with a dense head on one GPU: the layers' forward and
backward passes, the norm over all gradients, and clipping, as a training program calls them.

    python examples/train_transitions.py --length 256 --channels 128 --hidden 512 --blocks 4 --steps 20

The data are synthetic: the head learns to answer a fixed random projection of its input.
"""
import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "alphafold2-webgpu_b200"))

import torch

import af2cuda


def parameters(channels: int, hidden: int, blocks: int, bins: int, dtype, seed: int = 0) -> dict:
    """Random weights: a list of transitions by the names their entry point takes, and the head's."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*size):
        return (torch.randn(size, generator=g, device="cuda") * size[0] ** -0.5).to(dtype)

    def zeros(n):
        return torch.zeros(n, device="cuda", dtype=dtype)

    return {"blocks": [{"gateWeight": normal(channels, hidden), "gateBias": zeros(hidden),
                        "valueWeight": normal(channels, hidden), "valueBias": zeros(hidden),
                        "outputWeight": normal(hidden, channels), "outputBias": zeros(channels)} for _ in range(blocks)],
            "head": {"weight": normal(channels, bins), "bias": zeros(bins)}}


def answer(device, p: dict, x):
    """The model's answer for rows x [rows, channels], nothing kept for a backward pass."""
    for w in p["blocks"]:
        x = af2cuda.encode_gated_transition_tensors(device, x, w, residual=x)
    return af2cuda.encode_dense_tensors(device, x, p["head"]["weight"], bias=p["head"]["bias"])


def loss_and_gradients(device, p: dict, x, target):
    """The mean squared error against target [rows, bins], and its gradient by every weight (laid out as
    `p`)."""
    inputs, kept = [], []
    for w in p["blocks"]:
        inputs.append(x)
        x, saved = af2cuda.encode_gated_transition_tensors(device, x, w, residual=x, save=True)
        kept.append(saved)
    out = af2cuda.encode_dense_tensors(device, x, p["head"]["weight"], bias=p["head"]["bias"])
    error = out.float() - target
    loss = error.square().mean()
    d = (error * (2 / error.numel())).to(out.dtype)

    head = af2cuda.encode_dense_backward_tensors(device, d, x, p["head"]["weight"], bias=True)
    d = head.pop("x")
    grads = {"blocks": [None] * len(p["blocks"]), "head": head}
    for i in reversed(range(len(p["blocks"]))):
        g = af2cuda.encode_gated_transition_backward_tensors(device, d, inputs[i], p["blocks"][i], saved=kept[i])
        d = d + g.pop("x")  # the residual passes d on as it is
        grads["blocks"][i] = g
    return loss, grads


def flat(p: dict) -> list:
    return [w[name] for w in [*p["blocks"], p["head"]] for name in sorted(w)]


def train_step(device, p: dict, x, target, rate: float, max_norm: float):
    """One step of gradient descent with clipped gradients; the loss and the norm before clipping."""
    loss, grads = loss_and_gradients(device, p, x, target)
    grads = flat(grads)
    norm = af2cuda.encode_clip_gradients_tensors(device, grads, max_norm)
    torch._foreach_add_(flat(p), grads, alpha=-rate)
    return loss, norm


def main(argv=None) -> list:
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    a.add_argument("--length", type=int, default=128, help="residues; the pair has length^2 rows")
    a.add_argument("--channels", type=int, default=128)
    a.add_argument("--hidden", type=int, default=512)
    a.add_argument("--blocks", type=int, default=4)
    a.add_argument("--bins", type=int, default=64)
    a.add_argument("--steps", type=int, default=20)
    a.add_argument("--rate", type=float, default=1.0)
    a.add_argument("--max-norm", type=float, default=1.0)
    a.add_argument("--dtype", choices=("float32", "bfloat16", "float16"), default="float32")
    a = a.parse_args(argv)

    device = af2cuda.Device(0)
    dtype = getattr(torch, a.dtype)
    p = parameters(a.channels, a.hidden, a.blocks, a.bins, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((a.length * a.length, a.channels), generator=g, device="cuda").to(dtype)
    target = x.float() @ torch.randn((a.channels, a.bins), generator=g, device="cuda") * a.channels ** -0.5
    losses = []
    for step in range(a.steps):
        loss, norm = train_step(device, p, x, target, a.rate, a.max_norm)
        losses.append(float(loss))
        print(f"step {step:3d}  loss {losses[-1]:.5f}  gradient norm {float(norm):.4f}")
    return losses


if __name__ == "__main__":
    main()
