"""The layers with learned weights in 64 bits, for the tests."""
from __future__ import annotations

import math

import torch

# unit roundoff: the most, relative, that rounding to the type changes a value by
ROUNDOFF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
# what it changes a whole tensor by in the 2-norm: the errors spread evenly over the spacing, whose
# root mean square, relative to values spread evenly over a binade, is 0.42 of the roundoff
UNIT = {k: v / 2 for k, v in ROUNDOFF.items()}


def act(kind: str, z):
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "sigmoid":
        return torch.sigmoid(z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    return z


def slope(kind: str, z):
    if kind == "relu":
        return (z > 0).double()
    if kind == "sigmoid":
        return torch.sigmoid(z) * torch.sigmoid(-z)
    if kind == "silu":
        s = torch.sigmoid(z)
        return s + z * s * torch.sigmoid(-z)
    if kind == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def dense(x, weight, bias, residual, kind, d_out=None) -> dict:
    x, weight = x.double(), weight.double()
    z = x @ weight
    if bias is not None:
        z = z + bias.double()
    y = act(kind, z)
    out = {"y": y if residual is None else y + residual.double()}
    if d_out is not None:
        dz = d_out.double() * slope(kind, z)
        out |= {"x": dz @ weight.t(), "weight": x.t() @ dz, "bias": dz.sum(0)}
    return out


def gated(x, weights: dict, residual, kind, d_out=None) -> dict:
    x = x.double()
    w = {k: v.double() for k, v in weights.items() if v is not None}
    g, v = x @ w["gateWeight"], x @ w["valueWeight"]
    if "gateBias" in w:
        g = g + w["gateBias"]
    if "valueBias" in w:
        v = v + w["valueBias"]
    a = act(kind, g)
    h = a * v
    y = h @ w["outputWeight"]
    if "outputBias" in w:
        y = y + w["outputBias"]
    out = {"y": y if residual is None else y + residual.double()}
    if d_out is not None:
        dy = d_out.double()
        dh = dy @ w["outputWeight"].t()
        dg, dv = dh * v * slope(kind, g), dh * a
        out |= {"x": dg @ w["gateWeight"].t() + dv @ w["valueWeight"].t(), "gateWeight": x.t() @ dg,
                "valueWeight": x.t() @ dv, "outputWeight": h.t() @ dy, "gateBias": dg.sum(0),
                "valueBias": dv.sum(0), "outputBias": dy.sum(0)}
    return out


def relative(got, want) -> float:
    """2-norm of the difference over the 2-norm of the reference."""
    d, n = (got.double() - want).norm().item(), want.norm().item()
    return d / n if n else d
