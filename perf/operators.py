"""The training and serving operators of a transition block, as they are measured.

Three operators that a transition with learned weights is made of:

* the dense layer, ``act(x W + b) (+ residual)``, with its backward pass;
* the gated transition, ``(act(x Wg + bg) * (x Wv + bv)) Wo + bo (+ residual)``, with its
  backward pass;
* the global norm of a set of gradients, and their clipping by it.

A case is a dict of sizes and options.  ``prepare`` makes its inputs from a seed, ``run`` makes one
pass: in elementary torch operations in 32 bits, rounded once at the end, where ``own`` is false;
through the framework's entry points where it is true.  ``exact`` gives the same outputs from the
definitions in 64 bits, and ``work`` what a pass cannot do without.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_ACTIVATIONS = ("none", "relu", "sigmoid", "silu", "gelu")
_CLIP_EPSILON = 1e-6


# ---- the cases -----------------------------------------------------------------------------------


def _gated(name, rows, channels, hidden, dtype, activation="silu", bias=True, residual=True, train=False):
    return {"name": name, "op": "gated", "rows": rows, "channels": channels, "hidden": hidden, "dtype": dtype,
            "activation": activation, "bias": bias, "residual": residual, "train": train}


def _dense(name, rows, inner, columns, dtype, activation="none", bias=True, residual=False, train=False):
    return {"name": name, "op": "dense", "rows": rows, "inner": inner, "columns": columns, "dtype": dtype,
            "activation": activation, "bias": bias, "residual": residual, "train": train}


def _gradients(name, blocks, channels, hidden, dtype, clip, limit=0.5):
    return {"name": name, "op": "gradients", "blocks": blocks, "channels": channels, "hidden": hidden,
            "dtype": dtype, "clip": clip, "limit": limit}


def listed():
    return [
        # serving one token through a wide gated transition: latency and the read of the weights
        _gated("gated_one_token", 1, 1024, 4096, "bf16"),
        # a few tokens at once (a small batch of sequences, one position each)
        _gated("gated_few_rows", 24, 512, 2048, "f16", activation="gelu"),
        # the pair of 512 residues through a pair-sized transition (128 -> 512 -> 128), inference
        _gated("gated_pair_512", 512 * 512, 128, 512, "bf16"),
        # a training step over an MSA of 64 sequences and 512 residues (256 -> 1024 -> 256)
        _gated("gated_msa_train", 64 * 512, 256, 1024, "bf16", train=True),
        # a training step of a wide transition over 8192 positions
        _gated("gated_wide_train", 8192, 1024, 4096, "bf16", bias=False, train=True),
        # a training step in full precision with odd sizes (a crop of 39 x 39 residues)
        _gated("gated_odd_f32_train", 39 * 39, 130, 390, "f32", activation="gelu", train=True),
        # one position through one projection
        _dense("dense_one_row", 1, 1024, 1024, "bf16", activation="relu"),
        # a training step of a projection with ragged sizes, none of them a multiple of a tile
        _dense("dense_ragged_train", 3001, 259, 387, "f16", activation="silu", train=True),
        # a training step of a wide layer over 16384 positions
        _dense("dense_wide_train", 16384, 1024, 4096, "bf16", activation="gelu", train=True),
        # the norm of one pair-sized block's gradients, for the log of a step
        _gradients("norm_one_block", 1, 128, 512, "f32", False),
        # clipping the f32 gradients of 48 pair-sized blocks: many small tensors
        _gradients("clip_pair_stack", 48, 128, 512, "f32", True),
        # clipping the bf16 gradients of 8 wide blocks: a few large tensors
        _gradients("clip_wide_stack", 8, 1024, 4096, "bf16", True),
    ]


#: The operations of the largest listed case; no drawn case has more.
_MOST_FLOPS = 18 * 8192 * 1024 * 4096
#: Elements of the largest intermediate that a drawn case may have.
_MOST_HIDDEN = 512 * 512 * 512


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("gated", "gated", "dense", "dense", "gradients"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    channels = _log_int(rng, 32, 1024)
    hidden = _log_int(rng, channels, 4 * channels)
    if rng.random() < 0.6:  # most layers have widths of whole 16-byte pieces; the others are odd
        channels, hidden = (channels + 7) // 8 * 8, (hidden + 7) // 8 * 8
    if op == "gradients":
        blocks = _log_int(rng, 1, max(1, min(64, 100_000_000 // (3 * channels * hidden))))
        case = _gradients("", blocks, channels, hidden, dtype, rng.random() < 0.7, rng.choice((0.5, 1e6)))
    else:
        train = rng.random() < 0.5
        rows = _log_int(rng, 1, 512 * 512)
        # f32 products cost several times the 16-bit ones
        most = _MOST_FLOPS // (6 if dtype == "f32" else 1)
        rows = max(1, min(rows, most // (18 * channels * hidden), _MOST_HIDDEN // hidden))
        activation = rng.choice(_ACTIVATIONS)
        bias, residual = rng.random() < 0.5, rng.random() < 0.5
        if op == "gated":
            case = _gated("", rows, channels, hidden, dtype, activation, bias, residual, train)
        else:
            inner, columns = (channels, hidden) if rng.random() < 0.5 else (hidden, channels)
            case = _dense("", rows, inner, columns, dtype, activation, bias, residual, train)
    del case["name"]
    return case


def _block_shapes(case):
    c, h = case["channels"], case["hidden"]
    return [(c,), (c,), (c, h), (h,), (c, h), (h,), (h, c), (c,)]  # a norm's two vectors, then the layers


def prepare(case, seed):
    """Normalised activations of unit variance, weights of variance 1 / fan-in, small biases, and
    for a training step the gradient that arrives at the output."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    if case["op"] == "gradients":
        # the scale of a gradient differs from tensor to tensor
        shapes = [s for _ in range(case["blocks"]) for s in _block_shapes(case)]
        grads = [normal(s, 10.0 ** -(1 + i % 3)) for i, s in enumerate(shapes)]
        # the clipped gradients go to one flat buffer, each tensor a view of its part
        flat = torch.empty(sum(t.numel() for t in grads), dtype=dtype, device="cuda")
        parts = torch.split(flat, [t.numel() for t in grads])
        return {"case": case, "gradients": grads, "flat": flat, "out": [p.view(t.shape) for p, t in zip(parts, grads)]}
    rows = case["rows"]
    if case["op"] == "dense":
        i, c = case["inner"], case["columns"]
        state = {"x": normal((rows, i)), "weight": normal((i, c), i ** -0.5),
                 "bias": normal((c,), 0.2) if case["bias"] else None,
                 "residual": normal((rows, c)) if case["residual"] else None}
        out = c
    else:
        c, h = case["channels"], case["hidden"]
        weights = {"gateWeight": normal((c, h), c ** -0.5), "valueWeight": normal((c, h), c ** -0.5),
                   "outputWeight": normal((h, c), h ** -0.5)}
        if case["bias"]:
            weights |= {"gateBias": normal((h,), 0.2), "valueBias": normal((h,), 0.2), "outputBias": normal((c,), 0.2)}
        state = {"x": normal((rows, c)), "weights": weights,
                 "residual": normal((rows, c)) if case["residual"] else None}
        out = c
    state["d_out"] = normal((rows, out), 1.0 / 16) if case["train"] else None
    return {"case": case, **state}


# ---- the plain form ------------------------------------------------------------------------------


def _act(kind, z):
    if kind == "none":
        return z
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return z * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))))
    s = 1 / (1 + torch.exp(-z))
    return s if kind == "sigmoid" else z * s


def _act_slope(kind, z):
    if kind == "none":
        return torch.ones_like(z)
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 - s) if kind == "sigmoid" else s * (1 + z * (1 - s))


def _plain_dense(s, case):
    dtype, kind = s["x"].dtype, case["activation"]
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(kind, z)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        dz = s["d_out"].float() * _act_slope(kind, z)
        out["d_x"] = (dz @ w.t()).to(dtype)
        out["d_weight"] = (x.t() @ dz).to(dtype)
        if s["bias"] is not None:
            out["d_bias"] = dz.sum(0).to(dtype)
    return out


def _plain_gated(s, case):
    dtype, kind = s["x"].dtype, case["activation"]
    w = {k: v.float() for k, v in s["weights"].items()}
    x = s["x"].float()
    gate, value = x @ w["gateWeight"], x @ w["valueWeight"]
    if case["bias"]:
        gate, value = gate + w["gateBias"], value + w["valueBias"]
    a = _act(kind, gate)
    hidden = a * value
    y = hidden @ w["outputWeight"]
    if case["bias"]:
        y = y + w["outputBias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        dy = s["d_out"].float()
        dh = dy @ w["outputWeight"].t()
        dg, dv = dh * value * _act_slope(kind, gate), dh * a
        out["d_x"] = (dg @ w["gateWeight"].t() + dv @ w["valueWeight"].t()).to(dtype)
        out["d_gateWeight"] = (x.t() @ dg).to(dtype)
        out["d_valueWeight"] = (x.t() @ dv).to(dtype)
        out["d_outputWeight"] = (hidden.t() @ dy).to(dtype)
        if case["bias"]:
            out["d_gateBias"] = dg.sum(0).to(dtype)
            out["d_valueBias"] = dv.sum(0).to(dtype)
            out["d_outputBias"] = dy.sum(0).to(dtype)
    return out


def _plain_gradients(s, case):
    norm = torch.stack([g.float().square().sum() for g in s["gradients"]]).sum().sqrt()
    if not case["clip"]:
        return {"norm": norm}
    scale = torch.clamp(case["limit"] / (norm + _CLIP_EPSILON), max=1.0)
    _ = [o.copy_(g.float() * scale) for o, g in zip(s["out"], s["gradients"])]
    return {"norm": norm, "clipped": s["flat"]}


# ---- through the framework -----------------------------------------------------------------------


_opened = {}


def _framework():
    """The framework's package and one open device, as a user's program has them."""
    if not _opened:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "alphafold2-webgpu_b200"))
        import af2cuda
        _opened["package"], _opened["device"] = af2cuda, af2cuda.Device(torch.cuda.current_device())
    return _opened["package"], _opened["device"]


def _own_dense(s, case):
    af2, device = _framework()
    if not case["train"]:
        return {"y": af2.encode_dense_tensors(device, s["x"], s["weight"], bias=s["bias"], residual=s["residual"],
                                              activation=case["activation"])}
    y, saved = af2.encode_dense_tensors(device, s["x"], s["weight"], bias=s["bias"], residual=s["residual"],
                                        activation=case["activation"], save=True)
    grads = af2.encode_dense_backward_tensors(device, s["d_out"], s["x"], s["weight"], saved=saved,
                                              bias=s["bias"] is not None, activation=case["activation"])
    out = {"y": y, "d_x": grads["x"], "d_weight": grads["weight"]}
    if s["bias"] is not None:
        out["d_bias"] = grads["bias"]
    return out


def _own_gated(s, case):
    af2, device = _framework()
    if not case["train"]:
        return {"y": af2.encode_gated_transition_tensors(device, s["x"], s["weights"], residual=s["residual"],
                                                         activation=case["activation"])}
    y, saved = af2.encode_gated_transition_tensors(device, s["x"], s["weights"], residual=s["residual"],
                                                   activation=case["activation"], save=True)
    grads = af2.encode_gated_transition_backward_tensors(device, s["d_out"], s["x"], s["weights"], saved=saved,
                                                         activation=case["activation"])
    return {"y": y, **{"d_" + k: v for k, v in grads.items()}}


def _own_gradients(s, case):
    af2, device = _framework()
    if not case["clip"]:
        return {"norm": af2.encode_gradient_norm_tensors(device, s["gradients"])}
    norm = af2.encode_clip_gradients_tensors(device, s["gradients"], case["limit"], out=s["out"])
    return {"norm": norm, "clipped": s["flat"]}


def run(state):
    case = state["case"]
    if own:
        return {"dense": _own_dense, "gated": _own_gated, "gradients": _own_gradients}[case["op"]](state, case)
    return {"dense": _plain_dense, "gated": _plain_gated, "gradients": _plain_gradients}[case["op"]](state, case)


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "gradients":
        n = case["blocks"] * sum(math.prod(s) for s in _block_shapes(case))
        return {"bytes": n * e * (2 if case["clip"] else 1) + 4, "flops": n * (3 if case["clip"] else 2)}
    rows = case["rows"]
    if case["op"] == "dense":
        i, c = case["inner"], case["columns"]
        tensors = rows * i + i * c + (c if case["bias"] else 0) + rows * c * (2 if case["residual"] else 1)
        if case["train"]:  # d_out in; d_x, d_weight and d_bias out
            tensors += rows * c + rows * i + i * c + (c if case["bias"] else 0)
        return {"bytes": e * tensors, "flops": (6 if case["train"] else 2) * rows * i * c}
    c, h = case["channels"], case["hidden"]
    weights = 3 * c * h + (2 * h + c if case["bias"] else 0)
    tensors = rows * c * (3 if case["residual"] else 2) + weights
    if case["train"]:  # d_out in; d_x and the weights' gradients out
        tensors += 2 * rows * c + weights
    return {"bytes": e * tensors, "flops": (18 if case["train"] else 6) * rows * c * h}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    up = lambda t: None if t is None else t.to(torch.float64)  # noqa: E731
    if case["op"] == "gradients":
        flat = torch.cat([up(g).flatten() for g in s["gradients"]])
        norm = torch.linalg.vector_norm(flat)
        if not case["clip"]:
            return {"norm": norm}
        factor = min(1.0, case["limit"] / (float(norm) + _CLIP_EPSILON))
        return {"norm": norm, "clipped": flat * factor}

    # value and slope of each activation, from the standard normal and logistic distributions
    normal_cdf = torch.special.ndtr
    normal_pdf = lambda z: torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)  # noqa: E731
    value_of = {"none": lambda z: z, "relu": lambda z: z.clamp(min=0), "sigmoid": torch.sigmoid,
                "silu": lambda z: z * torch.sigmoid(z), "gelu": lambda z: z * normal_cdf(z)}[case["activation"]]
    slope_of = {"none": lambda z: torch.ones_like(z), "relu": lambda z: torch.heaviside(z, torch.zeros_like(z)),
                "sigmoid": lambda z: torch.sigmoid(z) * torch.sigmoid(-z),
                "silu": lambda z: torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z),
                "gelu": lambda z: normal_cdf(z) + z * normal_pdf(z)}[case["activation"]]
    x, dy, skip = up(s["x"]), up(s["d_out"]), up(s["residual"])
    if case["op"] == "dense":
        w = up(s["weight"])
        z = torch.mm(x, w) if s["bias"] is None else torch.addmm(up(s["bias"]), x, w)
        answer = {"y": value_of(z) if skip is None else skip + value_of(z)}
        if case["train"]:
            dz = slope_of(z).mul_(dy)
            answer |= {"d_x": torch.mm(dz, w.mT), "d_weight": torch.mm(x.mT, dz)}
            if s["bias"] is not None:
                answer["d_bias"] = torch.mv(dz.mT, torch.ones_like(dz[:, 0]))
        return answer

    w = {k: up(v) for k, v in s["weights"].items()}
    project = lambda a, name: (torch.addmm(w[name + "Bias"], a, w[name + "Weight"]) if case["bias"]  # noqa: E731
                               else torch.mm(a, w[name + "Weight"]))
    g, v = project(x, "gate"), project(x, "value")
    h = value_of(g) * v
    y = project(h, "output")
    answer = {"y": y if skip is None else skip + y}
    if case["train"]:
        dh = torch.mm(dy, w["outputWeight"].mT)
        answer["d_outputWeight"] = torch.mm(h.mT, dy)
        del h
        dv = dh * value_of(g)
        dg = dh.mul_(v).mul_(slope_of(g))
        answer["d_x"] = torch.addmm(torch.mm(dg, w["gateWeight"].mT), dv, w["valueWeight"].mT)
        answer |= {"d_gateWeight": torch.mm(x.mT, dg), "d_valueWeight": torch.mm(x.mT, dv)}
        if case["bias"]:
            answer |= {"d_gateBias": torch.sum(dg, dim=0), "d_valueBias": torch.sum(dv, dim=0),
                       "d_outputBias": torch.sum(dy, dim=0)}
    return answer
