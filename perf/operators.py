"""Feed-forward operators of a transformer block on one MI355X: plain forms, calls and 64-bit values.

``gated``: v * act(g) of both projections z = x w^T + b (w holds the value rows, then the gate rows, or
the other way round). ``linear``: act(x w^T + b) + residual. Each in its forward direction and its
backward one, which takes the output's gradient and forms the projections again from x and w.
The listed cases are points of the ranges that ``draw`` samples: the feed-forward blocks of the UNet's
two levels, the text encoders' and the time embedding's MLPs, generic widths, rows from one to 8192.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_DEVICE = "cuda:0"
_SQRT_HALF = 0.7071067811865476


def _library():
    package = os.path.join(os.getcwd(), "sdxl-end2end_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import sdxl_hip
    return sdxl_hip


# ------------------------------------------------------------------------------------ the cases
def _gated(rows, width, inner, dtype="f16", activation="gelu", weights="same", bias=True, gate_first=False,
           backward=False, x_pad=0):
    return {"kind": "gated", "rows": rows, "width": width, "inner": inner, "dtype": dtype, "activation": activation,
            "weights": weights, "bias": bias, "gate_first": gate_first, "backward": backward, "x_pad": x_pad}


def _linear(rows, width, inner, dtype="f16", activation="none", weights="same", bias=True, residual=False,
            backward=False, x_pad=0):
    return {"kind": "linear", "rows": rows, "width": width, "inner": inner, "dtype": dtype, "activation": activation,
            "weights": weights, "bias": bias, "residual": residual, "backward": backward, "x_pad": x_pad}


def listed():
    cases = {
        # One row through a gated projection: serving one token, the weights' transfer is all there is.
        "gated_one_row": _gated(1, 1280, 5120, dtype="bf16", activation="silu", bias=False, gate_first=True),
        # The UNet's level-2 block, a 1024 x 1024 image with guidance (2 x 1024 tokens).
        "gated_l2": _gated(2048, 1280, 5120),
        # The level-1 block of a non-square image (2 x 38 x 65 tokens, no tile's multiple), E4M3 weights.
        "gated_l1_ragged_e4m3": _gated(4940, 640, 2560, weights="e4m3"),
        # A generic gated block without biases, an inner width of 8/3 of the width: long batch, bf16.
        "gated_wide": _gated(8192, 2048, 5456, dtype="bf16", activation="silu", bias=False, gate_first=True),
        # Training the level-2 block; the same for few ragged rows at level 1; and the largest call.
        "gated_backward_l2": _gated(2048, 1280, 5120, backward=True),
        "gated_backward_ragged": _gated(1111, 640, 2560, dtype="bf16", backward=True),
        "gated_backward_large": _gated(8192, 1280, 5120, dtype="bf16", activation="silu", backward=True),
        # The time embedding's first layer, a guided batch: the smallest call, all latency.
        "linear_time_embedding": _linear(2, 320, 1280, activation="silu"),
        # The text encoder's MLP, 2 x 77 tokens, in fp16.
        "linear_text_mlp": _linear(154, 1280, 5120, activation="gelu"),
        # The level-1 block's output projection with bias and residual.
        "linear_l1_out": _linear(8192, 2560, 640, residual=True),
        # Training the text encoder's MLP on 32 prompts, bf16; training the level-1 output projection.
        "linear_backward_text": _linear(2464, 1280, 5120, dtype="bf16", activation="gelu", backward=True),
        "linear_backward_l1_out": _linear(8192, 2560, 640, residual=True, backward=True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


_LARGEST_FLOPS = 12.0 * 8192 * 1280 * 5120


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    backward = rng.random() < 0.4
    rows = _log_int(rng, 16 if backward else 1, 16384)
    width = rng.choice((320, 640, 1280, 2048, 8 * _log_int(rng, 16, 256)))
    if rng.random() < 0.08:  # a row that no 16-byte load divides
        width += rng.randint(1, 7)
    inner = rng.choice((4 * width, 8 * (width // 3), 8 * _log_int(rng, 16, 700)))
    if rng.random() < 0.2:
        inner += rng.randint(1, 7)
    dtype = rng.choice(("f16", "bf16"))
    # (a step in the slope, as relu's, is a border that no two orders of summation agree on)
    activation = rng.choice(("gelu", "gelu", "silu", "gelu_tanh", "quick_gelu", "silu" if backward else "relu"))
    weights = "e4m3" if not backward and rng.random() < 0.25 else "same"
    bias, x_pad = rng.random() < 0.7, rng.choice((0, 0, 0, 64, 8))
    if rng.random() < 0.55:
        case = _gated(rows, width, inner, dtype, activation, weights, bias, rng.random() < 0.4, backward, x_pad)
    else:
        if rng.random() < 0.5:  # an output projection
            width, inner, activation = inner, width, "none"
        case = _linear(rows, width, inner, dtype, activation, weights, bias, rng.random() < 0.5, backward, x_pad)
    while work(case)["flops"] > _LARGEST_FLOPS:
        case["rows"] = case["rows"] * 2 // 3
    return case


# ------------------------------------------------------------------------------------ the inputs
def _e4m3_rows(w):
    """Codes and fp32 scales by rows: amax / 448, nearest even."""
    amax = w.abs().amax(dim=-1, keepdim=True)
    scale = torch.where(amax > 0, (amax / 448.0).clamp_min(1e-12), torch.ones_like(amax))
    codes = (w / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), scale.squeeze(-1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE)
    gen.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=_DEVICE, dtype=torch.float32) * std

    dtype = _DTYPES[case["dtype"]]
    rows, width, inner = case["rows"], case["width"], case["inner"]
    features = 2 * inner if case["kind"] == "gated" else inner
    # activations after a norm: unit variance, a few channels several times larger
    gain = 1.0 + 5.0 * (torch.rand(width, generator=gen, device=_DEVICE) < 0.01).float()
    wide = (normal(rows, width + case["x_pad"]) * torch.nn.functional.pad(gain, (0, case["x_pad"]), value=1.0)).to(dtype)
    w, w_scale = normal(features, width, std=width ** -0.5), None
    if case["weights"] == "e4m3":
        w, w_scale = _e4m3_rows(w)
    else:
        w = w.to(dtype)
    state = {"case": case, "x": wide[:, :width], "w": w, "w_scale": w_scale,
             "bias": normal(features, std=0.2).to(dtype) if case["bias"] else None}
    if case["backward"]:
        state["dout"] = normal(rows, inner, std=0.1).to(dtype)
    elif case.get("residual"):
        state["residual"] = normal(rows, inner).to(dtype)
    return state


# ------------------------------------------------------------------------------------ one pass, plain
def _sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _tanh_inner(z):
    return math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)


def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return torch.clamp_min(z, 0.0)
    if name == "gelu":
        return z * (0.5 * torch.erfc(z * -_SQRT_HALF))
    if name == "gelu_tanh":  # 0.5 (1 + tanh u) = sigmoid(2 u)
        return z * _sigmoid(2.0 * _tanh_inner(z))
    if name == "quick_gelu":
        return z * _sigmoid(1.702 * z)
    return z * _sigmoid(z)


def _act_slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.erfc(z * -_SQRT_HALF) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "gelu_tanh":
        s = _sigmoid(2.0 * _tanh_inner(z))
        return s + z * s * (1.0 - s) * (2.0 * math.sqrt(2.0 / math.pi)) * (1.0 + 3.0 * 0.044715 * z * z)
    c = 1.702 if name == "quick_gelu" else 1.0
    s = _sigmoid(c * z)
    return s + c * z * s * (1.0 - s)


def _plain(state):
    case = state["case"]
    x, dtype = state["x"].float(), state["x"].dtype
    if state["w_scale"] is not None:
        w = state["w"].view(torch.float8_e4m3fn).float() * state["w_scale"][:, None]
    else:
        w = state["w"].float()
    act, dz = case["activation"], None
    need_z = not case["backward"] or case["kind"] == "gated" or act != "none"
    if need_z:
        z = x @ w.t()
        if state["bias"] is not None:
            z = z + state["bias"].float()
    if case["kind"] == "gated":
        a, b = z[:, :case["inner"]], z[:, case["inner"]:]
        value, gate = (b, a) if case["gate_first"] else (a, b)
        if not case["backward"]:
            return (value * _act(act, gate)).to(dtype)
        dout = state["dout"].float()
        dvalue, dgate = dout * _act(act, gate), dout * value * _act_slope(act, gate)
        dz = torch.cat((dgate, dvalue) if case["gate_first"] else (dvalue, dgate), dim=1)
    elif not case["backward"]:
        out = _act(act, z)
        if case["residual"]:
            out = out + state["residual"].float()
        return out.to(dtype)
    else:
        dz = state["dout"].float()
        if need_z:
            dz = dz * _act_slope(act, z)
    grads = [(dz @ w).to(dtype), (dz.t() @ x).to(dtype)]
    if case["bias"]:
        grads.append(dz.sum(dim=0).to(dtype))
    return grads


def run(state):
    if not own:
        return _plain(state)
    case, lib = state["case"], _library()
    if case["backward"]:
        if case["kind"] == "gated":
            grads = lib.gated_linear_backward(state["dout"], state["x"], state["w"], bias=state["bias"],
                                              activation=case["activation"], gate_first=case["gate_first"])
        else:
            grads = lib.linear_act_backward(state["dout"], state["x"], state["w"], bias=state["bias"],
                                            activation=case["activation"])
        return [g for g in grads if g is not None]
    if case["kind"] == "gated":
        return lib.gated_linear(state["x"], state["w"], bias=state["bias"], w_scale=state["w_scale"],
                                activation=case["activation"], gate_first=case["gate_first"])
    return lib.linear_act(state["x"], state["w"], bias=state["bias"], w_scale=state["w_scale"],
                          activation=case["activation"], residual=state.get("residual"))


# ------------------------------------------------------------------------------------ its work
def work(case):
    rows, width, inner = case["rows"], case["width"], case["inner"]
    features = 2 * inner if case["kind"] == "gated" else inner
    product = 2.0 * rows * features * width
    w_bytes = features * width * (1 if case["weights"] == "e4m3" else 2) + (4 * features if case["weights"] == "e4m3" else 0)
    traffic = 2 * rows * width + w_bytes + 2 * rows * inner + (2 * features if case["bias"] else 0)
    if not case["backward"]:
        return {"bytes": float(traffic + (2 * rows * inner if case.get("residual") else 0)), "flops": product}
    products = 3 if case["kind"] == "gated" or case["activation"] != "none" else 2
    traffic += 2 * rows * width + 2 * features * width + (2 * features if case["bias"] else 0)
    if products == 2 and case["bias"]:
        traffic -= 2 * features  # the bias itself is not read
    return {"bytes": float(traffic), "flops": products * product}


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definition on 64-bit leaves; the gradients are automatic differentiation's."""
    data = prepare(case, seed)
    w = data["w"]
    if data["w_scale"] is not None:
        w = w.view(torch.float8_e4m3fn).double() * data["w_scale"].double().unsqueeze(1)
    leaves = [data["x"].double(), w.double()] + ([data["bias"].double()] if case["bias"] else [])
    for leaf in leaves:
        leaf.requires_grad_(case["backward"])
    z = torch.nn.functional.linear(leaves[0], leaves[1], leaves[2] if case["bias"] else None)
    first = z
    if case["kind"] == "gated":
        first, second = torch.split(z, case["inner"], dim=1)
        gate, value = (first, second) if case["gate_first"] else (second, first)
        first = gate
    name = case["activation"]
    if name == "gelu":
        out = first * torch.special.ndtr(first)
    elif name == "gelu_tanh":
        out = 0.5 * first * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (first + 0.044715 * first ** 3)))
    elif name == "silu":
        out = first * torch.sigmoid(first)
    elif name == "quick_gelu":
        out = first * torch.sigmoid(1.702 * first)
    elif name == "relu":
        out = torch.relu(first)
    else:
        out = first
    if case["kind"] == "gated":
        out = value * out
    elif case["residual"] and not case["backward"]:
        out = out + data["residual"].double()
    if not case["backward"]:
        return out
    return list(torch.autograd.grad(out, leaves, data["dout"].double()))
