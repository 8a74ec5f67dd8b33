"""Group norm and 8-bit integer linears on one MI355X: plain forms, calls and 64-bit values.

``group_norm``: act((x - mean) rstd gamma + beta), channels last, forward and backward. ``linear_i8`` and
``gated_i8``: products of 8-bit integers with a scale for each token and output channel, bias, activation and
residual (or value * act(gate)) in 16 bits. Their tokens come as 8-bit codes, as 16-bit rows that are
quantised by row, or out of a LayerNorm or a group norm as they do at the ends and in the blocks of a
spatial transformer. The listed cases are points of the ranges that ``draw`` samples.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_DEVICE = "cuda:0"
_SQRT_HALF = 0.7071067811865476


def _library():
    package = os.path.join(os.getcwd(), "sdxl-end2end_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import sdxl_hip
    return sdxl_hip


# ------------------------------------------------------------------------------------ the cases
def _norm(batch, pixels, channels, groups=32, dtype="f16", activation="silu", eps=1e-5, stats=False, backward=False,
          x_pad=0):
    return {"kind": "group_norm", "batch": batch, "pixels": pixels, "channels": channels, "groups": groups,
            "dtype": dtype, "activation": activation, "eps": eps, "stats": stats, "backward": backward, "x_pad": x_pad}


def _i8(kind, rows, width, inner, dtype="f16", activation="none", source="tokens", bias=True, residual=False,
        gate_first=False, x_pad=0):
    # source: codes (x is quantised), tokens (x is in 16 bits), layer_norm or group_norm (x goes through it)
    return {"kind": kind, "rows": rows, "width": width, "inner": inner, "dtype": dtype, "activation": activation,
            "source": source, "bias": bias, "residual": residual, "gate_first": gate_first, "x_pad": x_pad}


def listed():
    cases = {
        # The middle residual block of a 512 x 512 image with guidance: the smallest norm, all latency.
        "norm_mid_small": _norm(2, 256, 1280),
        # An upward residual block of level 1: the hidden state and its skip side by side, 640 + 320 channels.
        "norm_up_l1": _norm(2, 4096, 960),
        # The decoder's third stage, 512 x 512 pixels in its own fp32; the statistics are kept for training it.
        "norm_decoder_f32": _norm(1, 262144, 256, dtype="f32", stats=True),
        # Training the transformer's own norm at level 2 (eps 1e-6, no activation).
        "norm_backward_l2": _norm(2, 1024, 1280, activation="none", eps=1e-6, backward=True),
        # Training a level-0 residual block on a non-square latent, 95 x 121 pixels, in bf16.
        "norm_backward_ragged": _norm(3, 11495, 320, dtype="bf16", backward=True),
        # Training the decoder at half resolution, bf16: the largest norm.
        "norm_backward_large": _norm(2, 131072, 256, dtype="bf16", backward=True),
        # One token through a gated projection: serving, the weights' transfer is all there is.
        "gated_i8_one_row": _i8("gated_i8", 1, 1280, 5120, dtype="bf16", activation="silu", bias=False, gate_first=True),
        # The level-2 block's norm3 and gated projection, a 1024 x 1024 image with guidance.
        "gated_i8_l2": _i8("gated_i8", 2048, 1280, 5120, activation="gelu", source="layer_norm"),
        # The text encoder's MLP, 2 x 77 tokens.
        "linear_i8_text": _i8("linear_i8", 154, 1280, 5120, activation="gelu"),
        # A level-1 transformer's entry on a non-square image, 76 x 65 tokens: group norm, then proj_in.
        "linear_i8_proj_in": _i8("linear_i8", 4940, 640, 640, source="group_norm"),
        # The level-2 block's output projection over a batch of four, bf16, with bias and residual.
        "linear_i8_out": _i8("linear_i8", 8192, 5120, 1280, dtype="bf16", source="codes", residual=True),
        # A long batch through a wide gated projection: the largest product.
        "gated_i8_wide": _i8("gated_i8", 8192, 2048, 5456, dtype="bf16", activation="silu", bias=False, gate_first=True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


_LARGEST_ELEMENTS = 2 * 131072 * 256
_LARGEST_FLOPS = 4.0 * 8192 * 2048 * 5456


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_norm(rng):
    backward = rng.random() < 0.5
    groups = rng.choice((32, 32, 32, 16, 8, 1))
    channels = rng.choice((128, 256, 320, 512, 640, 960, 1280, 1920, 2560, groups * rng.randint(1, max(1, 640 // groups))))
    while channels % groups != 0:
        groups //= 2
    pixels = _log_int(rng, 1, 131072)
    batch = rng.choice((1, 1, 2, 2, 3, 4, 8))
    while batch * pixels * channels > _LARGEST_ELEMENTS:
        pixels = pixels * 2 // 3
    dtype = rng.choice(("f16", "f16", "bf16", "bf16", "f32"))
    if dtype == "f32":
        pixels = (pixels + 1) // 2
    if pixels * (channels // groups) < 32:  # a variance of a few values says little
        pixels = 32
    activation = rng.choice(("silu", "silu", "silu", "none", "none", "gelu", "quick_gelu", "gelu_tanh",
                             "silu" if backward else "relu"))
    return _norm(batch, pixels, channels, groups, dtype, activation, rng.choice((1e-5, 1e-6)),
                 not backward and rng.random() < 0.3, backward, rng.choice((0, 0, 0, 8, 64, 3)))


def _draw_i8(rng):
    kind = rng.choice(("linear_i8", "gated_i8"))
    rows = _log_int(rng, 1, 16384)
    width = rng.choice((320, 640, 1280, 2048, 16 * _log_int(rng, 8, 128)))
    inner = rng.choice((4 * width, width, 16 * _log_int(rng, 8, 340)))
    source = rng.choice(("codes", "tokens", "tokens", "layer_norm", "group_norm"))
    if rng.random() < 0.15 and source != "group_norm":  # rows that no 16-byte load divides
        width += rng.randint(1, 15)
    if rng.random() < 0.2:
        inner += rng.randint(1, 7)
    if source == "group_norm":
        width = 32 * max(1, width // 32)
        rows = max(rows, 8)
    if kind == "linear_i8" and source in ("codes", "tokens") and rng.random() < 0.5:  # an output projection
        width, inner = inner, width
    case = _i8(kind, rows, width, inner, rng.choice(("f16", "bf16")),
               rng.choice(("gelu", "silu", "gelu_tanh", "none" if kind == "linear_i8" else "gelu")), source,
               rng.random() < 0.7, kind == "linear_i8" and rng.random() < 0.5,
               kind == "gated_i8" and rng.random() < 0.4, rng.choice((0, 0, 0, 64, 16, 8)))
    while work(case)["flops"] > _LARGEST_FLOPS:
        case["rows"] = case["rows"] * 2 // 3
    return case


def draw(rng):
    return _draw_norm(rng) if rng.random() < 0.45 else _draw_i8(rng)


# ------------------------------------------------------------------------------------ the inputs
def _activations(normal, uniform, rows, channels, pad):
    """Hidden states as a norm meets them: channels with means of their own, a few of them several times larger."""
    gain = 1.0 + 5.0 * (uniform(channels) < 0.02).float()
    x = normal(rows, channels + pad)
    x[:, :channels] = (x[:, :channels] + normal(channels, std=0.7)) * gain
    return x


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE)
    gen.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=_DEVICE, dtype=torch.float32) * std

    def uniform(n):
        return torch.rand(n, generator=gen, device=_DEVICE)

    dtype = _DTYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "group_norm":
        batch, pixels, channels, groups = case["batch"], case["pixels"], case["channels"], case["groups"]
        x = _activations(normal, uniform, batch * pixels, channels, case["x_pad"]).to(dtype)
        state["x"] = x.view(batch, pixels, channels + case["x_pad"])[:, :, :channels]
        state["gamma"] = (1.0 + normal(channels, std=0.2)).to(dtype)
        state["beta"] = normal(channels, std=0.2).to(dtype)
        if case["backward"]:
            state["dout"] = normal(batch, pixels, channels, std=0.1).to(dtype)
            # mean and reciprocal deviation as the forward call left them
            first, second = [], []
            for image in state["x"]:
                v = image.double().reshape(pixels, groups, channels // groups)
                mean = v.mean(dim=(0, 2))
                first.append(mean)
                second.append(((v - mean.view(1, groups, 1)).square().mean(dim=(0, 2)) + case["eps"]).rsqrt())
            state["stats"] = torch.stack((torch.stack(first), torch.stack(second)), dim=2).float().contiguous()
        return state
    rows, width, inner = case["rows"], case["width"], case["inner"]
    features = 2 * inner if case["kind"] == "gated_i8" else inner
    pad = case["x_pad"]
    w = normal(features, width, std=width ** -0.5)
    state["w_scale"] = w.abs().amax(dim=1) / 127.0
    state["w"] = torch.round(w / state["w_scale"][:, None]).clamp(-127, 127).to(torch.int8)
    state["bias"] = normal(features, std=0.2).to(dtype) if case["bias"] else None
    state["residual"] = normal(rows, inner).to(dtype) if case["residual"] else None
    x = _activations(normal, uniform, rows, width, pad)
    if case["source"] == "codes":
        state["x_scale"] = (x[:, :width].abs().amax(dim=1) / 127.0).contiguous()
        state["x"] = torch.round(x / state["x_scale"][:, None]).clamp(-127, 127).to(torch.int8)[:, :width]
    else:
        state["x"] = x.to(dtype)[:, :width]
    if case["source"] in ("layer_norm", "group_norm"):
        state["gamma"] = (1.0 + normal(width, std=0.2)).to(dtype)
        state["beta"] = normal(width, std=0.2).to(dtype)
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


def _plain_norm(state):
    case, x, dtype = state["case"], state["x"].float(), state["x"].dtype
    batch, pixels, channels = x.shape
    groups = case["groups"]
    x = x.reshape(batch, pixels, groups, channels // groups)
    gamma, beta = (state[n].float().view(1, 1, groups, channels // groups) for n in ("gamma", "beta"))
    if case["backward"]:
        mean, rstd = (state["stats"][:, :, i].view(batch, 1, groups, 1) for i in (0, 1))
    else:
        mean = x.mean(dim=(1, 3), keepdim=True)
        rstd = torch.rsqrt((x - mean).square().mean(dim=(1, 3), keepdim=True) + case["eps"])
    normed = (x - mean) * rstd
    z = normed * gamma + beta
    if not case["backward"]:
        out = _act(case["activation"], z).reshape(batch, pixels, channels).to(dtype)
        if not case["stats"]:
            return out
        return [out, torch.stack((mean.view(batch, groups), rstd.view(batch, groups)), dim=2)]
    dz = state["dout"].float().view_as(x) * _act_slope(case["activation"], z)
    dbeta, dgamma = dz.sum(dim=(0, 1)), (dz * normed).sum(dim=(0, 1))
    dz = dz * gamma
    over = 1.0 / (pixels * (channels // groups))
    first = dz.sum(dim=(1, 3), keepdim=True) * over
    second = (dz * normed).sum(dim=(1, 3), keepdim=True) * over
    dx = rstd * (dz - first - normed * second)
    return [dx.reshape(batch, pixels, channels).to(dtype), dgamma.reshape(channels).to(dtype),
            dbeta.reshape(channels).to(dtype)]


_TRANSFORMER_EPS = {"layer_norm": 1e-5, "group_norm": 1e-6}


def _codes(x):
    """Rows of whole numbers up to 127 and what one of them stands for."""
    amax = x.abs().amax(dim=-1, keepdim=True)
    scale = torch.where(amax > 0, (amax / 127.0).clamp_min(1e-12), torch.ones_like(amax))
    return torch.round(x / scale).clamp(-127.0, 127.0), scale


def _plain_i8(state):
    case, x = state["case"], state["x"].float()
    dtype = _DTYPES[case["dtype"]]
    if case["source"] == "codes":
        scale = state["x_scale"][:, None]
    else:
        if case["source"] != "tokens":
            rows, width = x.shape
            # one image of all rows; a row alone, or the rows of 32 channel groups
            v = x.view(rows, 1, width) if case["source"] == "layer_norm" else x.view(rows, 32, width // 32)
            dims = 2 if case["source"] == "layer_norm" else (0, 2)
            v = v - v.mean(dim=dims, keepdim=True)
            v = v * torch.rsqrt(v.square().mean(dim=dims, keepdim=True) + _TRANSFORMER_EPS[case["source"]])
            x = v.reshape(rows, width) * state["gamma"].float() + state["beta"].float()
        x, scale = _codes(x)
    z = (x @ state["w"].float().t()) * scale * state["w_scale"]
    if state["bias"] is not None:
        z = z + state["bias"].float()
    if case["kind"] == "gated_i8":
        a, b = z[:, :case["inner"]], z[:, case["inner"]:]
        value, gate = (b, a) if case["gate_first"] else (a, b)
        return (value * _act(case["activation"], gate)).to(dtype)
    out = _act(case["activation"], z)
    if state["residual"] is not None:
        out = out + state["residual"].float()
    return out.to(dtype)


def run(state):
    case = state["case"]
    if not own:
        return _plain_norm(state) if case["kind"] == "group_norm" else _plain_i8(state)
    lib = _library()
    if case["kind"] == "group_norm":
        if case["backward"]:
            return list(lib.group_norm_backward(state["dout"], state["x"], state["gamma"], state["beta"], case["groups"],
                                                state["stats"], activation=case["activation"]))
        out = lib.group_norm(state["x"], state["gamma"], state["beta"], case["groups"], activation=case["activation"],
                             eps=case["eps"], with_stats=case["stats"])
        return list(out) if case["stats"] else out
    x, x_scale, source = state["x"], state.get("x_scale"), case["source"]
    if source == "layer_norm":
        x, x_scale = lib.layer_norm_i8(x, state["gamma"], state["beta"], eps=_TRANSFORMER_EPS[source])
    elif source == "group_norm":
        x, x_scale = lib.group_norm_i8(x.unsqueeze(0), state["gamma"], state["beta"], 32, eps=_TRANSFORMER_EPS[source])
        x = x.squeeze(0)
    if case["kind"] == "gated_i8":
        return lib.gated_linear_i8(x, state["w"], state["w_scale"], x_scale=x_scale, bias=state["bias"],
                                   activation=case["activation"], gate_first=case["gate_first"],
                                   dtype=_DTYPES[case["dtype"]])
    return lib.linear_i8(x, state["w"], state["w_scale"], x_scale=x_scale, bias=state["bias"],
                         residual=state["residual"], activation=case["activation"], dtype=_DTYPES[case["dtype"]])


# ------------------------------------------------------------------------------------ its work
def work(case):
    elem = _BYTES[case["dtype"]]
    if case["kind"] == "group_norm":
        elements = float(case["batch"] * case["pixels"] * case["channels"])
        stats = 8 * case["batch"] * case["groups"]
        if case["backward"]:  # x and dout in, dx out; dz, two sums and their two by the group, dx
            return {"bytes": elem * (3 * elements + 4 * case["channels"]) + stats, "flops": 20 * elements}
        return {"bytes": elem * (2 * elements + 2 * case["channels"]) + (stats if case["stats"] else 0),
                "flops": 12 * elements}
    rows, width, inner = case["rows"], case["width"], case["inner"]
    features = 2 * inner if case["kind"] == "gated_i8" else inner
    traffic = features * width + 4 * features + elem * rows * inner
    traffic += rows * width + 4 * rows if case["source"] == "codes" else elem * rows * width
    traffic += 2 * elem * width if case["source"] in ("layer_norm", "group_norm") else 0
    traffic += elem * features if case["bias"] else 0
    traffic += elem * rows * inner if case["residual"] else 0
    return {"bytes": float(traffic), "flops": 2.0 * rows * features * width}


# ------------------------------------------------------------------------------------ in 64 bits
def _exact_act(name, z):
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "quick_gelu":
        return z * torch.sigmoid(1.702 * z)
    return torch.relu(z) if name == "relu" else z


def _exact_norm(case, data):
    """Image by image, channels first; the gradients are automatic differentiation's."""
    outs, stats, grads = [], [], [[], 0.0, 0.0]
    for i in range(case["batch"]):
        x = data["x"][i].double().t().contiguous().requires_grad_(case["backward"])  # [channels, pixels]
        gamma, beta = (data[n].double().requires_grad_(case["backward"]) for n in ("gamma", "beta"))
        rows = x.reshape(case["groups"], -1)
        var, mean = torch.var_mean(rows, dim=1, unbiased=False, keepdim=True)
        root = torch.sqrt(var + case["eps"])
        z = ((rows - mean) / root).reshape(x.shape)
        out = _exact_act(case["activation"], torch.addcmul(beta[:, None], z, gamma[:, None])).t()
        if case["backward"]:
            got = torch.autograd.grad(out, (x, gamma, beta), data["dout"][i].double())
            grads[0].append(got[0].t().contiguous())
            grads[1], grads[2] = grads[1] + got[1], grads[2] + got[2]
        else:
            outs.append(out.contiguous())
            stats.append(torch.cat((mean, 1.0 / root), dim=1))
    if case["backward"]:
        return [torch.stack(grads[0]), grads[1], grads[2]]
    return [torch.stack(outs), torch.stack(stats)] if case["stats"] else torch.stack(outs)


def exact(case, seed):
    data = prepare(case, seed)
    if case["kind"] == "group_norm":
        return _exact_norm(case, data)
    x = data["x"].double()
    if case["source"] == "layer_norm":
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        x = torch.addcmul(data["beta"].double(), (x - mean) / torch.sqrt(var + _TRANSFORMER_EPS["layer_norm"]),
                          data["gamma"].double())
    elif case["source"] == "group_norm":
        by_group = x.t().reshape(32, -1)
        var, mean = torch.var_mean(by_group, dim=1, unbiased=False, keepdim=True)
        by_group = (by_group - mean) / torch.sqrt(var + _TRANSFORMER_EPS["group_norm"])
        x = torch.addcmul(data["beta"].double(), by_group.reshape(x.shape[1], -1).t(), data["gamma"].double())
    if case["source"] == "codes":
        x = x * data["x_scale"].double().unsqueeze(1)
    else:
        top = torch.linalg.vector_norm(x, ord=float("inf"), dim=1, keepdim=True)
        step = torch.where(top == 0, torch.ones_like(top), torch.maximum(top / 127, torch.full_like(top, 1e-12)))
        x = step * torch.round(x / step)
    w = data["w"].double() * data["w_scale"].double().unsqueeze(1)
    z = torch.nn.functional.linear(x, w, data["bias"].double() if case["bias"] else None)
    if case["kind"] == "gated_i8":
        first, second = torch.split(z, case["inner"], dim=1)
        gate, value = (first, second) if case["gate_first"] else (second, first)
        return value * _exact_act(case["activation"], gate)
    out = _exact_act(case["activation"], z)
    return out + data["residual"].double() if case["residual"] else out
