"""Workloads of the transformer-block operators: layer norm, and the matrix product with bias, activation and residual.

The cases are what a transformer meets in quantization-aware training and in inference through the simulation: single
tokens, prompts, training batches, in float32 and bfloat16, with ragged batches and odd feature counts.

`run` with own = False computes each operator from elementary torch operations in float32, rounded once at the end;
with own = True it makes the calls a user of aimet_amd.v2.nn.fused makes.  `exact` is the definition in float64.
"""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _norm(name, rows, width, dtype, direction):
    return {"name": name, "op": "layer_norm", "rows": rows, "width": width, "dtype": dtype, "direction": direction}


def _linear(name, rows, features, out, dtype, direction, activation, residual):
    return {"name": name, "op": "linear", "rows": rows, "in": features, "out": out, "dtype": dtype,
            "direction": direction, "activation": activation, "residual": residual}


def listed():
    return [
        # the norm before a block while one token at a time is generated: latency
        _norm("norm 1x4096 bf16", 1, 4096, "bf16", "forward"),
        # a training step of a small encoder, one norm of it
        _norm("norm 2048x1024 f32 train", 2048, 1024, "f32", "training"),
        # odd width and a ragged batch: no row starts on a vector boundary
        _norm("norm 1003x1001 f32 train", 1003, 1001, "f32", "training"),
        # a training step of a wide decoder over long sequences
        _norm("norm 16384x4096 bf16 train", 16384, 4096, "bf16", "training"),
        # a long prompt through a very wide norm
        _norm("norm 8192x8192 bf16", 8192, 8192, "bf16", "forward"),
        # up projection of one token: the weight is read once, nothing else counts
        _linear("linear 1x4096>11008 bf16", 1, 4096, 11008, "bf16", "forward", "silu", False),
        # down projection of a few concurrent requests, float32 simulation
        _linear("linear 16x4096>4096 f32", 16, 4096, 4096, "f32", "forward", "none", True),
        # down projection of a prompt
        _linear("linear 2048x11008>4096 bf16", 2048, 11008, 4096, "bf16", "forward", "none", True),
        # a training step of an encoder's up projection in float32, as quantization-aware training runs it
        _linear("linear 2048x1024>4096 f32 train", 2048, 1024, 4096, "f32", "training", "gelu", False),
        # odd sizes in every direction, with the fine-tuned head's ReLU and a skip connection
        _linear("linear 1021x1003>1531 bf16 train", 1021, 1003, 1531, "bf16", "training", "relu", True),
        # a wide square layer in float32
        _linear("linear 4096x4096>4096 f32 train", 4096, 4096, 4096, "f32", "training", "silu", True),
        # a training step of a decoder's up projection
        _linear("linear 4096x4096>11008 bf16 train", 4096, 4096, 11008, "bf16", "training", "gelu", False),
    ]


def _size(rng, low, high):
    """Spread over the logarithm; half of the sizes are multiples of 64, a quarter of 8, a quarter whatever comes."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    step = rng.choice((64, 64, 8, 1))
    return min(high, max(low, n // step * step))


def draw(rng):
    dtype = rng.choice(("f32", "bf16"))
    direction = rng.choice(("forward", "training"))
    if rng.random() < 0.4:
        while True:
            rows, width = _size(rng, 1, 32768), _size(rng, 64, 16384)
            if rows * width <= 16384 * 4096:
                return {"op": "layer_norm", "rows": rows, "width": width, "dtype": dtype, "direction": direction}
    # float32 training takes the smooth activations: at the kink of a ReLU the gradient is decided by the last bit
    smooth = ("none", "gelu", "gelu_tanh", "silu")
    activation = rng.choice(smooth if dtype == "f32" and direction == "training" else smooth + ("relu",))
    residual = rng.random() < 0.5
    while True:
        rows, features, out = _size(rng, 1, 8192), _size(rng, 64, 12288), _size(rng, 64, 12288)
        most = 4096 * 4096 * (4096 if dtype == "f32" else 11008)
        if rows * features * out <= most:
            return {"op": "linear", "rows": rows, "in": features, "out": out, "dtype": dtype, "direction": direction,
                    "activation": activation, "residual": residual}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _DTYPE[case["dtype"]]
    training = case["direction"] == "training"

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def leaf(t):
        return t.to(dtype).requires_grad_(training)

    rows = case["rows"]
    if case["op"] == "layer_norm":
        width = case["width"]
        # activations of a residual stream: a mean per feature, and a few features far larger than the others
        scale = 1.0 + 20.0 * (torch.rand(width, generator=g, device="cuda") < 0.005).float()
        x = normal(rows, width) * scale + 0.3 * normal(width)
        state = {"x": leaf(x), "weight": leaf(1.0 + 0.2 * normal(width)), "bias": leaf(0.1 * normal(width)),
                 "eps": 1e-5}
        if training:
            state["grad"] = normal(rows, width).to(dtype)
    else:
        features, out = case["in"], case["out"]
        state = {"x": leaf(normal(rows, features)), "weight": leaf(normal(out, features) / math.sqrt(features)),
                 "bias": leaf(0.3 * normal(out)),
                 "residual": leaf(normal(rows, out)) if case["residual"] else None,
                 "activation": case["activation"]}
        if training:
            state["grad"] = normal(rows, out).to(dtype)
    state["op"], state["training"] = case["op"], training
    return state


# ----------------------------------------------------------------------------------------------- the plain forms
def _plain_layer_norm(s):
    dtype = s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + s["eps"])
    xhat = centred * rstd
    y = (xhat * w + b).to(dtype)
    if not s["training"]:
        return {"y": y}
    g = s["grad"].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(dtype), "dweight": (g * xhat).sum(0).to(dtype), "dbias": g.sum(0).to(dtype)}


def _plain_activation(z, kind):
    """(value, derivative) at z."""
    if kind == "none":
        return z, None
    if kind == "relu":
        return z.clamp(min=0.0), (z > 0).float()
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if kind == "gelu":
        cdf = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    value, slope = _plain_activation(x @ w.t() + s["bias"].float(), s["activation"])
    y = (value if s["residual"] is None else value + s["residual"].float()).to(dtype)
    if not s["training"]:
        return {"y": y}
    g = s["grad"].float()
    dz = g if slope is None else g * slope
    out = {"y": y, "dx": (dz @ w).to(dtype), "dweight": (dz.t() @ x).to(dtype), "dbias": dz.sum(0).to(dtype)}
    if s["residual"] is not None:
        out["dresidual"] = s["grad"]
    return out


# ------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from aimet_amd.v2.nn import fused
    if s["op"] == "layer_norm":
        leaves = {"dx": s["x"], "dweight": s["weight"], "dbias": s["bias"]}
        y = fused.layer_norm(s["x"], (s["x"].shape[1],), s["weight"], s["bias"], s["eps"])
    else:
        leaves = {"dx": s["x"], "dweight": s["weight"], "dbias": s["bias"]}
        if s["residual"] is not None:
            leaves["dresidual"] = s["residual"]
        y = fused.linear(s["x"], s["weight"], s["bias"], s["activation"], s["residual"])
    if not s["training"]:
        return {"y": y}
    grads = torch.autograd.grad(y, list(leaves.values()), s["grad"])
    return {"y": y, **dict(zip(leaves, grads))}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_layer_norm(state) if state["op"] == "layer_norm" else _plain_linear(state)


def work(case):
    size = _DTYPE[case["dtype"]].itemsize
    training = case["direction"] == "training"
    if case["op"] == "layer_norm":
        n, width = case["rows"] * case["width"], case["width"]
        # forward: x, weight, bias -> y; training adds grad -> dx, dweight, dbias
        return {"bytes": size * (4 * n + 4 * width if training else 2 * n + 2 * width),
                "flops": (18 if training else 7) * n}
    rows, features, out = case["rows"], case["in"], case["out"]
    bytes_ = rows * features + out * features + out + rows * out * (2 if case["residual"] else 1)
    if training:
        bytes_ += rows * out + rows * features + out * features + out
    return {"bytes": size * bytes_, "flops": 2 * rows * features * out * (3 if training else 1)}


def exact(case, seed):
    """The operators' definitions in float64, gradients by differentiating them."""
    state = prepare(case, seed)
    names = [n for n in ("x", "weight", "bias", "residual") if state.get(n) is not None]
    v = {n: state[n].detach().double().requires_grad_(state["training"]) for n in names}
    if case["op"] == "layer_norm":
        y = torch.nn.functional.layer_norm(v["x"], (case["width"],), v["weight"], v["bias"], state["eps"])
    else:
        z = torch.nn.functional.linear(v["x"], v["weight"], v["bias"])
        y = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu,
             "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["activation"]](z)
        if "residual" in v:
            y = y + v["residual"]
    out = {"y": y.detach()}
    if state["training"]:
        grads = torch.autograd.grad(y, [v[n] for n in names], state["grad"].double())
        out.update({"d" + n: d for n, d in zip(names, grads)})
    return out
