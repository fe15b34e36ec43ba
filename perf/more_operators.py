"""The dense feed-forward operators, as cases that can be timed and compared.

Where `own` is false, `run` computes each operator from elementary torch operations in 32 bits (in 64 where values are
rounded to 8 bits, which borders decide); where it is true, it makes the calls that a user makes of this package. A case is one
pass through one of three operators:

  norm    root mean square norm of each row, after the residual's addition where there is one; the result in the inputs' type,
          or in 8 bits with a power of two for each 32 values (returned as the values that these stand for)
  linear  a @ w.T with bias, activation and residual added as it is written; matrices of 16 bits, or of 8 bits with such powers
          (then activations are quantised in the call)
  gated   activation(a @ gate.T) * (a @ up.T)

With `train` set the pass also computes the gradients, from one of the results. Sizes are those of this repository's configurations
(8192^3, 8192 x 8191 x 1000) or generic ones.
"""
import math

import torch

own = False

_FLOATS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-6


def listed():
    return [
        # A decoding batch's residual streams, normed and quantised for 8-bit products: the smallest call, where latency is all.
        {"name": "norm_tokens", "op": "norm", "dtype": "bf16", "m": 16, "k": 4096, "residual": True, "out": "mx8", "train": False},
        # The same of a long prompt.
        {"name": "norm_prompt", "op": "norm", "dtype": "bf16", "m": 16384, "k": 8192, "residual": True, "out": "mx8", "train": False},
        # A training step's norm with its gradients.
        {"name": "norm_train", "op": "norm", "dtype": "bf16", "m": 8192, "k": 4096, "residual": True, "out": "same", "train": True},
        # One token through a layer's last product: the stream of the matrix.
        {"name": "linear_token", "op": "linear", "dtype": "bf16", "out": "bf16", "m": 1, "n": 8192, "k": 8192, "bias": False,
         "activation": "none", "residual": True, "train": False},
        # A server's batch of single tokens against an 8-bit matrix.
        {"name": "linear_batch", "op": "linear", "dtype": "mx8", "out": "bf16", "m": 64, "n": 8192, "k": 8192, "bias": True,
         "activation": "silu", "residual": False, "train": False},
        # The ragged configuration: nothing but the rows is a multiple of a tile.
        {"name": "linear_ragged", "op": "linear", "dtype": "f16", "out": "f32", "m": 8192, "n": 8191, "k": 1000, "bias": True,
         "activation": "relu", "residual": False, "train": False},
        # The size of the headline metric: a long prompt against a wide layer, in 8 bits.
        {"name": "linear_square", "op": "linear", "dtype": "mx8", "out": "bf16", "m": 8192, "n": 8192, "k": 8192, "bias": False,
         "activation": "none", "residual": True, "train": False},
        # A training step of a layer with bias and activation.
        {"name": "linear_train", "op": "linear", "dtype": "bf16", "out": "bf16", "m": 8192, "n": 4096, "k": 4096, "bias": True,
         "activation": "gelu", "residual": True, "train": True},
        # Four tokens through the first half of a gated block.
        {"name": "gated_tokens", "op": "gated", "dtype": "bf16", "out": "bf16", "m": 4, "n": 8192, "k": 4096, "activation": "silu",
         "train": False},
        # A middling prompt, odd sizes, 8-bit matrices.
        {"name": "gated_odd", "op": "gated", "dtype": "mx8", "out": "f16", "m": 1001, "n": 2050, "k": 1000, "activation": "gelu_tanh",
         "train": False},
        # A long prompt through the first half of a gated block.
        {"name": "gated_prompt", "op": "gated", "dtype": "bf16", "out": "bf16", "m": 8192, "n": 8192, "k": 4096, "activation": "silu",
         "train": False},
        # A training step of it.
        {"name": "gated_train", "op": "gated", "dtype": "bf16", "out": "bf16", "m": 4096, "n": 8192, "k": 2048, "activation": "silu",
         "train": True},
    ]


def _cost(case):
    """A rough time in seconds of the plain form, for keeping drawn cases within the largest listed one."""
    needed = work(case)
    return needed["flops"] / 1e14 + needed["bytes"] / 1e12


def draw(rng):
    """One more case of the same passes, sizes over the whole range of each, two thirds of them multiples of nothing."""
    def size(low, high):
        value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        if rng.random() < 0.35:
            step = 128 if value >= 512 else (32 if value >= 64 else 1)
            value = value // step * step
        return max(low, min(high, value))

    op = rng.choice(["norm", "norm", "linear", "linear", "linear", "gated", "gated", "gated"])
    train = rng.random() < 0.35
    if op == "norm":
        case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "m": size(1, 16384), "k": size(64, 16384),
                "residual": rng.random() < 0.7, "out": "same" if train else rng.choice(["same", "mx8"]), "train": train}
    else:
        dtype = rng.choice(["bf16", "f16"] if train else ["bf16", "f16", "mx8"])
        # (8-bit products give 16-bit results; a training step's results are in its own type)
        out = dtype if train else rng.choice(["bf16", "f16"] if dtype == "mx8" else ["bf16", "f16", "f32"])
        case = {"op": op, "dtype": dtype, "out": out, "m": size(1, 8192), "n": size(256, 8192), "k": size(64, 8192)}
        if op == "linear":
            case |= {"bias": rng.random() < 0.5, "activation": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                     "residual": rng.random() < 0.5}
        else:
            case |= {"activation": rng.choice(["relu", "silu", "gelu", "gelu_tanh"])}
        case["train"] = train
    limit = max(_cost(one) for one in listed())
    while _cost(case) > limit:
        side = max((s for s in ("m", "n", "k") if s in case), key=lambda s: case[s])
        case[side] = case[side] * 3 // 4
    return case


# ---- the inputs ----------------------------------------------------------------------------------------------------

def _normal(shape, generator):
    return torch.randn(shape, device="cuda:0", generator=generator)


def _activations(rows, k, generator):
    """Normal values, 32 bits; one channel of 64 is eight times as large, as the channels of hidden states are; rows differ in size."""
    x = _normal((rows, k), generator)
    x *= 1.0 + 7.0 * (torch.rand((k,), device="cuda:0", generator=generator) < 1 / 64)
    x *= torch.exp(0.5 * _normal((rows, 1), generator))
    return x


def _weights(n, k, dtype, generator):
    """A layer's matrix: of 16 bits, or as an 8-bit checkpoint holds it, e4m3 codes and a scale's exponent for each 32 columns."""
    w = _normal((n, k), generator) / math.sqrt(k)
    if dtype != "mx8":
        return w.to(_FLOATS[dtype])
    exponents, values = _quantized(w)
    return {"codes": values.flatten(1)[:, :k].to(torch.float8_e4m3fn), "scales": (exponents + 127).to(torch.uint8)}


def _kept(matrix, k):
    """A matrix as a program keeps it for its calls."""
    if own and isinstance(matrix, dict):
        import numkong_amd as nk

        return nk.Mx8Matrix(matrix["codes"], matrix["scales"])
    return matrix


def prepare(case, seed):
    generator = torch.Generator(device="cuda:0").manual_seed(seed)
    state, m, k = dict(case), case["m"], case["k"]
    if case["op"] == "norm":
        kind = _FLOATS[case["dtype"]]
        state["x"] = _activations(m, k, generator).to(kind)
        state["residual"] = _activations(m, k, generator).to(kind) if case["residual"] else None
        state["weight"] = (1 + 0.2 * _normal((k,), generator)).to(kind)
        if case["train"]:
            state["grad"] = _normal((m, k), generator).to(kind)
            state["grad_total"] = _normal((m, k), generator).to(kind) if case["residual"] else None
        return state
    n, kind = case["n"], torch.bfloat16 if case["dtype"] == "mx8" else _FLOATS[case["dtype"]]
    state["a"] = _activations(m, k, generator).to(kind)
    if case["op"] == "linear":
        state["w"] = _kept(_weights(n, k, case["dtype"], generator), k)
        state["bias"] = (0.1 * _normal((n,), generator)).to(kind) if case["bias"] else None
        state["residual"] = _normal((m, n), generator).to(_FLOATS[case["out"]]) if case["residual"] else None
    else:
        state["gate"] = _kept(_weights(n, k, case["dtype"], generator), k)
        state["up"] = _kept(_weights(n, k, case["dtype"], generator), k)
    if case["train"]:
        state["grad"] = _normal((m, n), generator).to(_FLOATS[case["out"]])
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _quantized(x):
    """Exponents (rows, blocks) and the values in units of the scale (rows, blocks, 32), in x's type; the last block of a row is filled
    with zeros. The scale is the smallest power of two that keeps a block's largest magnitude within e4m3's 448."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).reshape(x.shape[0], -1, 32)
    largest = x.abs().amax(2)
    mantissa, exponent = torch.frexp(largest)
    exponents = (exponent - 9 + (mantissa > 0.875)).clamp(min=-127)
    exponents = torch.where(largest == 0, -127, exponents)
    scaled = torch.ldexp(x, -exponents[..., None])
    step = torch.ldexp(torch.ones_like(scaled), (torch.frexp(scaled).exponent - 1).clamp(min=-6) - 3)
    return exponents, torch.round(scaled / step) * step


def _rounded(x):
    """x as its quantised values, in x's type."""
    exponents, values = _quantized(x)
    return torch.ldexp(values, exponents[..., None]).flatten(1)[:, :x.shape[1]]


def _matrix(w):
    """A layer's matrix in 32 bits."""
    if not isinstance(w, dict):
        return w.float()
    powers = torch.ldexp(torch.ones_like(w["scales"], dtype=torch.float32), w["scales"].int() - 127)
    return w["codes"].float() * powers.repeat_interleave(32, 1)[:, :w["codes"].shape[1]]


def _activated(x, kind):
    if kind == "relu":
        return torch.where(x > 0, x, 0.0)
    if kind == "silu":
        return x / (1 + torch.exp(-x))
    if kind == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _slope(x, kind):
    """The activation's derivative."""
    if kind == "relu":
        return (x > 0).to(x.dtype)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-x))
        return s * (1 + x * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x)
    return torch.ones_like(x)


def _norm_plain(state):
    kind = state["x"].dtype
    total = state["x"] if state["residual"] is None else (state["x"].float() + state["residual"].float()).to(kind)
    s, w = total.float(), state["weight"].float()
    result = {} if state["residual"] is None else {"total": total}
    if state["out"] == "mx8":
        s = total.double()
        y = s / torch.sqrt((s * s).mean(1, keepdim=True) + _EPS) * state["weight"].double()
        return result | {"y": _rounded(y).to(torch.bfloat16)}
    scale = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + _EPS)
    result["y"] = (s * scale * w).to(kind)
    if state["train"]:
        grad = state["grad"].float()
        inner = (grad * w * s).mean(1, keepdim=True)
        of_total = scale * (grad * w - s * scale * scale * inner)
        if state["grad_total"] is not None:
            of_total = of_total + state["grad_total"].float()
        result["grad_x"] = of_total.to(kind)
        result["grad_weight"] = (grad * s * scale).sum(0).to(kind)
        if state["residual"] is not None:
            result["grad_residual"] = result["grad_x"]
    return result


def _linear_plain(state):
    out = _FLOATS[state["out"]]
    a = _rounded(state["a"].float()) if state["dtype"] == "mx8" else state["a"].float()
    w = _matrix(state["w"])
    pre = a @ w.T
    if state["bias"] is not None:
        pre = pre + state["bias"].float()
    y = _activated(pre, state["activation"])
    if state["residual"] is not None:
        y = y + state["residual"].float()
    result = {"y": y.to(out)}
    if state["train"]:
        grad = state["grad"].float() * _slope(pre, state["activation"])
        result["grad_a"], result["grad_w"] = (grad @ w).to(state["a"].dtype), (grad.T @ a).to(state["w"].dtype)
        if state["bias"] is not None:
            result["grad_bias"] = grad.sum(0).to(state["bias"].dtype)
        if state["residual"] is not None:
            result["grad_residual"] = state["grad"]
    return result


def _gated_plain(state):
    out, kind = _FLOATS[state["out"]], state["activation"]
    a = _rounded(state["a"].float()) if state["dtype"] == "mx8" else state["a"].float()
    gate, up = _matrix(state["gate"]), _matrix(state["up"])
    g, u = a @ gate.T, a @ up.T
    result = {"y": (_activated(g, kind) * u).to(out)}
    if state["train"]:
        grad = state["grad"].float()
        of_g, of_u = grad * u * _slope(g, kind), grad * _activated(g, kind)
        result["grad_a"] = (of_g @ gate + of_u @ up).to(state["a"].dtype)
        result["grad_gate"], result["grad_up"] = (of_g.T @ a).to(state["gate"].dtype), (of_u.T @ a).to(state["up"].dtype)
    return result


def _leaf(t):
    return None if t is None else t.detach().requires_grad_()


def _gradients(results, grads, **inputs):
    """The gradients of those inputs that there are, by name."""
    names = [name for name, t in inputs.items() if t is not None]
    return dict(zip(("grad_" + name for name in names), torch.autograd.grad(results, [inputs[name] for name in names], grads)))


def _norm_own(state):
    import numkong_amd as nk

    x, weight, residual = state["x"], state["weight"], state["residual"]
    if state["out"] == "mx8":
        y = nk.rms_norm_mx8(x, weight, residual, eps=_EPS)
        result = {}
        if residual is not None:
            y, result["total"] = y
        return result | {"y": nk.mx8_dequantize(y, torch.bfloat16)}
    if not state["train"]:
        y = nk.rms_norm(x, weight, residual, eps=_EPS)
        return {"y": y} if residual is None else {"y": y[0], "total": y[1]}
    x, weight, residual = _leaf(x), _leaf(weight), _leaf(residual)
    if residual is None:
        y = nk.rms_norm(x, weight, eps=_EPS)
        return {"y": y.detach()} | _gradients([y], [state["grad"]], x=x, weight=weight)
    y, total = nk.rms_norm(x, weight, residual, eps=_EPS)
    found = _gradients([y, total], [state["grad"], state["grad_total"]], x=x, weight=weight, residual=residual)
    return {"y": y.detach(), "total": total.detach()} | found


def _linear_own(state):
    import numkong_amd as nk

    kind = dict(activation=None if state["activation"] == "none" else state["activation"], out_dtype=_FLOATS[state["out"]])
    if not state["train"]:
        return {"y": nk.linear(state["a"], state["w"], state["bias"], residual=state["residual"], **kind)}
    a, w, bias, residual = (_leaf(state[name]) for name in ("a", "w", "bias", "residual"))
    y = nk.linear(a, w, bias, residual=residual, **kind)
    return {"y": y.detach()} | _gradients([y], [state["grad"]], a=a, w=w, bias=bias, residual=residual)


def _gated_own(state):
    import numkong_amd as nk

    kind = dict(activation=state["activation"], out_dtype=_FLOATS[state["out"]])
    if not state["train"]:
        return {"y": nk.gated_linear(state["a"], state["gate"], state["up"], **kind)}
    a, gate, up = (_leaf(state[name]) for name in ("a", "gate", "up"))
    y = nk.gated_linear(a, gate, up, **kind)
    return {"y": y.detach()} | _gradients([y], [state["grad"]], a=a, gate=gate, up=up)


def run(state):
    """One pass."""
    op = state["op"]
    if own:
        return _norm_own(state) if op == "norm" else _linear_own(state) if op == "linear" else _gated_own(state)
    return _norm_plain(state) if op == "norm" else _linear_plain(state) if op == "linear" else _gated_plain(state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _exact_rounded(x):
    """Each 32 of a row: the smallest power of two that leaves none above 448, then the nearest of e4m3's values, of two equally near
    ones the one whose last bit is zero."""
    blocks = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))
    largest = blocks.abs().amax(2, keepdim=True)
    power = torch.exp2(torch.ceil(torch.log2((largest / 448).clamp(min=2.0 ** -127))))
    power = torch.where(largest > 448 * power, 2 * power, power)
    power = torch.where((largest <= 224 * power) & (power > 2.0 ** -127), power / 2, power)
    units = blocks.abs() / power
    grid = torch.tensor([mantissa * 2.0 ** -9 for mantissa in range(8)]
                        + [(8 + mantissa) * 2.0 ** (exponent - 10) for exponent in range(1, 16) for mantissa in range(8)][:119],
                        dtype=torch.float64, device=x.device)
    above = torch.searchsorted(grid, units.contiguous()).clamp(max=126)  # the first that is not below
    below = (above - 1).clamp(min=0)
    to_above, to_below = grid[above] - units, units - grid[below]
    code = torch.where((to_above < to_below) | ((to_above == to_below) & (above % 2 == 0)), above, below)
    return (torch.copysign(grid[code], blocks) * power).flatten(1)[:, :x.shape[1]]


def _exact_matrix(w):
    if not hasattr(w, "codes") and not isinstance(w, dict):
        return w.double()
    codes, scales = (w["codes"], w["scales"]) if isinstance(w, dict) else (w.codes, w.scales)
    block = torch.arange(codes.shape[1], device=codes.device).div(32, rounding_mode="floor")
    return codes.to(torch.float64) * torch.exp2(scales.double() - 127)[:, block]


_EXACT = {
    "none": lambda x: x,
    "relu": torch.relu,
    "silu": torch.nn.functional.silu,
    "gelu": torch.nn.functional.gelu,
    "gelu_tanh": lambda x: torch.nn.functional.gelu(x, approximate="tanh"),
}


def exact(case, seed):
    state = prepare(case, seed)
    wide = lambda name: None if state.get(name) is None else state[name].double().requires_grad_(case["train"])  # noqa: E731
    if case["op"] == "norm":
        x, residual, weight = wide("x"), wide("residual"), wide("weight")
        total = x
        if residual is not None:
            held = (x.detach() + residual.detach()).to(state["x"].dtype).double()  # as it is held for the next layer
            total = x + residual + (held - x.detach() - residual.detach())
        y = total * torch.rsqrt(total.pow(2).mean(1, keepdim=True) + _EPS) * weight
        result = {"y": _exact_rounded(y) if case["out"] == "mx8" else y}
        if residual is not None:
            result["total"] = (x + residual).detach()
        leaves, results, grads = {"x": x, "weight": weight, "residual": residual}, [y], [state.get("grad")]
        if residual is not None:
            results, grads = [y, total], [state.get("grad"), state.get("grad_total")]
    else:
        a = _exact_rounded(state["a"]) if case["dtype"] == "mx8" else wide("a")
        if case["op"] == "linear":
            w = _exact_matrix(state["w"]).requires_grad_(case["train"])
            bias, residual = wide("bias"), wide("residual")
            y = torch.matmul(a, w.T)
            y = _EXACT[case["activation"]](y if bias is None else y + bias)
            y = y if residual is None else y + residual
            leaves = {"a": a, "w": w, "bias": bias, "residual": residual}
        else:
            gate, up = (_exact_matrix(state[name]).requires_grad_(case["train"]) for name in ("gate", "up"))
            y = _EXACT[case["activation"]](torch.matmul(a, gate.T)) * torch.matmul(a, up.T)
            leaves = {"a": a, "gate": gate, "up": up}
        result, results, grads = {"y": y}, [y], [state.get("grad")]
    if case["train"]:
        result |= _gradients(results, [g.double() for g in grads], **leaves)
    return {name: t.detach() for name, t in result.items()}


def work(case):
    """Operands read once, results written once; 8-bit matrices at 33 bytes for each 32 values."""
    m, k = case["m"], case["k"]
    if case["op"] == "norm":
        size, values = _BYTES[case["dtype"]], case["m"] * case["k"]
        moved = values * size * (3 if case["residual"] else 1)  # x; the residual and the total
        # (quantised values are also written as what they stand for)
        moved += values * (33 / 32 + 2) if case["out"] == "mx8" else values * size
        if case["train"]:  # gradients of the results, of x
            moved += values * size * (3 if case["residual"] else 2)
        return {"bytes": moved, "flops": values * (12 if case["train"] else 5)}
    n, out = case["n"], _BYTES[case["out"]]
    matrices, steps = (2 if case["op"] == "gated" else 1), 3 if case["train"] else 1
    width = 33 / 32 if case["dtype"] == "mx8" else 2
    moved = 2 * m * k + matrices * n * k * width + m * n * out
    if case.get("residual"):
        moved += m * n * out
    if case["train"]:
        moved += m * n * out + 2 * m * k + matrices * n * k * width
    return {"bytes": moved, "flops": 2 * matrices * m * n * k * steps}
