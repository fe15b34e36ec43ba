"""The microscaled 4-bit operators and the routing to experts, as cases that can be timed and compared.

Where `own` is false, `run` computes each operator from elementary torch operations in 32 bits; where it is true, it makes
the calls that a user makes of this package. A case is one of four passes:

  quantize   values to 4-bit codes with a scale per 32 of a row, and back to the values that these stand for
  dots       activations (quantised in the call) times a 4-bit matrix that the program keeps
  route      scores to experts and weights, with the gradient of the scores where `train` is set
  experts    each token's row times the matrices of the experts that it was sent to, summed by weight where `combine` is set

Sizes are those of this repository's configurations (8192^3, 8192 x 8191 x 1000) or generic ones.
"""
import math

import torch

own = False

_FLOATS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # A decoding batch's activations: the smallest call, where latency is all.
        {"name": "quantize_tokens", "op": "quantize", "dtype": "bf16", "m": 16, "k": 4096},
        # A whole matrix of weights in single precision, as a checkpoint is converted.
        {"name": "quantize_matrix", "op": "quantize", "dtype": "f32", "m": 8192, "k": 8192},
        # One token against a layer: the stream of the matrix.
        {"name": "dots_token", "op": "dots", "dtype": "bf16", "out": "bf16", "m": 1, "n": 8192, "k": 8192},
        # A server's batch of single tokens.
        {"name": "dots_batch", "op": "dots", "dtype": "bf16", "out": "bf16", "m": 64, "n": 8192, "k": 8192},
        # The ragged configuration: nothing but the rows is a multiple of a tile, the last block of a row is cut.
        {"name": "dots_ragged", "op": "dots", "dtype": "f16", "out": "f32", "m": 8192, "n": 8191, "k": 1000},
        # The size of the headline metric: a long prompt against a wide layer.
        {"name": "dots_square", "op": "dots", "dtype": "bf16", "out": "bf16", "m": 8192, "n": 8192, "k": 8192},
        # The router of a decoding batch.
        {"name": "route_tokens", "op": "route", "dtype": "f32", "tokens": 16, "experts": 64, "top_k": 4, "score": "softmax",
         "renorm": True, "groups": 1, "top_groups": 1, "train": False, "padded": 0.0},
        # The router of a long prompt: scores by sigmoid, a bias for balance, experts in groups.
        {"name": "route_prompt", "op": "route", "dtype": "f32", "tokens": 16384, "experts": 256, "top_k": 8,
         "score": "sigmoid", "renorm": True, "groups": 8, "top_groups": 4, "train": False, "padded": 0.0},
        # The router in training: the gradient of its scores as well, some of the tokens padding.
        {"name": "route_train", "op": "route", "dtype": "bf16", "tokens": 8192, "experts": 128, "top_k": 8,
         "score": "softmax", "renorm": True, "groups": 1, "top_groups": 1, "train": True, "padded": 0.05},
        # Four tokens, each to eight experts of many: the stream of the matrices that they hit.
        {"name": "experts_tokens", "op": "experts", "dtype": "bf16", "out": "bf16", "tokens": 4, "experts": 128, "top_k": 8,
         "n": 2048, "k": 2048, "combine": False, "padded": 0.0},
        # A long prompt through the first product of a layer of experts.
        {"name": "experts_prompt", "op": "experts", "dtype": "bf16", "out": "bf16", "tokens": 4096, "experts": 64, "top_k": 8,
         "n": 2048, "k": 2048, "combine": False, "padded": 0.0},
        # A middling batch through the last product, summed by weight; odd sizes, some of the tokens padding.
        {"name": "experts_combine", "op": "experts", "dtype": "f16", "out": "f32", "tokens": 1001, "experts": 32, "top_k": 4,
         "n": 2050, "k": 1000, "combine": True, "padded": 0.05},
    ]


def _cost(case):
    """A rough time in seconds of the plain form, for keeping drawn cases within the largest listed one."""
    needed = work(case)
    return needed["flops"] / 1e14 + needed["bytes"] / 1e12


def draw(rng):
    """One more case of the same four passes, sizes over the whole range of each, two thirds of them multiples of nothing."""
    def size(low, high):
        value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        if rng.random() < 0.35:
            step = 128 if value >= 512 else (32 if value >= 64 else 1)
            value = value // step * step
        return max(low, min(high, value))

    op = rng.choice(["quantize", "dots", "dots", "dots", "route", "route", "experts", "experts", "experts"])
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "quantize":
        case |= {"m": size(1, 16384), "k": size(32, 16384)}
    elif op == "dots":
        case |= {"out": rng.choice(["bf16", "f32", "f16"]), "m": size(1, 8192), "n": size(256, 8192), "k": size(64, 8192)}
    elif op == "route":
        score = rng.choice(["softmax", "sigmoid"])
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * rng.randint(4, 256 // groups)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(10, experts // groups * top_groups))
        # (the weight of a single expert is not renormalised: it would be the same for every token)
        case |= {"tokens": size(1, 16384), "experts": experts, "top_k": top_k, "score": score,
                 "renorm": top_k > 1 and rng.random() < 0.7, "groups": groups, "top_groups": top_groups, "train": rng.random() < 0.5,
                 "padded": rng.choice([0.0, 0.1])}
    else:
        experts = rng.choice([8, 16, 32, 60, 64, 128])
        case |= {"out": rng.choice(["bf16", "bf16", "f32"]), "tokens": size(1, 4096), "experts": experts,
                 "top_k": rng.randint(1, 8), "n": size(256, 4096), "k": size(128, 4096), "combine": rng.random() < 0.5,
                 "padded": rng.choice([0.0, 0.1])}
        while case["experts"] * case["n"] * case["k"] > 64 * 2048 * 2048 * 2:
            case["n" if case["n"] > case["k"] else "k"] //= 2
    limit = max(_cost(one) for one in listed())
    while _cost(case) > limit:
        side = max((s for s in ("m", "n", "k", "tokens") if s in case), key=lambda s: case[s])
        case[side] = case[side] * 3 // 4
    return case


# ---- the inputs ----------------------------------------------------------------------------------------------------

def _activations(rows, k, dtype, generator):
    """Normal values; one channel of 64 is eight times as large, as the channels of hidden states are; rows differ in size."""
    x = torch.randn((rows, k), device="cuda:0", generator=generator)
    x *= 1.0 + 7.0 * (torch.rand((k,), device="cuda:0", generator=generator) < 1 / 64)
    x *= torch.exp(0.5 * torch.randn((rows, 1), device="cuda:0", generator=generator))
    return x.to(_FLOATS[dtype])


def _weights(rows, k, generator):
    """A matrix of weights as a 4-bit checkpoint holds it: codes, two to a byte with the even column in the low half, and
    a scale's exponent (biased by 127) for each 32 columns."""
    codes = torch.empty((rows, (k + 1) // 2), dtype=torch.uint8, device="cuda:0")
    scales = torch.empty((rows, (k + 31) // 32), dtype=torch.uint8, device="cuda:0")
    slab = max(1, (1 << 26) // k)
    for first in range(0, rows, slab):
        w = torch.randn((min(slab, rows - first), k), device="cuda:0", generator=generator) / math.sqrt(k)
        exponents, values = _quantized(w)
        scales[first:first + slab] = (exponents + 127).to(torch.uint8)
        nibbles = (_grid_code(values.abs()) + 8 * torch.signbit(values)).to(torch.uint8).reshape(w.shape[0], -1)
        nibbles = nibbles[:, :k]
        if k % 2:
            nibbles = torch.cat([nibbles, nibbles.new_zeros((w.shape[0], 1))], 1)
        codes[first:first + slab] = nibbles[:, 0::2] | nibbles[:, 1::2] << 4
    return codes, scales


def _routed(case, generator):
    """Experts of each token, some of them more popular than others, and their weights; padding goes to no expert (-1)."""
    scores = torch.randn((case["tokens"], case["experts"]), device="cuda:0", generator=generator)
    scores += 0.5 * torch.randn((case["experts"],), device="cuda:0", generator=generator)
    best = torch.topk(scores, case["top_k"], dim=1)
    padding = torch.rand((case["tokens"], 1), device="cuda:0", generator=generator) < case["padded"]
    return best.indices.masked_fill(padding, -1).to(torch.int32), torch.softmax(best.values, 1).masked_fill(padding, 0.0)


def prepare(case, seed):
    generator = torch.Generator(device="cuda:0").manual_seed(seed)
    state = dict(case)
    if case["op"] == "quantize":
        state["x"] = _activations(case["m"], case["k"], case["dtype"], generator)
    elif case["op"] == "dots":
        state["a"] = _activations(case["m"], case["k"], case["dtype"], generator)
        state["codes"], state["scales"] = _weights(case["n"], case["k"], generator)
        if own:  # the matrix as a program keeps it: laid out once for the product
            import numkong_amd as nk

            state["packed"] = nk.mx_pack(nk.MxMatrix(state["codes"], state["scales"], case["k"]))
    elif case["op"] == "route":
        logits = torch.randn((case["tokens"], case["experts"]), device="cuda:0", generator=generator)
        logits += 0.5 * torch.randn((case["experts"],), device="cuda:0", generator=generator)
        padding = torch.rand((case["tokens"], 1), device="cuda:0", generator=generator) < case["padded"]
        state["logits"] = (1.5 * logits).masked_fill(padding, -math.inf).to(_FLOATS[case["dtype"]])
        # the bias that a balanced training run has left behind (with sigmoid scores, as it is used)
        bias = 0.1 * torch.randn((case["experts"],), device="cuda:0", generator=generator)
        state["bias"] = bias if case["score"] == "sigmoid" else None
        state["grad"] = torch.randn((case["tokens"], case["top_k"]), device="cuda:0", generator=generator)
    else:
        state["a"] = _activations(case["tokens"], case["k"], case["dtype"], generator)
        codes, scales = _weights(case["experts"] * case["n"], case["k"], generator)
        state["codes"] = codes.reshape(case["experts"], case["n"], -1)
        state["scales"] = scales.reshape(case["experts"], case["n"], -1)
        state["chosen"], state["weights"] = _routed(case, generator)
        if own:
            import numkong_amd as nk

            state["packed"] = nk.mx_pack(nk.MxMatrix(state["codes"], state["scales"], case["k"]))
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _grid_code(magnitude):
    """The 3-bit code of a magnitude that is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6."""
    return torch.where(magnitude < 2, 2 * magnitude, torch.where(magnitude < 4, magnitude + 2, magnitude / 2 + 4))


def _quantized(x):
    """Exponents (rows, blocks) and the values in units of the scale (rows, blocks, 32) of 32-bit values; the last block
    of a row is filled with zeros."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % 32)).reshape(rows, -1, 32)
    largest = x.abs().amax(2)
    exponents = (torch.frexp(largest).exponent - 3).clamp(-127, 127)
    exponents = torch.where(largest == 0, -127, exponents)
    scaled = torch.ldexp(x, -exponents[..., None])
    step = torch.ldexp(torch.ones_like(scaled), (torch.frexp(scaled).exponent - 1).clamp(min=0) - 1)
    return exponents, (torch.round(scaled / step) * step).clamp(-6, 6)


def _rounded(x):
    """x as its quantised values, 32 bits."""
    exponents, values = _quantized(x.float())
    return torch.ldexp(values, exponents[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _dequantized(codes, scales, k):
    """(..., rows, k) values of codes and scales, 32 bits."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    values = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).flatten(-2)[..., :k]
    powers = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return values * powers.repeat_interleave(32, -1)[..., :k]


def _route_plain(state):
    logits = state["logits"].float()
    tokens, experts = logits.shape
    masked = logits == -math.inf
    top = logits.amax(1, keepdim=True)
    exponentials = torch.where(masked, 0.0, torch.exp(logits - top))
    if state["score"] == "softmax":
        scores = exponentials / exponentials.sum(1, keepdim=True).clamp(min=1e-37)
        choice = logits
    else:
        scores = 1 / (1 + torch.exp(-logits))
        choice = (scores + state["bias"]).masked_fill(masked, -math.inf)
    if state["groups"] > 1:
        inside = choice.reshape(tokens, state["groups"], -1)
        if state["score"] == "softmax":
            of_group = inside.amax(2)
        else:
            two = torch.topk(inside, min(2, inside.shape[2]), dim=2).values
            of_group = two.sum(2)
        chosen_groups = torch.sort(of_group, dim=1, descending=True, stable=True).indices[:, :state["top_groups"]]
        stays = torch.zeros_like(of_group, dtype=torch.bool).scatter_(1, chosen_groups, True)
        choice = inside.masked_fill(~stays[..., None], -math.inf).reshape(tokens, experts)
    order = torch.sort(choice, dim=1, descending=True, stable=True)
    chosen = order.indices[:, :state["top_k"]]
    empty = order.values[:, :state["top_k"]] == -math.inf
    picked = scores.gather(1, chosen).masked_fill(empty, 0.0)
    total = picked.sum(1, keepdim=True) + 1e-20
    weights = 2.5 * (picked / total if state["renorm"] else picked)
    result = {"weights": weights, "experts": chosen.masked_fill(empty, -1).to(torch.int32)}
    if state["train"]:
        grad = state["grad"].masked_fill(empty, 0.0)
        of_picked = 2.5 * ((grad - (grad * picked).sum(1, keepdim=True) / total) / total if state["renorm"] else grad)
        if state["score"] == "softmax":
            of_scores = torch.zeros_like(scores).scatter_add_(1, chosen, of_picked.masked_fill(empty, 0.0))
            of_logits = scores * (of_scores - (of_scores * scores).sum(1, keepdim=True))
        else:
            slope = picked * (1 - picked)
            of_logits = torch.zeros_like(scores).scatter_add_(1, chosen, (of_picked * slope).masked_fill(empty, 0.0))
        result["grad_logits"] = of_logits.to(state["logits"].dtype)
    return result


def _experts_plain(state):
    a, chosen = _rounded(state["a"]), state["chosen"].reshape(-1).long()
    slots, top_k, experts = chosen.numel(), state["top_k"], state["codes"].shape[0]
    n, k = state["n"], state["k"]
    token = torch.arange(slots, device=a.device) // top_k
    if slots <= experts:  # few rows: the matrices that they need
        at = chosen.clamp(min=0)
        y = torch.bmm(_dequantized(state["codes"][at], state["scales"][at], k), a[token][:, :, None]).reshape(slots, n)
    else:  # many: the rows of each expert, filled up to the same number
        counts = torch.bincount(chosen + 1, minlength=experts + 1)[1:]
        order = torch.sort(chosen, stable=True).indices[slots - counts.sum():]
        expert = chosen[order]
        place = torch.arange(order.numel(), device=a.device) - (counts.cumsum(0) - counts)[expert]
        rows = torch.zeros((experts, int(counts.max()), k), device=a.device)
        rows[expert, place] = a[token[order]]
        product = torch.bmm(_dequantized(state["codes"], state["scales"], k), rows.transpose(1, 2).contiguous())
        y = torch.zeros((slots, n), device=a.device)
        y[order] = product.transpose(1, 2)[expert, place]
    y = torch.where(chosen[:, None] < 0, 0.0, y).reshape(-1, top_k, n)
    if state["combine"]:
        y = (y * state["weights"][:, :, None]).sum(1)
    return y.to(_FLOATS[state["out"]])


def run(state):
    """One pass."""
    op = state["op"]
    if own:
        import numkong_amd as nk

        if op == "quantize":
            return nk.mx_dequantize(nk.mx_quantize(state["x"]), state["x"].dtype)
        if op == "dots":
            return nk.mx_dots_packed(state["a"], state["packed"], out_dtype=_FLOATS[state["out"]])
        if op == "route":
            kind = dict(score=state["score"], renormalize=state["renorm"], scale=2.5)
            weights, experts = nk.experts_route(state["logits"], state["top_k"], bias=state["bias"], groups=state["groups"],
                                                top_groups=state["top_groups"], group_top=2 if state["bias"] is not None else 1, **kind)
            result = {"weights": weights, "experts": experts}
            if state["train"]:
                result["grad_logits"] = nk.experts_route_backward(state["grad"], state["logits"], experts, **kind)
            return result
        plan = nk.experts_plan(state["chosen"], state["experts"])
        return nk.mx_dots_experts(state["a"], state["packed"], plan, weights=state["weights"] if state["combine"] else None,
                                  out_dtype=_FLOATS[state["out"]])
    if op == "quantize":
        return _rounded(state["x"]).to(state["x"].dtype)
    if op == "dots":
        a = _rounded(state["a"])
        return (a @ _dequantized(state["codes"], state["scales"], state["k"]).T).to(_FLOATS[state["out"]])
    return _route_plain(state) if op == "route" else _experts_plain(state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _exact_rounded(x):
    """Each 32 of a row: the power of two that brings the largest into [4, 8), then the nearest of the eight magnitudes,
    of two equally near ones the one with the even code."""
    x = x.double()
    blocks = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))
    largest = blocks.abs().amax(2, keepdim=True)
    power = torch.exp2(torch.floor(torch.log2(largest.clamp(min=2.0 ** -125))) - 2)
    power = torch.where(largest >= 8 * power, 2 * power, torch.where(largest < 4 * power, (power / 2).clamp(min=2.0 ** -127), power))
    units = (blocks.abs() / power)
    found = torch.zeros_like(units)
    for above, (bound, closed) in {0.5: (0.25, False), 1.0: (0.75, True), 1.5: (1.25, False), 2.0: (1.75, True),
                                   3.0: (2.5, False), 4.0: (3.5, True), 6.0: (5.0, False)}.items():
        found = torch.where((units >= bound) if closed else (units > bound), above, found)
    return (torch.copysign(found, blocks) * power).flatten(1)[:, :x.shape[1]]


def _exact_matrix(codes, scales, k):
    low, high = codes.bitwise_and(15), codes.bitwise_right_shift(4)
    code = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.int64, device=codes.device)
    code[..., 0::2], code[..., 1::2] = low.long(), high.long()
    code = code[..., :k]
    exponent, mantissa = code.bitwise_right_shift(1).bitwise_and(3), code.bitwise_and(1)
    magnitude = torch.where(exponent == 0, 0.5 * mantissa.double(), (1 + 0.5 * mantissa.double()) * torch.exp2(exponent.double() - 1))
    block = torch.arange(k, device=codes.device).div(32, rounding_mode="floor")
    return torch.where(code > 7, -magnitude, magnitude) * torch.exp2(scales.double() - 127)[..., block]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_rounded(state["x"])
    if case["op"] == "dots":
        return _exact_rounded(state["a"]) @ _exact_matrix(state["codes"], state["scales"], case["k"]).T
    if case["op"] == "experts":
        a = _exact_rounded(state["a"])
        y = torch.zeros((case["tokens"], case["top_k"], case["n"]), dtype=torch.float64, device=a.device)
        for expert in range(case["experts"]):
            token, slot = torch.nonzero(state["chosen"] == expert, as_tuple=True)
            if token.numel():
                y[token, slot] = a[token] @ _exact_matrix(state["codes"][expert], state["scales"][expert], case["k"]).T
        return (y * state["weights"].double()[:, :, None]).sum(1) if case["combine"] else y
    logits = state["logits"].double()
    masked = torch.isneginf(logits)
    every = masked.all(1, keepdim=True)
    scores = torch.softmax(logits.masked_fill(every, 0.0), 1) if case["score"] == "softmax" else torch.sigmoid(logits)
    scores = scores.masked_fill(masked, 0.0)
    choice = (scores if state["bias"] is None else scores + state["bias"].double()).masked_fill(masked, -math.inf)
    if case["groups"] > 1:
        inside = choice.unflatten(1, (case["groups"], -1))
        best = inside.sort(2, descending=True).values[:, :, :1 if state["bias"] is None else 2].sum(2)
        rank = best.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
        choice = inside.masked_fill((rank >= case["top_groups"])[:, :, None], -math.inf).flatten(1)
    chosen = choice.argsort(dim=1, descending=True, stable=True)[:, :case["top_k"]]
    there = choice.gather(1, chosen) > -math.inf
    leaf = logits.masked_fill(masked, -1e30).masked_fill(every, 0.0).requires_grad_()
    again = torch.softmax(leaf, 1) if case["score"] == "softmax" else torch.sigmoid(leaf)
    picked = again.gather(1, chosen) * there
    weights = 2.5 * (picked / (picked.sum(1, keepdim=True) + 1e-20) if case["renorm"] else picked)
    result = {"weights": weights.detach(), "experts": None}
    if case["train"]:
        (weights * state["grad"].double()).sum().backward()
        result["grad_logits"] = leaf.grad.masked_fill(masked, 0.0)
    return result


def work(case):
    """Operands read once, results written once; 4-bit matrices at 17 bytes for each 32 values. The experts' product reads
    the matrices of those experts that its tokens are expected to hit."""
    matrix = lambda rows, k: rows * (k / 2 + k / 32)  # noqa: E731
    if case["op"] == "quantize":
        values = case["m"] * case["k"]
        return {"bytes": 2 * values * _BYTES[case["dtype"]] + matrix(case["m"], case["k"]), "flops": 2 * values}
    if case["op"] == "dots":
        moved = case["m"] * case["k"] * _BYTES[case["dtype"]] + matrix(case["n"], case["k"]) + case["m"] * case["n"] * _BYTES[case["out"]]
        return {"bytes": moved, "flops": 2 * case["m"] * case["n"] * case["k"]}
    if case["op"] == "route":
        scores, chosen = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        moved = scores * _BYTES[case["dtype"]] + 8 * chosen
        if case["train"]:
            moved += scores * _BYTES[case["dtype"]] + 4 * chosen
        return {"bytes": moved, "flops": scores * (8 if case["train"] else 4)}
    slots = case["tokens"] * case["top_k"] * (1 - case["padded"])
    hit = case["experts"] * (1 - (1 - min(1.0, case["top_k"] / case["experts"])) ** (case["tokens"] * (1 - case["padded"])))
    moved = case["tokens"] * case["k"] * _BYTES[case["dtype"]] + hit * matrix(case["n"], case["k"])
    moved += case["tokens"] * case["n"] * _BYTES[case["out"]] * (1 if case["combine"] else case["top_k"])
    return {"bytes": moved, "flops": 2 * slots * case["n"] * case["k"]}
