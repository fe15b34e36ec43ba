"""Plain 64-bit forms of the dense feed-forward operators, and how far 32-bit sums and 16-bit results may be from them."""
import math

import numpy as np
import torch

FLOATS = (torch.float32, torch.bfloat16, torch.float16)
HALVES = (torch.bfloat16, torch.float16)
UNIT = 2.0**-24  # half a step of f32, relative
ROUNDING = {dtype: torch.finfo(dtype).eps / 2 for dtype in FLOATS}
SMALLEST = {dtype: torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 for dtype in FLOATS}
ACTIVATIONS = (None, "relu", "silu", "gelu", "gelu_tanh")


def normal(rows, depth, dtype, seed, spread=0.5):
    generator = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, depth), generator=generator) * torch.exp(spread * torch.randn((rows, 1), generator=generator))
    return x.to(dtype)


def strided(x, pad, offset=0, device="cuda:0"):
    """The same matrix on the GPU, its rows `pad` values further apart and its start `offset` values into the allocation; NaN around it."""
    rows, depth = x.shape
    store = torch.full((rows * (depth + pad) + offset,), float("nan"), dtype=x.dtype, device=device)
    view = store[offset:].reshape(rows, depth + pad)[:, :depth]
    view.copy_(x)
    return view


# ---- 8-bit blocks --------------------------------------------------------------------------------------------------

GRID = np.concatenate([np.arange(8) * 2.0**-9] + [(8 + np.arange(8)) * 2.0 ** (e - 10) for e in range(1, 16)])[:127]  # e4m3's magnitudes


def quantize(x):
    """(codes, scale bytes) of the rows of a 64-bit matrix, by comparing with every magnitude of e4m3."""
    x = np.asarray(x.double().cpu() if isinstance(x, torch.Tensor) else x, dtype=np.float64)
    rows, depth = x.shape
    codes, scales = np.zeros((rows, depth), np.uint8), np.zeros((rows, (depth + 31) // 32), np.uint8)
    powers = 2.0 ** np.arange(-127, 128)
    for block in range(scales.shape[1]):
        part = x[:, block * 32:block * 32 + 32]
        bad = ~np.isfinite(part).all(1)
        part = np.where(bad[:, None], 0, part)
        scale = np.searchsorted(448 * powers, np.abs(part).max(1))  # the first power that is large enough
        units = np.abs(part) / powers[scale][:, None]
        high = np.minimum(np.searchsorted(GRID, units), 126)
        low = np.maximum(high - 1, 0)
        up, down = GRID[high] - units, units - GRID[low]
        code = np.where((up < down) | ((up == down) & (high % 2 == 0)), high, low) + 128 * np.signbit(part)
        codes[:, block * 32:block * 32 + 32] = np.where(bad[:, None], 0, code)
        scales[:, block] = np.where(bad, 255, scale)
    return codes, scales


def values(codes, scales):
    """What codes and scale bytes stand for."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    magnitude = np.append(GRID, np.nan)[codes & 127]
    powers = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return np.where(codes > 127, -magnitude, magnitude) * np.repeat(powers, 32, axis=1)[:, :codes.shape[1]]


def bytes_of(matrix):
    """(codes, scales) of an Mx8Matrix as arrays of bytes."""
    return matrix.codes.cpu().contiguous().view(torch.uint8).numpy(), matrix.scales.cpu().numpy()


def matrix_values(matrix):
    return torch.from_numpy(values(*bytes_of(matrix)))


# ---- activations ---------------------------------------------------------------------------------------------------


def activate(kind, x):
    if kind == "relu":
        return torch.clamp(x, min=0)
    if kind == "silu":
        return x * torch.sigmoid(x)
    if kind == "gelu":
        return 0.5 * x * torch.erfc(-x * math.sqrt(0.5))
    if kind == "gelu_tanh":
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x**3))
    return x


def slope(kind, x):
    if kind is None:
        return torch.ones_like(x)
    x = x.detach().clone().requires_grad_()
    return torch.autograd.grad(activate(kind, x).sum(), x)[0]


# Over all x: |f'| <= 1.13 and |f''| <= 1.13 for the smooth ones (gelu: f' largest at sqrt 2, f'' at 0, where it is 0.8).
STEEPEST, BEND = 1.13, 1.13


def activation_error(kind, p, error):
    """How far f(p) may be off: what p's error makes of it, and some roundings of the functions themselves (of e^x's argument as well)."""
    own = 0.0 if kind in (None, "relu") else (16 + 4 * p.abs().clamp(max=100)) * UNIT * (activate(kind, p).abs() + 1e-30)
    return (1.0 if kind in (None, "relu") else STEEPEST) * error + own


def slope_error(kind, p, error):
    if kind is None:
        return torch.zeros_like(p)
    if kind == "relu":
        return (p.abs() <= error).double()  # on which side of zero p is
    return BEND * error + (32 + 4 * p.abs().clamp(max=110)) * UNIT * (1 + 0 * p)


# ---- products ------------------------------------------------------------------------------------------------------


def sum_error(depth, magnitude):
    """A product's 32-bit sums: products of 16-bit values are exact, a matrix instruction adds them up in eights with a rounding each, and
    partial sums of up to 32 wavefronts or pieces of the depth are added; each rounding is off by at most 2^-24 of at most `magnitude`."""
    return (depth / 8 + 40) * UNIT * magnitude


def mx8_sum_error(a, w):
    """Of 8-bit products: in each 32 of the depth every product may lose what is below 2^-13 of the largest (the instruction's own
    rounding, as probed), and sums between lanes keep 18 bits."""
    depth = a.shape[1]
    pad = torch.nn.functional.pad
    a, w = pad(a, (0, -depth % 32)).abs().unflatten(1, (-1, 32)), pad(w, (0, -depth % 32)).abs().unflatten(1, (-1, 32))
    largest = a.amax(2) @ w.amax(2).T
    return 32 * 2.0**-13 * largest + (depth / 32 + 40) * 2.0**-18 * largest


def assert_within(got, truth, allowed, what="result"):
    got, truth = got.double().cpu(), truth.double().cpu()
    allowed = (allowed if isinstance(allowed, torch.Tensor) else torch.tensor(float(allowed))).double().cpu().expand(truth.shape)
    assert got.shape == truth.shape
    assert torch.equal(torch.isnan(got), torch.isnan(truth)), f"{what}: NaNs elsewhere"
    infinite = torch.isinf(truth)
    assert torch.equal(got[infinite], truth[infinite]), f"{what}: infinities elsewhere"
    fine = torch.isfinite(truth)
    over = ((got - truth).abs() - allowed)[fine]
    if over.numel():
        worst = ((got - truth).abs() / allowed.clamp(min=1e-300))[fine].max()
        assert not (over > 0).any(), f"{what}: off by {worst:.3g} of what is allowed"


def rounded(error, truth, dtype):
    """`error` and the rounding of a result to `dtype`."""
    return error + ROUNDING[dtype] * (truth.abs() + error) + SMALLEST[dtype]


class Linear:
    """The product and its gradients in 64 bits, with what each may be off by. `a`, `w`, `w_up`: 64-bit values; `half`: their type."""

    def __init__(self, a, w, w_up=None, bias=None, activation=None, residual=None, half=torch.bfloat16, sums=None):
        self.a, self.w, self.w_up, self.kind, self.half = a, w, w_up, activation, half
        self.p = a @ w.T
        self.p_error = (sums or sum_error)(a.shape[1], a.abs() @ w.abs().T) if sums is not mx8_sum_error else mx8_sum_error(a, w)
        if bias is not None:
            self.p = self.p + bias
            self.p_error = self.p_error + UNIT * (self.p.abs() + self.p_error)
        f, f_error = activate(activation, self.p), activation_error(activation, self.p, self.p_error)
        self.f, self.f_error = f, f_error
        if w_up is not None:
            self.q = a @ w_up.T
            self.q_error = sum_error(a.shape[1], a.abs() @ w_up.abs().T) if sums is not mx8_sum_error else mx8_sum_error(a, w_up)
            self.y = f * self.q
            self.y_error = f_error * (self.q.abs() + self.q_error) + f.abs() * self.q_error + UNIT * self.y.abs()
        else:
            self.y, self.y_error = f, f_error
        if residual is not None:
            self.y = self.y + residual
            self.y_error = self.y_error + UNIT * (self.y.abs() + self.y_error)

    def check(self, y, what="y"):
        assert_within(y, self.y, rounded(self.y_error, self.y, y.dtype), what)

    def gradients(self, grad):
        """{name: (truth, error)}; `bias` is the sum of d."""
        s, s_error = slope(self.kind, self.p), slope_error(self.kind, self.p, self.p_error)
        g = grad.abs()
        half = ROUNDING[self.half]
        if self.w_up is None:
            pairs = [(grad * s, g * s_error, self.w)]
        else:
            q, q_error = self.q.abs(), self.q_error
            pairs = [(grad * s * self.q, g * ((s.abs() + s_error) * q_error + s_error * q), self.w), (grad * self.f, g * self.f_error, self.w_up)]
        found, of_a, of_a_error = {}, 0, 0
        for i, (d, error, w) in enumerate(pairs):
            error = error + 4 * UNIT * (d.abs() + error)
            if i == 0:
                found["bias"] = d.sum(0), error.sum(0) + (d.shape[0] + 8) * UNIT * (d.abs() + error).sum(0)
            error = error + half * (d.abs() + error) + SMALLEST[self.half]  # as an operand of the matrix instructions
            of_a = of_a + d @ w
            of_a_error = of_a_error + error @ w.abs() + sum_error(2 * d.shape[1], (d.abs() + error) @ w.abs())
            found["w_up" if i else "w"] = d.T @ self.a, error.T @ self.a.abs() + sum_error(d.shape[0], (d.abs() + error).T @ self.a.abs())
        found["a"] = of_a, of_a_error
        return found

    def check_gradients(self, grad, **got):
        truth = self.gradients(grad.double())
        for name, t in got.items():
            value, error = truth[name]
            assert_within(t, value, rounded(error, value, t.dtype), f"gradient of {name}")


# ---- the norm ------------------------------------------------------------------------------------------------------


def norm(total, weight=None, eps=1e-6):
    t = total.double()
    y = t / torch.sqrt(t.square().mean(1, keepdim=True) + eps)
    return y if weight is None else y * weight.double()


def norm_gradients(grad, total, weight=None, grad_total=None, eps=1e-6):
    """((of x, its error), (of weight, its error)) in 64 bits."""
    t, g = total.double(), grad.double()
    gw = g if weight is None else g * weight.double()
    s = 1 / torch.sqrt(t.square().mean(1, keepdim=True) + eps)
    depth = t.shape[1]
    sums = (depth / 64 + 40) * UNIT  # adding up a row's products: a thread's own, lanes, wavefronts
    shift, shift_size = (gw * t).mean(1, keepdim=True) * s * s, (gw * t).abs().mean(1, keepdim=True) * s * s
    of_x = s * (gw - t * shift)
    error = s * (gw.abs() + t.abs() * shift_size) * (3 * sums + 16 * UNIT)
    if grad_total is not None:
        of_x = of_x + grad_total.double()
        error = error + 2 * UNIT * of_x.abs()
    parts = g * t * s
    of_weight, weight_error = parts.sum(0), parts.abs().sum(0) * (sums + (t.shape[0] + 40) * UNIT)
    return (of_x, error), (of_weight, weight_error)
