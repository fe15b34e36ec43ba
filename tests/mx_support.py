"""Plain 64-bit forms of the microscaled 4-bit operators and of the routing to experts, on the CPU."""
import numpy as np
import torch

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def quantize(x):
    """(codes one to a value, scale bytes) of the rows of a float matrix, by comparing with every element of the grid."""
    x = np.asarray(x.double().cpu() if isinstance(x, torch.Tensor) else x, dtype=np.float64)
    rows, depth = x.shape
    blocks = (depth + 31) // 32
    codes, scales = np.zeros((rows, depth), dtype=np.uint8), np.zeros((rows, blocks), dtype=np.uint8)
    for block in range(blocks):
        part = x[:, block * 32:block * 32 + 32]
        bad = ~np.isfinite(part).all(1)
        largest = np.where(np.isfinite(part), np.abs(part), 0).max(1)
        exponent = np.where(largest > 0, np.frexp(largest)[1] - 1 - 2, -127).clip(-127, 127)
        units = np.where(np.isfinite(part), part, 0) / np.exp2(exponent)[:, None]
        distance = np.abs(np.abs(units)[:, :, None] - GRID[:8])
        nearest = distance.min(2, keepdims=True)
        # of two equally near magnitudes the one with the even code
        code = np.where(distance == nearest, np.arange(8) % 2 * 8 + np.arange(8), 99).argmin(2)
        code = (code + 8 * np.signbit(part)).astype(np.uint8)
        codes[:, block * 32:block * 32 + 32] = np.where(bad[:, None], 0, code)
        scales[:, block] = np.where(bad, 255, exponent + 127)
    return codes, scales


def values(codes, scales):
    """What codes (one to a value) and scale bytes stand for."""
    powers = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return GRID[codes] * np.repeat(powers, 32, axis=1)[:, :codes.shape[1]]


def unpacked(packed_codes, depth):
    """One code to a value, from two to a byte."""
    packed_codes = np.asarray(packed_codes.cpu() if isinstance(packed_codes, torch.Tensor) else packed_codes)
    both = np.stack([packed_codes & 15, packed_codes >> 4], -1)
    return both.reshape(*packed_codes.shape[:-1], -1)[..., :depth]


def packed(codes):
    """Two codes to a byte, the even column in the low half."""
    if codes.shape[-1] % 2:
        codes = np.concatenate([codes, np.zeros((*codes.shape[:-1], 1), np.uint8)], -1)
    return codes[..., 0::2] | codes[..., 1::2] << 4


def rounded(x):
    return values(*quantize(x))


def sum_bound(depth, magnitude):
    """How far a product's 32-bit sums may be from the truth. The sum over a block is exact (whole quarters below 2^13), so
    is its scaling; depth / 32 block sums and the partial sums of eight wavefronts are added in 32 bits, each addition off
    by at most 2^-23 of what has been added, which is at most `magnitude`, the sum of the products' magnitudes."""
    return ((depth + 31) // 32 + 8) * 2.0**-23 * magnitude


FLOATS = (torch.float32, torch.bfloat16, torch.float16)
ROUNDING = {dtype: torch.finfo(dtype).eps / 2 for dtype in FLOATS}  # half a unit of the last place
SMALLEST = {dtype: torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 for dtype in FLOATS}  # half the smallest subnormal


def close(result, truth, magnitude, depth, extra=0.0):
    """Asserts that a product's results are as near as its sums and the rounding of its results allow."""
    got = result.double().cpu().numpy()
    allowed = sum_bound(depth, magnitude) + extra
    allowed = allowed + ROUNDING[result.dtype] * (np.abs(truth) + allowed) + SMALLEST[result.dtype]
    worst = np.abs(got - truth) / allowed
    assert np.array_equal(np.isnan(got), np.isnan(truth))
    assert not np.any(worst > 1), f"off by {np.nanmax(worst):.3g} of what is allowed at {np.unravel_index(np.nanargmax(worst), worst.shape)}"


def scores(logits, score):
    """64-bit scores; logits of -inf have none."""
    logits = np.asarray(logits, dtype=np.float64)
    masked = np.isneginf(logits)
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            return 1 / (1 + np.exp(-logits))
        top = logits.max(1, keepdims=True)
        e = np.where(masked, 0, np.exp(logits - np.where(np.isneginf(top), 0, top)))
        return e / np.maximum(e.sum(1, keepdims=True), 1e-300)


def choice(logits, score, bias=None, groups=1, top_groups=1, group_top=1):
    """64-bit selection scores, -inf where an expert cannot be chosen; groups that drop out as well."""
    logits = np.asarray(logits, dtype=np.float64)
    selection = logits if bias is None else np.where(np.isneginf(logits), -np.inf, scores(logits, score) + np.asarray(bias, np.float64))
    if groups > 1:
        inside = selection.reshape(len(logits), groups, -1)
        of_group = np.sort(inside, 2)[:, :, ::-1][:, :, :group_top].sum(2)
        order = np.argsort(-of_group, axis=1, kind="stable")
        keep = np.zeros_like(of_group, dtype=bool)
        np.put_along_axis(keep, order[:, :top_groups], True, 1)
        selection = np.where(keep[:, :, None], inside, -np.inf).reshape(selection.shape)
    return selection


def weights(logits, chosen, score, renormalize, scale):
    s = scores(logits, score)
    there = chosen >= 0
    picked = np.where(there, np.take_along_axis(s, np.maximum(chosen, 0), 1), 0)
    if renormalize:
        picked = picked / (picked.sum(1, keepdims=True) + 1e-20)
    return scale * picked
