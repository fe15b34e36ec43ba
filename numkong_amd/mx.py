"""Microscaled 4-bit floats and the routing to experts: the Python side of ``include/numkong_amd/mx.h``.

A matrix of 4-bit floats (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) has one power of two for each 32 values of
a row. ``mx_quantize`` makes one of a float matrix, ``mx_pack`` lays a matrix (or a stack of them, one for each expert) out
for products, ``mx_dots_packed`` multiplies as ``dots_packed`` does. Around a layer of experts, ``experts_route`` picks the
experts of each token from their scores (its gradient: ``experts_route_backward``), ``experts_plan`` sorts the rows, and
``mx_dots_experts`` multiplies each token's row with its experts' matrices in one launch.

Operands live in GPU memory, and the work is queued on torch's current stream of their device, without waiting for it, as
torch's own calls are; workspaces come from torch's allocator for that stream. Operands in host memory (numpy arrays, torch
CPU tensors) are copied to the current GPU, and the result back: those calls return when it is there.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

from . import api
from .api import NK_BF16, NK_F16, NK_F32, NumKongAmdError, _as_tensor, _is_numpy

BLOCK = 32  # values of a row that share a scale


class _Route(ctypes.Structure):
    _fields_ = [("sigmoid", ctypes.c_int), ("renormalize", ctypes.c_int), ("scale", ctypes.c_float), ("groups", ctypes.c_int),
                ("top_groups", ctypes.c_int), ("group_top", ctypes.c_int)]


_LIB = None
_CALLS = None  # csrc/mx_calls.cpp: the calls in their ordinary form; each gives None for what is to go the general way below
_device = _stream = None  # the current device's index, a device's current stream as a number: torch's own (see _library)


def _library():
    """The shared library with the entry points of mx.h bound, and the torch module."""
    global _LIB, _CALLS, _device, _stream
    if _LIB is None:
        import torch

        _device = torch.cuda.current_device
        # (a Stream object of torch's takes 2 us to make; a product of few rows takes 8)
        _stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)

        lib = api.library()
        sz, vp, i32 = ctypes.c_uint64, ctypes.c_void_p, ctypes.c_int
        how = ctypes.POINTER(_Route)
        for name, result, arguments in (
            ("mx_quantize_async", i32, [i32, vp, sz, sz, sz, vp, sz, vp, sz, vp]),
            ("mx_dequantize_async", i32, [i32, vp, sz, vp, sz, sz, sz, vp, sz, vp]),
            ("mx_packed_size", sz, [sz, sz, sz]),
            ("mx_pack_async", i32, [vp, sz, sz, vp, sz, sz, sz, sz, sz, vp, vp]),
            ("mx_dots_workspace_size", sz, [sz, sz, sz, i32]),
            ("mx_dots_packed_async", i32, [i32, vp, sz, vp, sz, vp, i32, vp, sz, sz, sz, sz, vp, sz, vp]),
            ("experts_route_async", i32, [i32, vp, sz, sz, sz, sz, vp, how, vp, vp, vp]),
            ("experts_route_backward_async", i32, [i32, vp, sz, sz, sz, sz, how, vp, vp, vp, sz, vp]),
            ("experts_plan_size", sz, [sz, sz]),
            ("experts_plan_async", i32, [vp, sz, sz, vp, vp]),
            ("mx_experts_workspace_size", sz, [sz, sz, sz, sz, sz, i32, i32]),
            ("mx_dots_experts_async", i32, [i32, vp, sz, vp, sz, sz, vp, vp, sz, sz, sz, vp, i32, vp, sz, sz, sz, vp, sz, vp]),
        ):
            function = getattr(lib, "nk_amd_" + name)
            function.restype, function.argtypes = result, arguments
        codes = {torch.float32: NK_F32, torch.bfloat16: NK_BF16, torch.float16: NK_F16}
        _LIB = lib, torch, codes
        try:
            from .lib import _mx_calls
        except ImportError:  # built for another torch, or not at all
            _mx_calls = None
        else:
            _mx_calls.bind(*(ctypes.cast(getattr(lib, "nk_amd_" + name), ctypes.c_void_p).value for name in (
                "mx_quantize_async", "mx_dequantize_async", "mx_dots_workspace_size", "mx_dots_packed_async", "experts_route_async",
                "experts_route_backward_async", "experts_plan_size", "experts_plan_async", "mx_experts_workspace_size", "mx_dots_experts_async")))
            _mx_calls.bind_packed_size(ctypes.cast(lib.nk_amd_mx_packed_size, ctypes.c_void_p).value)
        _CALLS = _mx_calls
    return _LIB


def _check(status: int, where: str) -> None:
    if status:
        message = api.library().nk_hip_last_error()
        raise NumKongAmdError(f"{where}: {message.decode() if message else 'failed'}")


def _tensor(t, what: str):
    t = _as_tensor(t)
    if not hasattr(t, "data_ptr"):
        raise TypeError(f"{what} must be a torch.Tensor, a numpy array or export DLPack")
    return t


def _floats(t, what: str, dims: int = 2):
    """The tensor of a float operand, rows of adjacent values."""
    lib, torch, codes = _LIB or _library()
    if not isinstance(t, torch.Tensor):
        t = _tensor(t, what)
    if t.dtype not in codes:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{what} must be {dims}-dimensional, got {t.dim()} dimensions")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{what} rows must be contiguous (stride of the last dimension must be 1)")
    return t


def _row_bytes(t) -> int:
    """Bytes from one row of a matrix to the next."""
    rows, columns = t.shape
    return (t.stride(0) if rows > 1 else columns) * t.itemsize


_ROUTE = _PRODUCT = None  # what autograd knows of the calls below (torch's classes, made when the first is needed)


def _autograd():
    global _ROUTE, _PRODUCT
    if _ROUTE is None:
        import torch

        class Route(torch.autograd.Function):
            @staticmethod
            def forward(ctx, logits, top_k, score, bias, groups, top_groups, group_top, renormalize, scale):
                weights, experts = experts_route(logits, top_k, score, bias, groups, top_groups, group_top, renormalize, scale)
                ctx.save_for_backward(logits, experts)
                ctx.kind = score, renormalize, scale
                ctx.mark_non_differentiable(experts)
                return weights, experts

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, grad_weights, _):
                return (experts_route_backward(grad_weights, *ctx.saved_tensors, *ctx.kind), *[None] * 8)

        class Product(torch.autograd.Function):
            @staticmethod
            def forward(ctx, what, product, *operands):
                ctx.what = what
                return product()

            @staticmethod
            def backward(ctx, _):
                raise NumKongAmdError(f"{ctx.what} has no gradient: detach its operands, or call it under torch.no_grad()")

        _PRODUCT, _ROUTE = Product, Route


def _tracked(torch, *operands) -> bool:
    """Does autograd follow one of the operands?"""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands)


def _without_gradient(what: str, out, product, *operands):
    """The result of a product for autograd, which says so when a gradient is asked for that there is none of."""
    if out is not None:
        raise NumKongAmdError(f"{what} with out= takes no operands that require a gradient")
    _autograd()
    return _PRODUCT.apply(what, product, *operands)


def _home(*operands):
    """The index of the GPU that the operands are on, None where all are in host memory."""
    home, host = None, False
    for t in operands:
        if t is None:
            continue
        if not t.is_cuda:
            host = True
        elif home is None:
            home = t.get_device()
        elif t.get_device() != home:
            raise ValueError(f"operands are on different devices: cuda:{home} and {t.device}")
    if home is not None and host:
        raise ValueError("operands are partly in GPU memory and partly in host memory")
    return home


def _to_gpu(t):
    """An operand of host memory (a tensor, or an MxMatrix) on the current GPU."""
    import torch

    if not torch.cuda.is_available():
        raise NumKongAmdError("no GPU: this library has no CPU fallback")
    if isinstance(t, MxMatrix):
        return MxMatrix(_tensor(t.codes, "codes").cuda(), _tensor(t.scales, "scales").cuda(), t.depth)
    return None if t is None else t.cuda()


def _to_host(result, as_numpy: bool, out=None):
    """A result as a caller with operands in host memory has them: a CPU tensor, a numpy array, or in `out`."""
    if out is not None:
        _tensor(out, "out").copy_(result)
        return out
    return result.detach().cpu().numpy() if as_numpy else result.cpu()


def _new(torch, rows, columns, dtype, device):
    """A matrix of whatever (by its strides: torch.empty takes half as long again, and a call of few tokens makes several)."""
    return torch.empty_strided((rows, columns), (columns or 1, 1), dtype=dtype, device=device)


def _result(torch, out, shape, dtype, like):
    """The matrix that a call writes: `out` where one is given, else a new one."""
    if out is None:
        return _new(torch, *shape, dtype, like.device) if len(shape) == 2 else torch.empty(shape, dtype=dtype, device=like.device)
    t = _tensor(out, "out")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"out has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"out must have dtype {dtype}")
    if t.device != like.device:
        raise ValueError(f"out is on {t.device}, the operands on {like.device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("out rows must be contiguous")
    if t.dim() == 2 and t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError("out rows share memory")
    return t


def _check_host_out(out, shape, dtype):
    """What `_result` asks of an `out` in host memory."""
    if out is not None:
        t = _tensor(out, "out")
        if tuple(t.shape) != tuple(shape):
            raise ValueError(f"out has shape {tuple(t.shape)}, expected {tuple(shape)}")
        if t.dtype != dtype:
            raise TypeError(f"out must have dtype {dtype}")
        if t.is_cuda:
            raise ValueError("out is in GPU memory, the operands in host memory")


def _check_room(buffer, needed: int, what: str) -> None:
    """What a kernel finds its way in by sizes alone has to be as large as these say."""
    if not needed:
        raise ValueError(f"{what} is of sizes that are not supported")
    if buffer.nbytes < needed or not buffer.is_contiguous():
        raise ValueError(f"{what} has to be {needed} adjacent bytes for these sizes, got {buffer.nbytes}")


def _out_dtype(out, out_dtype):
    lib, torch, codes = _LIB or _library()
    if out_dtype is None:
        out_dtype = _tensor(out, "out").dtype if out is not None else torch.float32
    if out_dtype not in codes:
        raise TypeError(f"results are float32, bfloat16 or float16, not {out_dtype}")
    return out_dtype


class MxMatrix:
    """Rows of 4-bit codes and their scales: ``codes`` (..., rows, (depth + 1) // 2) uint8, the even column of a pair in the
    low half of its byte, and ``scales`` (..., rows, (depth + 31) // 32) uint8, exponents biased by 127 (255: the block is
    NaN). One leading dimension makes a stack of matrices, as ``mx_pack`` takes them for experts."""

    __slots__ = ("codes", "scales", "depth")

    def __init__(self, codes, scales, depth: int):
        import torch

        codes, scales, depth = _tensor(codes, "codes"), _tensor(scales, "scales"), int(depth)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8")
        if depth < 0:
            raise ValueError("depth must not be negative")
        if codes.dim() not in (2, 3) or scales.dim() != codes.dim() or codes.shape[:-1] != scales.shape[:-1]:
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} must have the same rows, 2 or 3 dimensions")
        if codes.shape[-1] != (depth + 1) // 2 or scales.shape[-1] != (depth + BLOCK - 1) // BLOCK:
            raise ValueError(f"depth {depth} needs {(depth + 1) // 2} bytes of codes and {(depth + BLOCK - 1) // BLOCK} scales a row, "
                             f"got {codes.shape[-1]} and {scales.shape[-1]}")
        for t, what in ((codes, "codes"), (scales, "scales")):
            if t.shape[-1] > 1 and t.stride(-1) != 1:
                raise ValueError(f"{what} rows must be contiguous")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on the same device")
        self.codes, self.scales, self.depth = codes, scales, depth

    @property
    def shape(self):
        return (*self.codes.shape[:-1], self.depth)

    @classmethod
    def _made(cls, codes, scales, depth):
        """One whose parts are known to be right."""
        matrix = cls.__new__(cls)
        matrix.codes, matrix.scales, matrix.depth = codes, scales, depth
        return matrix

    def __repr__(self):
        return f"MxMatrix(shape={tuple(self.shape)}, device={self.codes.device})"


@dataclass
class MxPackedMatrix:
    """One matrix (width x depth) or a stack of ``count`` of them, laid out for products; ``buffer`` is a uint8 tensor in GPU
    memory that holds the relocatable image."""

    count: int
    width: int
    depth: int
    buffer: "object"

    @property
    def nbytes(self) -> int:
        return int(self.buffer.numel())

    @property
    def shape(self):
        return (self.count, self.width, self.depth) if self.count != 1 else (self.width, self.depth)

    @classmethod
    def packed_size(cls, width: int, depth: int, count: int = 1) -> int:
        return int(_library()[0].nk_amd_mx_packed_size(count, width, depth))


def mx_quantize(x) -> MxMatrix:
    """The rows of ``x`` (float32, bfloat16 or float16) as 4-bit codes with a scale for each 32 values: the power of two
    that brings the block's largest magnitude into [4, 8); codes to nearest, ties to even, stopping at 6. A block that holds a
    NaN or an infinity becomes NaN. Codes and scales are whole numbers, which no gradient passes."""
    if _CALLS is not None and (made := _CALLS.quantize(x)) is not None:
        return MxMatrix._made(*made, x.shape[1])
    lib, torch, dtype_codes = _LIB or _library()
    t = _floats(x, "x")
    rows, depth = t.shape
    if not t.is_cuda:
        m = mx_quantize(_to_gpu(t))
        codes, scales = m.codes.cpu(), m.scales.cpu()
        return MxMatrix._made(codes.numpy(), scales.numpy(), depth) if _is_numpy(x) else MxMatrix._made(codes, scales, depth)
    if t.get_device() != _device():
        with torch.cuda.device(t.device):
            return mx_quantize(t)
    code_bytes, blocks = (depth + 1) // 2, (depth + BLOCK - 1) // BLOCK
    device, u8 = t.device, torch.uint8
    codes, scales = _new(torch, rows, code_bytes, u8, device), _new(torch, rows, blocks, u8, device)
    _check(lib.nk_amd_mx_quantize_async(dtype_codes[t.dtype], t.data_ptr(), rows, depth, _row_bytes(t), codes.data_ptr(), code_bytes,
                                        scales.data_ptr(), blocks, _stream(t.get_device())), "mx_quantize")
    return MxMatrix._made(codes, scales, depth)


def _matrix_of(a, what: str) -> MxMatrix:
    """An MxMatrix whose parts are tensors (mx_quantize of a numpy array has given one of arrays)."""
    if not isinstance(a, MxMatrix):
        raise TypeError(f"{what} must be an MxMatrix")
    return a if hasattr(a.codes, "data_ptr") else MxMatrix(a.codes, a.scales, a.depth)


def mx_dequantize(matrix: MxMatrix, dtype=None, out=None):
    """The values that a matrix of codes and scales stands for, in float32 (default), bfloat16 (both exact) or float16."""
    lib, torch, dtype_codes = _LIB or _library()
    if _CALLS is not None and out is None and type(matrix) is MxMatrix:
        if (made := _CALLS.dequantize(matrix.codes, matrix.scales, matrix.depth, dtype or torch.float32)) is not None:
            return made
    m = _matrix_of(matrix, "matrix")
    dtype = _out_dtype(out, dtype)
    if m.codes.dim() != 2:
        raise ValueError("mx_dequantize takes one matrix, not a stack")
    rows, depth = m.shape
    if not m.codes.is_cuda:
        _check_host_out(out, (rows, depth), dtype)
        return _to_host(mx_dequantize(_to_gpu(m), dtype), _is_numpy(matrix.codes), out)
    if m.codes.get_device() != _device():
        with torch.cuda.device(m.codes.device):
            return mx_dequantize(m, dtype, out)
    result = _result(torch, out, (rows, depth), dtype, m.codes)
    _check(lib.nk_amd_mx_dequantize_async(dtype_codes[dtype], m.codes.data_ptr(), _row_bytes(m.codes), m.scales.data_ptr(),
                                          _row_bytes(m.scales), rows, depth, result.data_ptr(), _row_bytes(result),
                                          _stream(m.codes.get_device())), "mx_dequantize")
    return result if out is None else out


def mx_pack(b) -> MxPackedMatrix:
    """Lay ``b`` out for products: an MxMatrix or floats (quantised first), width x depth, or count x width x depth for a
    stack of matrices (``mx_dots_experts``). The image is in GPU memory."""
    lib, torch, dtype_codes = _LIB or _library()
    if not isinstance(b, MxMatrix):
        b = _tensor(b, "b")
        b = _floats(b, "b", 3 if b.dim() == 3 else 2)
        rows = b if b.is_cuda else _to_gpu(b)
        flat = mx_quantize(rows.flatten(0, 1) if b.dim() == 3 else rows)
        b = MxMatrix(flat.codes.reshape(*b.shape[:-1], flat.codes.shape[-1]), flat.scales.reshape(*b.shape[:-1], flat.scales.shape[-1]), b.shape[-1])
    b = _matrix_of(b, "b")
    if not b.codes.is_cuda:
        b = _to_gpu(b)
    if b.codes.get_device() != _device():
        with torch.cuda.device(b.codes.device):
            return mx_pack(b)
    stacked = b.codes.dim() == 3
    count, width = b.codes.shape[:2] if stacked else (1, b.codes.shape[0])
    size = lib.nk_amd_mx_packed_size(count, width, b.depth)
    if size == 0:
        raise NumKongAmdError("nk_amd_mx_packed_size returned 0 (unsupported dimensions)")
    buffer = torch.empty(size, dtype=torch.uint8, device=b.codes.device)
    _check(lib.nk_amd_mx_pack_async(b.codes.data_ptr(), b.codes.stride(-2), b.codes.stride(0) if stacked else 0, b.scales.data_ptr(),
                                    b.scales.stride(-2), b.scales.stride(0) if stacked else 0, count, width, b.depth,
                                    buffer.data_ptr(), _stream(buffer.get_device())), "mx_pack")
    return MxPackedMatrix(count, width, b.depth, buffer)


def _left_operand(a, dtype_codes):
    """What a product's call says of A: (tensor, scales or None, depth, dtype code, bytes between rows of scales)."""
    if isinstance(a, MxMatrix):
        a = _matrix_of(a, "a")
        if a.codes.dim() != 2:
            raise ValueError("a must be one matrix, not a stack")
        return a.codes, a.scales, a.depth, 0, _row_bytes(a.scales)
    a = _floats(a, "a")
    return a, None, a.shape[1], dtype_codes[a.dtype], 0


def mx_dots_packed(a, packed: MxPackedMatrix, out=None, out_dtype=None):
    """``C[height x width] = a @ B.T`` with 4-bit operands and 32-bit sums. ``a``: floats, quantised on the way exactly as
    ``mx_quantize`` does, or an MxMatrix; the result is float32 (default), bfloat16 or float16 (``out_dtype``, or ``out``'s).
    There is no gradient: a backward pass through the result raises."""
    lib, torch, dtype_codes = _LIB or _library()
    if _CALLS is not None and out is None and type(packed) is MxPackedMatrix and packed.count == 1:
        values, scales, depth = (a.codes, a.scales, a.depth) if type(a) is MxMatrix else (a, None, None)
        if (made := _CALLS.dots(values, scales, depth, packed.buffer, packed.width, packed.depth, out_dtype or torch.float32)) is not None:
            return made
    if not isinstance(packed, MxPackedMatrix):
        raise TypeError("packed must be an MxPackedMatrix from mx_pack()")
    if packed.count != 1:
        raise ValueError("packed is a stack of matrices: mx_dots_experts() takes it")
    t, scales, depth, a_dtype, scales_stride = _left_operand(a, dtype_codes)
    if depth != packed.depth:
        raise ValueError(f"depth mismatch: a has {depth} columns, packed matrix has depth {packed.depth}")
    out_dtype = _out_dtype(out, out_dtype)
    height, width = t.shape[0], packed.width
    if not t.is_cuda:
        _check_host_out(out, (height, width), out_dtype)
        as_numpy = _is_numpy(a.codes if isinstance(a, MxMatrix) else a)
        return _to_host(mx_dots_packed(_to_gpu(a if isinstance(a, MxMatrix) else t), packed, None, out_dtype), as_numpy, out)
    index = t.get_device()
    if packed.buffer.get_device() != index:
        raise ValueError(f"a is on {t.device}, packed on {packed.buffer.device}")
    if _tracked(torch, t):
        return _without_gradient("mx_dots_packed", out, lambda: mx_dots_packed(a, packed, None, out_dtype), t)
    if index != _device():
        with torch.cuda.device(index):
            return mx_dots_packed(a, packed, out, out_dtype)
    _check_room(packed.buffer, lib.nk_amd_mx_packed_size(1, width, depth), "the packed image")
    result = _result(torch, out, (height, width), out_dtype, t)
    needed = lib.nk_amd_mx_dots_workspace_size(height, width, depth, scales is not None)
    workspace = torch.empty_strided((needed,), (1,), dtype=torch.uint8, device=t.device) if needed else None
    _check(lib.nk_amd_mx_dots_packed_async(
        a_dtype, t.data_ptr(), _row_bytes(t), scales.data_ptr() if scales is not None else None, scales_stride,
        packed.buffer.data_ptr(), dtype_codes[out_dtype], result.data_ptr(), _row_bytes(result), height, width, depth,
        workspace.data_ptr() if needed else None, needed, _stream(index)), "mx_dots_packed")
    return result if out is None else out


# ---- experts -------------------------------------------------------------------------------------------------------

_SCORES = {"softmax": 0, "sigmoid": 1}


def _route_kind(score, renormalize, scale, groups=1, top_groups=1, group_top=1):
    if score not in _SCORES:
        raise ValueError(f"score must be one of {sorted(_SCORES)}, got {score!r}")
    if not math.isfinite(ctypes.c_float(scale).value):
        raise ValueError("scale must be a finite 32-bit number")
    if any(not -(1 << 31) <= number < 1 << 31 for number in (groups, top_groups, group_top)):  # (ctypes would keep their low bits)
        raise ValueError("groups, top_groups and group_top must be 32-bit numbers")
    return _Route(_SCORES[score], int(bool(renormalize)), scale, groups, top_groups, group_top)


def experts_route(logits, top_k: int, score: str = "softmax", bias=None, groups: int = 1, top_groups: int = 1,
                  group_top: int = 1, renormalize: bool = True, scale: float = 1.0):
    """The ``top_k`` experts of each row of ``logits`` (tokens x experts): ``(weights, experts)``, float32 and int32, both
    tokens x top_k, the largest selection score first, ties to the lowest index.

    Scores are the row's softmax or each logit's sigmoid. Experts are selected by their logits, or by score + ``bias``
    (float32, one for each expert) where a bias is given; the weights are the scores themselves, divided by their sum over
    the chosen where ``renormalize`` is set, times ``scale``. With ``groups`` > 1 the experts stand in groups of equal size, of
    which the ``top_groups`` stay whose ``group_top`` (1 or 2) best selection scores have the largest sum (without a bias:
    the sum of logits; the sum of scores that a bias of zeros gives is another). A logit of -inf is never chosen and adds
    nothing to its group; a row with too few others in the groups that stay gets expert -1 with weight 0.

    The weights have a gradient for ``logits`` (``experts_route_backward``), which autograd follows; none for ``bias``."""
    if _CALLS is not None:
        if (made := _CALLS.route(logits, top_k, bias, _SCORES.get(score), bool(renormalize), scale, groups, top_groups, group_top)) is not None:
            return made
    lib, torch, dtype_codes = _LIB or _library()
    t = _floats(logits, "logits")
    tokens, experts = t.shape
    how = _route_kind(score, renormalize, scale, groups, top_groups, group_top)
    if bias is not None:
        bias = _tensor(bias, "bias")
        if bias.dtype != torch.float32 or tuple(bias.shape) != (experts,):
            raise ValueError(f"bias must be {experts} float32 values")
        bias = bias.contiguous()
    index = _home(t, bias)
    if index is None:
        found = experts_route(_to_gpu(t), top_k, score, _to_gpu(bias), groups, top_groups, group_top, renormalize, scale)
        return tuple(_to_host(one, _is_numpy(logits)) for one in found)
    if _tracked(torch, t):
        _autograd()
        return _ROUTE.apply(t, top_k, score, bias, groups, top_groups, group_top, renormalize, scale)
    if index != _device():
        with torch.cuda.device(index):
            return experts_route(t, top_k, score, bias, groups, top_groups, group_top, renormalize, scale)
    # (no token: the library looks at the rest before room is made for results that are refused)
    _check(lib.nk_amd_experts_route_async(dtype_codes[t.dtype], None, 0, 0, experts, top_k, None, how, None, None, None), "experts_route")
    device = t.device
    weights, chosen = _new(torch, tokens, top_k, torch.float32, device), _new(torch, tokens, top_k, torch.int32, device)
    _check(lib.nk_amd_experts_route_async(dtype_codes[t.dtype], t.data_ptr(), _row_bytes(t), tokens, experts, top_k,
                                          bias.data_ptr() if bias is not None else None, how, weights.data_ptr(), chosen.data_ptr(),
                                          _stream(index)), "experts_route")
    return weights, chosen


def experts_route_backward(grad_weights, logits, experts, score: str = "softmax", renormalize: bool = True, scale: float = 1.0):
    """The gradient of ``logits`` (their type and shape) from ``grad_weights``, that of the weights that ``experts_route``
    gave for them together with ``experts``. The selection itself has none, and neither has a bias."""
    if _CALLS is not None:
        if (made := _CALLS.route_backward(grad_weights, logits, experts, _SCORES.get(score), bool(renormalize), scale)) is not None:
            return made
    lib, torch, dtype_codes = _LIB or _library()
    t = _floats(logits, "logits")
    grad_weights, experts = _tensor(grad_weights, "grad_weights"), _tensor(experts, "experts")
    tokens, count = t.shape
    how = _route_kind(score, renormalize, scale)
    if grad_weights.dim() != 2 or grad_weights.shape != experts.shape or grad_weights.shape[0] != tokens:
        raise ValueError(f"grad_weights {tuple(grad_weights.shape)} and experts {tuple(experts.shape)} must be tokens x top_k, tokens {tokens}")
    if grad_weights.dtype != torch.float32 or experts.dtype != torch.int32:
        raise TypeError("grad_weights must be float32 and experts int32")
    index = _home(t, grad_weights, experts)
    if index is None:
        found = experts_route_backward(_to_gpu(grad_weights), _to_gpu(t), _to_gpu(experts), score, renormalize, scale)
        return _to_host(found, _is_numpy(logits))
    if index != _device():
        with torch.cuda.device(index):
            return experts_route_backward(grad_weights, t, experts, score, renormalize, scale)
    grad_weights, experts = grad_weights.contiguous(), experts.contiguous()
    result = _new(torch, tokens, count, t.dtype, t.device)
    _check(lib.nk_amd_experts_route_backward_async(
        dtype_codes[t.dtype], t.data_ptr(), _row_bytes(t), tokens, count, experts.shape[1], how, experts.data_ptr(),
        grad_weights.data_ptr(), result.data_ptr(), _row_bytes(result), _stream(index)), "experts_route_backward")
    return result


@dataclass
class ExpertsPlan:
    """The rows of each expert, for any number of ``mx_dots_experts`` calls over the same routing."""

    tokens: int
    top_k: int
    experts: int
    buffer: "object"


def experts_plan(chosen, experts: int) -> ExpertsPlan:
    """Sort the slots of ``chosen`` (tokens x top_k, int32, as ``experts_route`` gives them) by expert, keeping their order.
    Entries outside [0, ``experts``) go to no expert: -1 for padding, or experts that another process holds."""
    if _CALLS is not None and (made := _CALLS.plan(chosen, experts)) is not None:
        return ExpertsPlan(*chosen.shape, experts, made)
    lib, torch, _ = _LIB or _library()
    chosen = _tensor(chosen, "chosen")
    if chosen.dim() != 2 or chosen.dtype != torch.int32:
        raise ValueError("chosen must be a tokens x top_k matrix of int32")
    tokens, top_k = chosen.shape
    size = lib.nk_amd_experts_plan_size(tokens * top_k, experts) if 0 < experts < 1 << 32 else 0
    if size == 0:
        raise ValueError("a plan is for 1 to 1024 experts and fewer than 2^30 slots")
    if not chosen.is_cuda:
        chosen = _to_gpu(chosen)
    index = chosen.get_device()
    if index != _device():
        with torch.cuda.device(index):
            return experts_plan(chosen, experts)
    chosen = chosen.contiguous()
    buffer = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=chosen.device)
    _check(lib.nk_amd_experts_plan_async(chosen.data_ptr(), tokens * top_k, experts, buffer.data_ptr(), _stream(index)), "experts_plan")
    return ExpertsPlan(tokens, top_k, experts, buffer)


def mx_dots_experts(a, packed: MxPackedMatrix, plan: ExpertsPlan, weights=None, out=None, out_dtype=None):
    """``y[token, i] = B[expert i of the token] @ a[token]`` (tokens x top_k x width), zeros where a slot has no expert. ``a``
    has a row for each token, or one for each slot (tokens * top_k rows); floats or an MxMatrix as in ``mx_dots_packed``.
    With ``weights`` (tokens x top_k, float32) the rows of a token are summed by weight instead: tokens x width, slots without
    an expert left out. There is no gradient: a backward pass through the result raises."""
    lib, torch, dtype_codes = _LIB or _library()
    if _CALLS is not None and out is None and type(packed) is MxPackedMatrix and type(plan) is ExpertsPlan:
        values, scales, depth = (a.codes, a.scales, a.depth) if type(a) is MxMatrix else (a, None, None)
        if (made := _CALLS.experts(values, scales, depth, packed.buffer, packed.count, packed.width, packed.depth, plan.buffer, plan.tokens,
                                   plan.top_k, plan.experts, weights, out_dtype or torch.float32)) is not None:
            return made
    if not isinstance(packed, MxPackedMatrix):
        raise TypeError("packed must be an MxPackedMatrix from mx_pack()")
    if not isinstance(plan, ExpertsPlan):
        raise TypeError("plan must be an ExpertsPlan from experts_plan()")
    if packed.count != plan.experts:
        raise ValueError(f"packed holds {packed.count} matrices, the plan is for {plan.experts} experts")
    t, scales, depth, a_dtype, scales_stride = _left_operand(a, dtype_codes)
    if depth != packed.depth:
        raise ValueError(f"depth mismatch: a has {depth} columns, packed matrices have depth {packed.depth}")
    tokens, top_k, width, rows = plan.tokens, plan.top_k, packed.width, t.shape[0]
    slots = tokens * top_k
    if rows not in (tokens, slots):
        raise ValueError(f"a has {rows} rows, expected {tokens} (one for each token) or {slots} (one for each slot)")
    if weights is not None:
        weights = _tensor(weights, "weights")
        if weights.dtype != torch.float32 or tuple(weights.shape) != (tokens, top_k):
            raise ValueError(f"weights must be {tokens} x {top_k} float32 values")
    out_dtype = _out_dtype(out, out_dtype)
    shape = (tokens, width) if weights is not None else (tokens, top_k, width)
    index = _home(t, weights)
    if index is None:
        _check_host_out(out, shape, out_dtype)
        as_numpy = _is_numpy(a.codes if isinstance(a, MxMatrix) else a)
        found = mx_dots_experts(_to_gpu(a if isinstance(a, MxMatrix) else t), packed, plan, _to_gpu(weights), None, out_dtype)
        return _to_host(found, as_numpy, out)
    for buffer, what in ((packed.buffer, "packed"), (plan.buffer, "plan")):
        if buffer.get_device() != index:
            raise ValueError(f"a is on {t.device}, {what} on {buffer.device}")
    if _tracked(torch, t, weights):
        return _without_gradient("mx_dots_experts", out, lambda: mx_dots_experts(a, packed, plan, weights, None, out_dtype), t, weights)
    if index != _device():
        with torch.cuda.device(index):
            return mx_dots_experts(a, packed, plan, weights, out, out_dtype)
    _check_room(packed.buffer, lib.nk_amd_mx_packed_size(plan.experts, width, depth), "the packed image")
    _check_room(plan.buffer, lib.nk_amd_experts_plan_size(slots, plan.experts), "the plan")
    result = _result(torch, out, shape, out_dtype, t)
    if weights is not None:
        weights, stride = weights.contiguous(), _row_bytes(result)
    elif result.is_contiguous():
        stride = width * result.itemsize
    else:
        raise ValueError("out must be contiguous")
    if not slots:
        result.zero_()
        return result if out is None else out
    share, code, is_codes = top_k if rows == tokens else 1, dtype_codes[out_dtype], scales is not None
    needed = lib.nk_amd_mx_experts_workspace_size(slots, share, plan.experts, width, depth, is_codes, weights is not None)
    workspace = torch.empty_strided((needed,), (1,), dtype=torch.uint8, device=t.device) if needed else None
    _check(lib.nk_amd_mx_dots_experts_async(
        a_dtype, t.data_ptr(), _row_bytes(t), scales.data_ptr() if is_codes else None, scales_stride, share, packed.buffer.data_ptr(),
        plan.buffer.data_ptr(), slots, plan.experts, top_k, weights.data_ptr() if weights is not None else None, code,
        result.data_ptr(), stride, width, depth, workspace.data_ptr() if needed else None, needed, _stream(index)), "mx_dots_experts")
    return result if out is None else out
