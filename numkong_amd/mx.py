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
from contextlib import nullcontext
from dataclasses import dataclass

from . import api
from .api import NK_BF16, NK_F16, NK_F32, NumKongAmdError, _as_tensor, _is_numpy

BLOCK = 32  # values of a row that share a scale


class _Route(ctypes.Structure):
    _fields_ = [("sigmoid", ctypes.c_int), ("renormalize", ctypes.c_int), ("scale", ctypes.c_float), ("groups", ctypes.c_int),
                ("top_groups", ctypes.c_int), ("group_top", ctypes.c_int)]


_LIB = None


def _library():
    """The shared library with the entry points of mx.h bound, and the torch module."""
    global _LIB
    if _LIB is None:
        import torch

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
            ("mx_experts_workspace_size", sz, [sz, sz, sz, sz, sz, i32, i32, i32]),
            ("mx_dots_experts_async", i32, [i32, vp, sz, vp, sz, sz, vp, vp, sz, sz, sz, vp, i32, vp, sz, sz, sz, vp, sz, vp]),
        ):
            function = getattr(lib, "nk_amd_" + name)
            function.restype, function.argtypes = result, arguments
        codes = {torch.float32: NK_F32, torch.bfloat16: NK_BF16, torch.float16: NK_F16}
        _LIB = lib, torch, codes
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
    lib, torch, codes = _library()
    t = _tensor(t, what)
    if t.dtype not in codes:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{what} must be {dims}-dimensional, got {t.dim()} dimensions")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what} rows must be contiguous (stride of the last dimension must be 1)")
    if t.shape[0] > 1 and t.stride(0) < 0:
        raise ValueError(f"{what} rows must not run backwards")
    return t


def _row_bytes(t) -> int:
    """Bytes from one row of a matrix to the next."""
    return (t.stride(0) if t.shape[0] > 1 else t.shape[1]) * t.element_size()


def _on(device):
    """What makes `device` the current one while a call queues its work (nothing where it is)."""
    import torch

    return nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(torch, device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _home(*operands):
    """The GPU that a call runs on (where its device operands are), and whether its results go back to host memory."""
    import torch

    devices = {t.device for t in operands if t is not None and t.is_cuda}
    if len(devices) > 1:
        raise ValueError(f"operands are on different devices: {sorted(map(str, devices))}")
    if devices:
        for t in operands:
            if t is not None and not t.is_cuda:
                raise ValueError("operands are partly in GPU memory and partly in host memory")
        return devices.pop(), False
    if not torch.cuda.is_available():
        raise NumKongAmdError("no GPU: this library has no CPU fallback")
    return torch.device("cuda", torch.cuda.current_device()), True


def _given_back(result, host: bool, as_numpy: bool, out=None):
    """A result as the caller has its operands: in host memory, as a numpy array, or in `out`."""
    if out is not None:
        target = _tensor(out, "out")
        if target.data_ptr() != result.data_ptr():
            target.copy_(result)
        return out
    if host:
        result = result.cpu()
    return result.numpy() if as_numpy else result


def _result(torch, out, shape, dtype, device, host: bool):
    """The matrix that a call writes: `out` where it can be written in place, else a new one."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    t = _tensor(out, "out")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"out has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"out must have dtype {dtype}")
    if host:
        return torch.empty(shape, dtype=dtype, device=device)
    if t.device != device:
        raise ValueError(f"out is on {t.device}, the operands on {device}")
    if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("out rows must be contiguous")
    return t


def _out_dtype(out, out_dtype):
    lib, torch, codes = _library()
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

    def _to(self, device):
        return self if self.codes.device == device else MxMatrix(self.codes.to(device), self.scales.to(device), self.depth)

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


def _quantized(lib, torch, dtype_codes, x, device):
    """Codes and scales of the rows of a device matrix."""
    rows, depth = x.shape
    codes = torch.empty((rows, (depth + 1) // 2), dtype=torch.uint8, device=device)
    scales = torch.empty((rows, (depth + BLOCK - 1) // BLOCK), dtype=torch.uint8, device=device)
    _check(lib.nk_amd_mx_quantize_async(dtype_codes[x.dtype], x.data_ptr(), rows, depth, _row_bytes(x), codes.data_ptr(),
                                        codes.shape[1], scales.data_ptr(), scales.shape[1], _stream(torch, device)), "mx_quantize")
    return codes, scales


def mx_quantize(x) -> MxMatrix:
    """The rows of ``x`` (float32, bfloat16 or float16) as 4-bit codes with a scale for each 32 values: the power of two
    that brings the block's largest magnitude into [4, 8); codes to nearest, ties to even, stopping at 6. A block that holds a
    NaN or an infinity becomes NaN."""
    lib, torch, dtype_codes = _library()
    as_numpy, x = _is_numpy(x), _floats(x, "x")
    device, host = _home(x)
    with _on(device):
        codes, scales = _quantized(lib, torch, dtype_codes, x.to(device) if host else x, device)
    if host:
        codes, scales = codes.cpu(), scales.cpu()
    matrix = MxMatrix(codes, scales, x.shape[1])
    if as_numpy:
        matrix.codes, matrix.scales = matrix.codes.numpy(), matrix.scales.numpy()
    return matrix


def _matrix_of(a, what: str) -> MxMatrix:
    """An MxMatrix whose parts are tensors (one made of numpy arrays is looked at anew)."""
    if not isinstance(a, MxMatrix):
        raise TypeError(f"{what} must be an MxMatrix")
    return a if hasattr(a.codes, "data_ptr") else MxMatrix(a.codes, a.scales, a.depth)


def mx_dequantize(matrix: MxMatrix, dtype=None, out=None):
    """The values that a matrix of codes and scales stands for, in float32 (default), bfloat16 (both exact) or float16."""
    lib, torch, dtype_codes = _library()
    as_numpy = isinstance(matrix, MxMatrix) and _is_numpy(matrix.codes)
    matrix = _matrix_of(matrix, "matrix")
    dtype = _out_dtype(out, dtype)
    if matrix.codes.dim() != 2:
        raise ValueError("mx_dequantize takes one matrix, not a stack")
    device, host = _home(matrix.codes)
    rows, depth = matrix.shape
    with _on(device):
        m = matrix._to(device)
        result = _result(torch, out, (rows, depth), dtype, device, host)
        _check(lib.nk_amd_mx_dequantize_async(dtype_codes[dtype], m.codes.data_ptr(), _row_bytes(m.codes), m.scales.data_ptr(),
                                              _row_bytes(m.scales), rows, depth, result.data_ptr(), _row_bytes(result),
                                              _stream(torch, device)), "mx_dequantize")
        return _given_back(result, host, as_numpy, out)


def mx_pack(b) -> MxPackedMatrix:
    """Lay ``b`` out for products: an MxMatrix or floats (quantised first), width x depth, or count x width x depth for a
    stack of matrices (``mx_dots_experts``). The image is in GPU memory."""
    lib, torch, dtype_codes = _library()
    if not isinstance(b, MxMatrix):
        b = _tensor(b, "b")
        b = _floats(b, "b", 3 if b.dim() == 3 else 2)
        device, host = _home(b)
        b = b.to(device) if host else b
        with _on(device):
            flat = b if b.dim() == 2 else b.reshape(-1, b.shape[2])
            codes, scales = _quantized(lib, torch, dtype_codes, flat, device)
        b = MxMatrix(codes.reshape(*b.shape[:-1], -1) if codes.numel() else codes.new_empty((*b.shape[:-1], codes.shape[-1])),
                     scales.reshape(*b.shape[:-1], -1) if scales.numel() else scales.new_empty((*b.shape[:-1], scales.shape[-1])), b.shape[-1])
    b = _matrix_of(b, "b")
    device, _ = _home(b.codes)
    count, width = (1, b.codes.shape[0]) if b.codes.dim() == 2 else b.codes.shape[:2]
    size = lib.nk_amd_mx_packed_size(count, width, b.depth)
    if size == 0:
        raise NumKongAmdError("nk_amd_mx_packed_size returned 0 (unsupported dimensions)")
    with _on(device):
        b = b._to(device)
        if min(*b.codes.stride(), *b.scales.stride(), 0) < 0:
            raise ValueError("rows must not run backwards")
        stacked = b.codes.dim() == 3
        buffer = torch.empty(size, dtype=torch.uint8, device=device)
        _check(lib.nk_amd_mx_pack_async(b.codes.data_ptr(), b.codes.stride(-2), b.codes.stride(0) if stacked else 0,
                                        b.scales.data_ptr(), b.scales.stride(-2), b.scales.stride(0) if stacked else 0, count, width,
                                        b.depth, buffer.data_ptr(), _stream(torch, device)), "mx_pack")
    return MxPackedMatrix(count, width, b.depth, buffer)


def _left_operand(a, dtype_codes, what="a"):
    """What a product's call says of A: (tensor, scales or None, depth, dtype code, whether it came as numpy)."""
    if isinstance(a, MxMatrix):
        as_numpy = _is_numpy(a.codes)
        a = _matrix_of(a, what)
        if a.codes.dim() != 2:
            raise ValueError(f"{what} must be one matrix, not a stack")
        return a.codes, a.scales, a.depth, 0, as_numpy
    as_numpy, a = _is_numpy(a), _floats(a, what)
    return a, None, a.shape[1], dtype_codes[a.dtype], as_numpy


def mx_dots_packed(a, packed: MxPackedMatrix, out=None, out_dtype=None):
    """``C[height x width] = a @ B.T`` with 4-bit operands and 32-bit sums. ``a``: floats, quantised on the way exactly as
    ``mx_quantize`` does, or an MxMatrix; the result is float32 (default), bfloat16 or float16 (``out_dtype``, or ``out``'s)."""
    lib, torch, dtype_codes = _library()
    if not isinstance(packed, MxPackedMatrix):
        raise TypeError("packed must be an MxPackedMatrix from mx_pack()")
    if packed.count != 1:
        raise ValueError("packed is a stack of matrices: mx_dots_experts() takes it")
    a, scales, depth, a_dtype, as_numpy = _left_operand(a, dtype_codes)
    if depth != packed.depth:
        raise ValueError(f"depth mismatch: a has {depth} columns, packed matrix has depth {packed.depth}")
    out_dtype = _out_dtype(out, out_dtype)
    device, host = _home(a)
    if packed.buffer.device != device:
        raise ValueError(f"a is on {device}, packed on {packed.buffer.device}")
    height = a.shape[0]
    with _on(device):
        if host:
            a, scales = a.to(device), scales.to(device) if scales is not None else None
        result = _result(torch, out, (height, packed.width), out_dtype, device, host)
        needed = lib.nk_amd_mx_dots_workspace_size(height, packed.width, depth, scales is not None)
        workspace = torch.empty(needed, dtype=torch.uint8, device=device) if needed else None
        _check(lib.nk_amd_mx_dots_packed_async(
            a_dtype, a.data_ptr(), _row_bytes(a), scales.data_ptr() if scales is not None else None,
            _row_bytes(scales) if scales is not None else 0, packed.buffer.data_ptr(), dtype_codes[out_dtype], result.data_ptr(),
            _row_bytes(result), height, packed.width, depth, workspace.data_ptr() if needed else None, needed,
            _stream(torch, device)), "mx_dots_packed")
        return _given_back(result, host, as_numpy, out)


# ---- experts -------------------------------------------------------------------------------------------------------

_SCORES = {"softmax": 0, "sigmoid": 1}


def _route_kind(score, renormalize, scale, groups=1, top_groups=1, group_top=1):
    if score not in _SCORES:
        raise ValueError(f"score must be one of {sorted(_SCORES)}, got {score!r}")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    return _Route(_SCORES[score], int(bool(renormalize)), scale, groups, top_groups, group_top)


def experts_route(logits, top_k: int, score: str = "softmax", bias=None, groups: int = 1, top_groups: int = 1,
                  group_top: int = 1, renormalize: bool = True, scale: float = 1.0):
    """The ``top_k`` experts of each row of ``logits`` (tokens x experts): ``(weights, experts)``, float32 and int32, both
    tokens x top_k, the largest selection score first, ties to the lowest index.

    Scores are the row's softmax or each logit's sigmoid. Experts are selected by their logits, or by score + ``bias``
    (float32, one for each expert) where a bias is given; the weights are the scores themselves, divided by their sum over
    the chosen where ``renormalize`` is set, times ``scale``. With ``groups`` > 1 the experts stand in groups of equal size, of
    which the ``top_groups`` stay whose ``group_top`` (1 or 2) best selection scores have the largest sum (without a bias:
    the sum of logits). A logit of -inf is never chosen; a row with too few others gets expert -1 with weight 0."""
    lib, torch, dtype_codes = _library()
    as_numpy, logits = _is_numpy(logits), _floats(logits, "logits")
    tokens, experts = logits.shape
    how = _route_kind(score, renormalize, scale, groups, top_groups, group_top)
    if bias is not None:
        bias = _tensor(bias, "bias")
        if bias.dtype != torch.float32 or tuple(bias.shape) != (experts,):
            raise ValueError(f"bias must be {experts} float32 values")
    device, host = _home(logits, bias)
    with _on(device):
        if host:
            logits, bias = logits.to(device), bias.to(device) if bias is not None else None
        if bias is not None:
            bias = bias.contiguous()
        weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
        chosen = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
        _check(lib.nk_amd_experts_route_async(dtype_codes[logits.dtype], logits.data_ptr(), _row_bytes(logits), tokens, experts, top_k,
                                              bias.data_ptr() if bias is not None else None, how, weights.data_ptr(),
                                              chosen.data_ptr(), _stream(torch, device)), "experts_route")
        return _given_back(weights, host, as_numpy), _given_back(chosen, host, as_numpy)


def experts_route_backward(grad_weights, logits, experts, score: str = "softmax", renormalize: bool = True, scale: float = 1.0):
    """The gradient of ``logits`` (their type and shape) from ``grad_weights``, that of the weights that ``experts_route``
    gave for them together with ``experts``. The selection itself has none, and neither has a bias."""
    lib, torch, dtype_codes = _library()
    as_numpy, logits = _is_numpy(logits), _floats(logits, "logits")
    grad_weights, experts = _tensor(grad_weights, "grad_weights"), _tensor(experts, "experts")
    tokens, count = logits.shape
    how = _route_kind(score, renormalize, scale)
    if grad_weights.dim() != 2 or grad_weights.shape != experts.shape or grad_weights.shape[0] != tokens:
        raise ValueError(f"grad_weights {tuple(grad_weights.shape)} and experts {tuple(experts.shape)} must be tokens x top_k, tokens {tokens}")
    if grad_weights.dtype != torch.float32 or experts.dtype != torch.int32:
        raise TypeError("grad_weights must be float32 and experts int32")
    device, host = _home(logits, grad_weights, experts)
    with _on(device):
        if host:
            logits, grad_weights, experts = logits.to(device), grad_weights.to(device), experts.to(device)
        grad_weights, experts = grad_weights.contiguous(), experts.contiguous()
        result = torch.empty((tokens, count), dtype=logits.dtype, device=device)
        _check(lib.nk_amd_experts_route_backward_async(
            dtype_codes[logits.dtype], logits.data_ptr(), _row_bytes(logits), tokens, count, experts.shape[1], how,
            experts.data_ptr(), grad_weights.data_ptr(), result.data_ptr(), _row_bytes(result), _stream(torch, device)),
            "experts_route_backward")
        return _given_back(result, host, as_numpy)


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
    lib, torch, _ = _library()
    chosen = _tensor(chosen, "chosen")
    if chosen.dim() != 2 or chosen.dtype != torch.int32:
        raise ValueError("chosen must be a tokens x top_k matrix of int32")
    tokens, top_k = chosen.shape
    size = lib.nk_amd_experts_plan_size(chosen.numel(), experts) if experts > 0 else 0
    if size == 0:
        raise ValueError("a plan is for 1 to 1024 experts and fewer than 2^30 slots")
    device, host = _home(chosen)
    with _on(device):
        chosen = chosen.to(device).contiguous()
        buffer = torch.empty(size, dtype=torch.uint8, device=device)
        _check(lib.nk_amd_experts_plan_async(chosen.data_ptr(), chosen.numel(), experts, buffer.data_ptr(), _stream(torch, device)),
               "experts_plan")
    return ExpertsPlan(tokens, top_k, experts, buffer)


def mx_dots_experts(a, packed: MxPackedMatrix, plan: ExpertsPlan, weights=None, out=None, out_dtype=None):
    """``y[token, i] = B[expert i of the token] @ a[token]`` (tokens x top_k x width), zeros where a slot has no expert. ``a``
    has a row for each token, or one for each slot (tokens * top_k rows); floats or an MxMatrix as in ``mx_dots_packed``.
    With ``weights`` (tokens x top_k, float32) the rows of a token are summed by weight instead: tokens x width, slots without
    an expert left out."""
    lib, torch, dtype_codes = _library()
    if not isinstance(packed, MxPackedMatrix):
        raise TypeError("packed must be an MxPackedMatrix from mx_pack()")
    if not isinstance(plan, ExpertsPlan):
        raise TypeError("plan must be an ExpertsPlan from experts_plan()")
    if packed.count != plan.experts:
        raise ValueError(f"packed holds {packed.count} matrices, the plan is for {plan.experts} experts")
    a, scales, depth, a_dtype, as_numpy = _left_operand(a, dtype_codes)
    if depth != packed.depth:
        raise ValueError(f"depth mismatch: a has {depth} columns, packed matrices have depth {packed.depth}")
    slots, rows = plan.tokens * plan.top_k, a.shape[0]
    if rows not in (plan.tokens, slots):
        raise ValueError(f"a has {rows} rows, expected {plan.tokens} (one for each token) or {slots} (one for each slot)")
    share = plan.top_k if rows == plan.tokens else 1
    if weights is not None:
        weights = _tensor(weights, "weights")
        if weights.dtype != torch.float32 or tuple(weights.shape) != (plan.tokens, plan.top_k):
            raise ValueError(f"weights must be {plan.tokens} x {plan.top_k} float32 values")
    out_dtype = _out_dtype(out, out_dtype)
    device, host = _home(a, weights)
    for buffer, what in ((packed.buffer, "packed"), (plan.buffer, "plan")):
        if buffer.device != device:
            raise ValueError(f"a is on {device}, {what} on {buffer.device}")
    shape = (plan.tokens, packed.width) if weights is not None else (plan.tokens, plan.top_k, packed.width)
    with _on(device):
        if host:
            a, scales = a.to(device), scales.to(device) if scales is not None else None
            weights = weights.to(device) if weights is not None else None
        if weights is not None:
            weights = weights.contiguous()
        result = _result(torch, out, shape, out_dtype, device, host)
        if weights is None and not result.is_contiguous():
            raise ValueError("out must be contiguous")
        if not slots:
            return _given_back(result.zero_(), host, as_numpy, out)
        flat = result if weights is not None else result.view(slots, packed.width)
        code = dtype_codes[out_dtype]
        needed = lib.nk_amd_mx_experts_workspace_size(slots, share, plan.experts, packed.width, depth, scales is not None, code,
                                                      weights is not None)
        workspace = torch.empty(needed, dtype=torch.uint8, device=device) if needed else None
        _check(lib.nk_amd_mx_dots_experts_async(
            a_dtype, a.data_ptr(), _row_bytes(a), scales.data_ptr() if scales is not None else None,
            _row_bytes(scales) if scales is not None else 0, share, packed.buffer.data_ptr(), plan.buffer.data_ptr(), slots,
            plan.experts, plan.top_k, weights.data_ptr() if weights is not None else None, code, flat.data_ptr(), _row_bytes(flat),
            packed.width, depth, workspace.data_ptr() if needed else None, needed, _stream(torch, device)), "mx_dots_experts")
        return _given_back(result, host, as_numpy, out)
