"""The dense feed-forward layer: the Python side of ``include/numkong_amd/dense.h``.

``rms_norm`` adds the residual and norms the rows, ``linear`` multiplies with a matrix of weights and adds bias, activation and residual
as it writes the result, ``gated_linear`` does both products of a gated layer at once. Matrices are plain tensors of bfloat16 or float16, with
gradients that autograd follows, or 8-bit ones: an ``Mx8Matrix`` has e4m3 codes with one power of two for each 32 values of a
row. ``mx8_quantize`` makes one, ``rms_norm_mx8`` gives its result as one, and a product with 8-bit weights quantises its activations on the way.

Operands live in GPU memory, and the work is queued on torch's current stream of their device, without waiting for it, as
torch's own calls are; workspaces come from torch's allocator for that stream. Operands in host memory (numpy arrays, torch
CPU tensors) are copied to the current GPU, and the result back: those calls return when it is there. There are no forward-mode
derivatives: operands with a tangent are refused.
"""
from __future__ import annotations

import ctypes

from . import mx
from .api import NK_BF16, NK_E4M3, NK_F16, NK_F32, NumKongAmdError, _is_numpy
from .mx import _check, _check_host_out, _floats, _home, _no_tangent, _result, _row_bytes, _tensor, _to_host, _tracked

BLOCK = 32  # values of a row that share a scale
ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}

_vp, _sz, _i32 = ctypes.c_void_p, ctypes.c_uint64, ctypes.c_int


class _RmsNorm(ctypes.Structure):
    _fields_ = [("rows", _sz), ("depth", _sz), ("eps", ctypes.c_float), ("dtype", _i32), ("x", _vp), ("x_stride", _sz), ("residual", _vp),
                ("residual_stride", _sz), ("total", _vp), ("total_stride", _sz), ("weight_dtype", _i32), ("weight", _vp), ("y_dtype", _i32),
                ("y", _vp), ("y_stride", _sz), ("y_scales", _vp), ("y_scales_stride", _sz)]


class _RmsNormBackward(ctypes.Structure):
    _fields_ = [("rows", _sz), ("depth", _sz), ("eps", ctypes.c_float), ("dtype", _i32), ("total", _vp), ("total_stride", _sz),
                ("weight_dtype", _i32), ("weight", _vp), ("grad_dtype", _i32), ("grad", _vp), ("grad_stride", _sz), ("grad_total", _vp),
                ("grad_total_stride", _sz), ("grad_x", _vp), ("grad_x_stride", _sz), ("grad_weight", _vp)]


class _Linear(ctypes.Structure):
    _fields_ = [("height", _sz), ("width", _sz), ("depth", _sz), ("gated", _i32), ("a_dtype", _i32), ("a", _vp), ("a_stride", _sz), ("a_scales", _vp),
                ("a_scales_stride", _sz), ("w_dtype", _i32), ("w", _vp), ("w_stride", _sz), ("w_scales", _vp), ("w_scales_stride", _sz),
                ("w_up", _vp), ("w_up_stride", _sz), ("w_up_scales", _vp), ("w_up_scales_stride", _sz), ("activation", _i32),
                ("bias_dtype", _i32), ("bias", _vp), ("residual_dtype", _i32), ("residual", _vp), ("residual_stride", _sz), ("c_dtype", _i32),
                ("c", _vp), ("c_stride", _sz), ("pre", _vp), ("pre_up", _vp), ("pre_stride", _sz)]


class _LinearBackward(ctypes.Structure):
    _fields_ = [("height", _sz), ("width", _sz), ("depth", _sz), ("gated", _i32), ("dtype", _i32), ("a", _vp), ("a_stride", _sz), ("w", _vp), ("w_stride", _sz),
                ("w_up", _vp), ("w_up_stride", _sz), ("activation", _i32), ("pre", _vp), ("pre_up", _vp), ("pre_stride", _sz),
                ("grad_dtype", _i32), ("grad", _vp), ("grad_stride", _sz), ("grad_a", _vp), ("grad_a_stride", _sz), ("grad_w", _vp),
                ("grad_w_stride", _sz), ("grad_w_up", _vp), ("grad_w_up_stride", _sz), ("bias_dtype", _i32), ("grad_bias", _vp)]


_LIB = None
_CALLS = None  # csrc/dense_calls.cpp: the calls in their ordinary form; each gives None for what is to go the general way below


def _library():
    """The shared library with the entry points of dense.h bound, the torch module, and the codes of its float types."""
    global _LIB, _CALLS
    if _LIB is None:
        lib, torch, codes = mx._library()
        of = ctypes.POINTER
        functions = (
            ("mx8_quantize_async", _i32, [_i32, _vp, _sz, _sz, _sz, _vp, _sz, _vp, _sz, _vp]),
            ("mx8_dequantize_async", _i32, [_i32, _vp, _sz, _vp, _sz, _sz, _sz, _vp, _sz, _vp]),
            ("rms_norm_async", _i32, [of(_RmsNorm), _vp]),
            ("rms_norm_backward_workspace_size", _sz, [of(_RmsNormBackward)]),
            ("rms_norm_backward_async", _i32, [of(_RmsNormBackward), _vp, _sz, _vp]),
            ("linear_workspace_size", _sz, [of(_Linear)]),
            ("linear_async", _i32, [of(_Linear), _vp, _sz, _vp]),
            ("linear_backward_workspace_size", _sz, [of(_LinearBackward)]),
            ("linear_backward_async", _i32, [of(_LinearBackward), _vp, _sz, _vp]),
        )
        for name, result, arguments in functions:
            function = getattr(lib, "nk_amd_" + name)
            function.restype, function.argtypes = result, arguments
        _LIB = lib, torch, codes
        try:
            from .lib import _dense_calls
        except ImportError:  # built for another torch, or not at all
            _dense_calls = None
        else:
            _dense_calls.bind(*(ctypes.cast(getattr(lib, name), _vp).value for name in (*("nk_amd_" + name for name, *_ in functions), "nk_hip_last_error")))
        _CALLS = _dense_calls
    return _LIB


def _workspace(torch, needed: int, device):
    return torch.empty_strided((needed,), (1,), dtype=torch.uint8, device=device) if needed else None


def _address(t):
    return None if t is None else t.data_ptr()


def _to_gpu(t):
    """An operand of host memory on the current GPU."""
    import torch

    if not torch.cuda.is_available():
        raise NumKongAmdError("no GPU: this library has no CPU fallback")
    if isinstance(t, Mx8Matrix):
        return Mx8Matrix(t.codes.cuda(), t.scales.cuda())
    return None if t is None else t.cuda()


def _vector(t, length: int, what: str):
    """A float vector of so many adjacent values, or None."""
    if t is None:
        return None
    lib, torch, codes = _library()
    t = _tensor(t, what)
    if t.dtype not in codes:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    if tuple(t.shape) != (length,):
        raise ValueError(f"{what} must have shape ({length},), got {tuple(t.shape)}")
    return t.contiguous()


def _rows_of(t):
    """A gradient as the kernels read it: autograd hands on expanded and transposed ones too."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


class Mx8Matrix:
    """Rows of 8-bit floats with a power of two for each 32: ``codes`` (rows, depth) float8_e4m3fn (or uint8, taken as such) and
    ``scales`` (rows, (depth + 31) // 32) uint8, exponents biased by 127 (255: the block is NaN). Rows of either may be strided."""

    __slots__ = ("codes", "scales")

    def __init__(self, codes, scales):
        import torch

        codes, scales = _tensor(codes, "codes"), _tensor(scales, "scales")
        if codes.dtype == torch.uint8:
            codes = codes.view(torch.float8_e4m3fn)
        if codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.uint8:
            raise TypeError("codes must be float8_e4m3fn or uint8, and scales uint8")
        if codes.dim() != 2 or scales.dim() != 2 or scales.shape != (codes.shape[0], (codes.shape[1] + BLOCK - 1) // BLOCK):
            raise ValueError(f"codes {tuple(codes.shape)} (2 dimensions) need a scale for each {BLOCK} values of a row, got scales {tuple(scales.shape)}")
        for t, what in ((codes, "codes"), (scales, "scales")):
            if t.shape[-1] > 1 and t.stride(-1) != 1:
                raise ValueError(f"{what} rows must be contiguous")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on the same device")
        self.codes, self.scales = codes, scales

    @property
    def shape(self):
        return tuple(self.codes.shape)

    @property
    def device(self):
        return self.codes.device

    @property
    def is_cuda(self):
        return self.codes.is_cuda

    def get_device(self):
        return self.codes.get_device()

    @classmethod
    def _made(cls, codes, scales):
        """One whose parts are known to be right."""
        matrix = cls.__new__(cls)
        matrix.codes, matrix.scales = codes, scales
        return matrix

    @classmethod
    def _empty(cls, torch, rows: int, depth: int, device):
        """Room for one; rows start where the products can read them in place."""
        blocks = (depth + BLOCK - 1) // BLOCK
        return cls._made(torch.empty_strided((rows, depth), (max((depth + 15) // 16 * 16, 1), 1), dtype=torch.float8_e4m3fn, device=device),
                         torch.empty_strided((rows, blocks), (max((blocks + 3) // 4 * 4, 1), 1), dtype=torch.uint8, device=device))

    def cpu(self) -> "Mx8Matrix":
        return Mx8Matrix(self.codes.cpu().contiguous(), self.scales.cpu().contiguous())

    def __repr__(self):
        return f"Mx8Matrix(shape={self.shape}, device={self.codes.device})"


def mx8_quantize(x) -> Mx8Matrix:
    """The rows of ``x`` (float32, bfloat16 or float16) as e4m3 codes with a scale for each 32 values: the smallest power of two
    (not below 2^-127) that keeps the block's largest magnitude within 448; codes to nearest, ties to even. A block that holds a NaN
    or an infinity becomes NaN. Codes and scales are numbers that no gradient passes."""
    lib, torch, dtype_codes = _library()
    if _CALLS is not None and (made := _CALLS.quantize(x)) is not None:
        return Mx8Matrix._made(*made)
    t = _floats(x, "x")
    if not t.is_cuda:
        return mx8_quantize(_to_gpu(t)).cpu()
    index = t.get_device()
    if index != mx._device():
        with torch.cuda.device(index):
            return mx8_quantize(t)
    rows, depth = t.shape
    m = Mx8Matrix._empty(torch, rows, depth, t.device)
    _check(lib.nk_amd_mx8_quantize_async(dtype_codes[t.dtype], t.data_ptr(), rows, depth, _row_bytes(t), m.codes.data_ptr(), _row_bytes(m.codes),
                                         m.scales.data_ptr(), _row_bytes(m.scales), mx._stream(index)), "mx8_quantize")
    return m


def mx8_dequantize(matrix: Mx8Matrix, dtype=None, out=None):
    """The values that codes and scales stand for, in float32 (default), bfloat16 (both exact, but for what is below their range)
    or float16."""
    lib, torch, dtype_codes = _library()
    if not isinstance(matrix, Mx8Matrix):
        raise TypeError("matrix must be an Mx8Matrix")
    if _CALLS is not None and out is None and (made := _CALLS.dequantize(matrix.codes, matrix.scales, dtype)) is not None:
        return made
    dtype = mx._out_dtype(out, dtype)
    if not matrix.is_cuda:
        _check_host_out(out, matrix.shape, dtype)
        return _to_host(mx8_dequantize(_to_gpu(matrix), dtype), False, out)
    index = matrix.get_device()
    if index != mx._device():
        with torch.cuda.device(index):
            return mx8_dequantize(matrix, dtype, out)
    rows, depth = matrix.shape
    result = _result(torch, out, (rows, depth), dtype, matrix.codes)
    _check(lib.nk_amd_mx8_dequantize_async(dtype_codes[dtype], matrix.codes.data_ptr(), _row_bytes(matrix.codes), matrix.scales.data_ptr(),
                                           _row_bytes(matrix.scales), rows, depth, result.data_ptr(), _row_bytes(result), mx._stream(index)), "mx8_dequantize")
    return result if out is None else out


_NORM = _LINEAR = _GATED = None  # what autograd knows of the calls below (torch's classes, made when the first is needed)


def _autograd():
    global _NORM, _LINEAR, _GATED
    if _NORM is None:
        import torch

        once = torch.autograd.function.once_differentiable

        class Norm(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, weight, residual, eps, out_dtype):
                ctx.set_materialize_grads(False)
                found = rms_norm(x, weight, residual, eps, out_dtype)
                ctx.save_for_backward(x if residual is None else found[1], weight)
                ctx.eps = eps
                return found

            @staticmethod
            @once
            def backward(ctx, grad, grad_total=None):
                total, weight = ctx.saved_tensors
                of_x, of_weight, of_residual = ctx.needs_input_grad[:3]
                if grad is None:  # nothing came back through y
                    found = grad_total, torch.zeros_like(weight) if of_weight else None
                else:
                    found = rms_norm_backward(_rows_of(grad), total, weight, None if grad_total is None else _rows_of(grad_total), ctx.eps, of_weight)
                return found[0] if of_x else None, found[1] if of_weight else None, found[0] if of_residual else None, None, None

        class Linear(torch.autograd.Function):
            @staticmethod
            def forward(ctx, a, w, bias, activation, residual, out_dtype):
                # (a gradient of the residual alone does without the sums)
                keeps = activation is not None and any(ctx.needs_input_grad[:3])
                found = linear(a, w, bias, activation, residual, out_dtype=out_dtype, sums=keeps)
                y, sums = found if keeps else (found, None)
                ctx.save_for_backward(a, w, sums)
                ctx.kind = activation, None if bias is None else bias.dtype, None if residual is None else residual.dtype
                return y

            @staticmethod
            @once
            def backward(ctx, grad):
                a, w, sums = ctx.saved_tensors
                activation, bias_dtype, residual_dtype = ctx.kind
                of_a, of_w, of_bias, _, of_residual, _ = ctx.needs_input_grad
                found = None, None, None
                if of_a or of_w or of_bias:
                    found = linear_backward(_rows_of(grad), a, w, sums, activation, of_a, of_w, bias_dtype if of_bias else None)
                return (*found, None, grad.to(residual_dtype) if of_residual else None, None)

        class Gated(torch.autograd.Function):
            @staticmethod
            def forward(ctx, a, gate, up, activation, out_dtype):
                y, *sums = gated_linear(a, gate, up, activation, out_dtype=out_dtype, sums=True)
                ctx.save_for_backward(a, gate, up, *sums)
                ctx.activation = activation
                return y

            @staticmethod
            @once
            def backward(ctx, grad):
                return (*gated_linear_backward(_rows_of(grad), *ctx.saved_tensors, ctx.activation, *ctx.needs_input_grad[:3]), None, None)

        _LINEAR, _GATED, _NORM = Linear, Gated, Norm


# ---- the norm ------------------------------------------------------------------------------------------------------


def _norm_operands(x, weight, residual, eps):
    lib, torch, dtype_codes = _library()
    t = _floats(x, "x")
    weight = _vector(weight, t.shape[1], "weight")
    if residual is not None:
        residual = _floats(residual, "residual")
        if residual.shape != t.shape or residual.dtype != t.dtype:
            raise ValueError(f"residual must be {tuple(t.shape)} of {t.dtype} as x is, got {tuple(residual.shape)} of {residual.dtype}")
    return t, weight, residual, _eps(eps)


def _eps(eps) -> float:
    eps = ctypes.c_float(eps).value
    if not 0 <= eps < float("inf"):
        raise ValueError("eps must be a finite 32-bit number that is not negative")
    return eps


def _norm(t, weight, residual, eps, y, y_dtype, scales, where):
    """Queues the norm of operands on the current GPU into `y`; the total, or None without a residual."""
    lib, torch, dtype_codes = _library()
    rows, depth = t.shape
    total = None if residual is None else mx._new(torch, rows, depth, t.dtype, t.device)
    n = _RmsNorm(rows, depth, eps, dtype_codes[t.dtype], t.data_ptr(), _row_bytes(t), _address(residual),
                 0 if residual is None else _row_bytes(residual), _address(total), 0 if total is None else _row_bytes(total),
                 0 if weight is None else dtype_codes[weight.dtype], _address(weight), y_dtype, y.data_ptr(), _row_bytes(y), _address(scales),
                 0 if scales is None else _row_bytes(scales))
    _check(lib.nk_amd_rms_norm_async(n, mx._stream(t.get_device())), where)
    return total


def rms_norm(x, weight=None, residual=None, eps: float = 1e-6, out_dtype=None):
    """``y = t * weight / sqrt(mean(t^2) + eps)`` of each row of ``t = x + residual``, in ``out_dtype`` (default: ``x``'s type).
    Without a residual the result is ``y``; with one it is ``(y, t)``, ``t`` rounded to ``x``'s type, and what is normed is ``t`` as it is
    returned. ``x`` and ``residual``: rows x depth of one float type, depth at most 32768; ``weight``: depth values of any.

    The results have gradients (``rms_norm_backward``), which autograd follows."""
    lib, torch, dtype_codes = _LIB or _library()
    if _CALLS is not None and (made := _CALLS.norm(x, weight, residual, eps, out_dtype, False)) is not None:
        return made[0] if residual is None else (made[0], made[2])
    t, weight, residual, eps = _norm_operands(x, weight, residual, eps)
    out_dtype = t.dtype if out_dtype is None else mx._out_dtype(None, out_dtype)
    index = _home(t, weight, residual)
    if index is None:
        found = rms_norm(_to_gpu(t), _to_gpu(weight), _to_gpu(residual), eps, out_dtype)
        return _to_host(found, _is_numpy(x)) if residual is None else tuple(_to_host(one, _is_numpy(x)) for one in found)
    if _tracked(torch, t, weight, residual):
        _autograd()
        return _NORM.apply(t, weight, residual, eps, out_dtype)
    if index != mx._device():
        with torch.cuda.device(index):
            return rms_norm(t, weight, residual, eps, out_dtype)
    y = mx._new(torch, *t.shape, out_dtype, t.device)
    total = _norm(t, weight, residual, eps, y, dtype_codes[out_dtype], None, "rms_norm")
    return y if residual is None else (y, total)


def rms_norm_mx8(x, weight=None, residual=None, eps: float = 1e-6):
    """``rms_norm`` with ``y`` as an ``Mx8Matrix``: the codes and scales of the exact values, not of values that were rounded before.
    There is no gradient: operands that require one are refused while autograd records."""
    lib, torch, dtype_codes = _LIB or _library()
    if _CALLS is not None and (made := _CALLS.norm(x, weight, residual, eps, None, True)) is not None:
        y = Mx8Matrix._made(*made[:2])
        return y if residual is None else (y, made[2])
    t, weight, residual, eps = _norm_operands(x, weight, residual, eps)
    index = _home(t, weight, residual)
    if _tracked(torch, t, weight, residual):
        raise NumKongAmdError("rms_norm_mx8 has no gradient: detach its operands, or call it under torch.no_grad()")
    if index is None:
        found = rms_norm_mx8(_to_gpu(t), _to_gpu(weight), _to_gpu(residual), eps)
        return found.cpu() if residual is None else (found[0].cpu(), _to_host(found[1], _is_numpy(x)))
    if index != mx._device():
        with torch.cuda.device(index):
            return rms_norm_mx8(t, weight, residual, eps)
    y = Mx8Matrix._empty(torch, *t.shape, t.device)
    total = _norm(t, weight, residual, eps, y.codes, NK_E4M3, y.scales, "rms_norm_mx8")
    return y if residual is None else (y, total)


def rms_norm_backward(grad, total, weight=None, grad_total=None, eps: float = 1e-6, need_weight: bool = True):
    """The gradients ``(of x, of weight)`` from ``grad``, that of ``y``: ``total`` is what was normed (``x``, or the sum that ``rms_norm``
    returned), ``grad_total`` the gradient that the sum has got from elsewhere. That of the residual is that of ``x``. The second is
    None without a ``weight``, or where it is not needed. Autograd does not follow this call."""
    lib, torch, dtype_codes = _LIB or _library()
    if _CALLS is not None and (made := _CALLS.norm_backward(grad, total, weight, grad_total, eps, need_weight)) is not None:
        return made
    t, g = _floats(total, "total"), _floats(grad, "grad")
    weight, eps = _vector(weight, t.shape[1], "weight"), _eps(eps)
    if g.shape != t.shape:
        raise ValueError(f"grad {tuple(g.shape)} and total {tuple(t.shape)} must have the same shape")
    if grad_total is not None:
        grad_total = _floats(grad_total, "grad_total")
        if grad_total.shape != t.shape or grad_total.dtype != t.dtype:
            raise ValueError(f"grad_total must be {tuple(t.shape)} of {t.dtype} as total is")
    _no_tangent(torch, g, t, weight, grad_total)
    index = _home(g, t, weight, grad_total)
    if index is None:
        found = rms_norm_backward(_to_gpu(g), _to_gpu(t), _to_gpu(weight), _to_gpu(grad_total), eps, need_weight)
        return tuple(None if one is None else _to_host(one, _is_numpy(total)) for one in found)
    if index != mx._device():
        with torch.cuda.device(index):
            return rms_norm_backward(g, t, weight, grad_total, eps, need_weight)
    rows, depth = t.shape
    of_x = mx._new(torch, rows, depth, t.dtype, t.device)
    of_weight = torch.empty((depth,), dtype=weight.dtype, device=t.device) if need_weight and weight is not None else None
    n = _RmsNormBackward(rows, depth, eps, dtype_codes[t.dtype], t.data_ptr(), _row_bytes(t), 0 if weight is None else dtype_codes[weight.dtype],
                         _address(weight), dtype_codes[g.dtype], g.data_ptr(), _row_bytes(g), _address(grad_total),
                         0 if grad_total is None else _row_bytes(grad_total), of_x.data_ptr(), _row_bytes(of_x), _address(of_weight))
    needed = lib.nk_amd_rms_norm_backward_workspace_size(n)
    workspace = _workspace(torch, needed, t.device)
    _check(lib.nk_amd_rms_norm_backward_async(n, _address(workspace), needed, mx._stream(index)), "rms_norm_backward")
    return of_x, of_weight


# ---- products ------------------------------------------------------------------------------------------------------


def _activation(kind):
    if kind not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {kind!r}")
    return ACTIVATIONS[kind]


def _matrix(w, what: str):
    """A matrix of weights: 16 bits, or an Mx8Matrix."""
    if isinstance(w, Mx8Matrix):
        return w
    lib, torch, _ = _library()
    w = _floats(w, what)
    if w.dtype == torch.float32:
        raise TypeError(f"{what} must be bfloat16, float16 or an Mx8Matrix, got {w.dtype}")
    return w


def _left(a, w):
    """The left operand for a matrix of weights."""
    if isinstance(a, Mx8Matrix):
        if not isinstance(w, Mx8Matrix):
            raise TypeError("a is an Mx8Matrix, the matrix of weights is not")
    else:
        a = _floats(a, "a")
        if not isinstance(w, Mx8Matrix) and a.dtype != w.dtype:
            raise TypeError(f"a has dtype {a.dtype}, the matrix of weights {w.dtype}")
    if a.shape[1] != w.shape[1]:
        raise ValueError(f"depth mismatch: a has {a.shape[1]} columns, the matrix of weights {w.shape[1]}")
    return a


def _product_dtype(a, w, out, out_dtype, sums):
    """The type of a product's results: A's, or bfloat16 where A is 8-bit or 32-bit and W 8-bit."""
    lib, torch, dtype_codes = _library()
    eight = isinstance(w, Mx8Matrix)
    if eight and sums:
        raise TypeError("sums are given by products of 16-bit matrices: those of 8-bit ones have no gradient, and not the bits of float32")
    if out_dtype is None and out is None:
        return torch.bfloat16 if isinstance(a, Mx8Matrix) or a.dtype == torch.float32 else a.dtype
    out_dtype = mx._out_dtype(out, out_dtype)
    if eight and out_dtype == torch.float32:
        raise TypeError("products of 8-bit matrices give bfloat16 or float16")
    return out_dtype


def _operand(m, codes):
    """(dtype, address, stride, address of scales, their stride) of an operand."""
    if m is None:
        return 0, None, 0, None, 0
    if isinstance(m, Mx8Matrix):
        return NK_E4M3, m.codes.data_ptr(), _row_bytes(m.codes), m.scales.data_ptr(), _row_bytes(m.scales)
    return codes[m.dtype], m.data_ptr(), _row_bytes(m), None, 0


def _rows_in_memory(t):
    """(address, rows, bytes from one to the next, bytes of one) of a vector or matrix."""
    rows = t.shape[0] if t.dim() == 2 else 1
    return t.data_ptr(), rows, _row_bytes(t) if t.dim() == 2 else 0, t.shape[-1] * t.itemsize


def _share_memory(x, y) -> bool:
    """Do two operands have bytes in common? (Rows that lie between one another's, at one distance, have none.)"""
    if not x.numel() or not y.numel():
        return False
    (x0, x_rows, x_step, x_size), (y0, y_rows, y_step, y_size) = _rows_in_memory(x), _rows_in_memory(y)
    if x0 + (x_rows - 1) * x_step + x_size <= y0 or y0 + (y_rows - 1) * y_step + y_size <= x0:
        return False
    if x_step != y_step or x_step < max(x_size, y_size):
        return True
    return (y0 - x0) % x_step < x_size or (x0 - y0) % x_step < y_size


def _check_out_alone(out, residual, **operands):
    """A result may be its residual, but no other operand: workgroups read those at any time."""
    if residual is not None and _share_memory(out, residual) and (out.data_ptr(), out.dtype, _row_bytes(out)) != (residual.data_ptr(), residual.dtype, _row_bytes(residual)):
        raise ValueError("out shares memory with residual, but is not residual itself")
    for name, m in operands.items():
        for t in (m.codes, m.scales) if isinstance(m, Mx8Matrix) else () if m is None else (m,):
            if _share_memory(out, t):
                raise ValueError(f"out shares memory with {name}")


def _parts(m):
    """An operand and its scales, if it has any."""
    return (m.codes, m.scales) if type(m) is Mx8Matrix else (m, None)


def _multiply(a, w, w_up, bias, activation, residual, out, out_dtype, sums, where):
    """Queues a product of operands on the current GPU: (result, [sums])."""
    lib, torch, dtype_codes = _library()
    height, depth = a.shape
    width, device = w.shape[0], a.device
    like = a.codes if isinstance(a, Mx8Matrix) else a
    result = _result(torch, out, (height, width), out_dtype, like)
    if out is not None:
        _check_out_alone(result, residual, a=a, w=w, w_up=w_up, bias=bias)
    kept = [mx._new(torch, height, width, torch.float32, device) for _ in range(0 if not sums else 1 if w_up is None else 2)]
    l = _Linear(height, width, depth, w_up is not None, *_operand(a, dtype_codes), *_operand(w, dtype_codes), *_operand(w_up, dtype_codes)[1:], activation,
                0 if bias is None else dtype_codes[bias.dtype], _address(bias), 0 if residual is None else dtype_codes[residual.dtype],
                _address(residual), 0 if residual is None else _row_bytes(residual), dtype_codes[out_dtype], result.data_ptr(), _row_bytes(result),
                kept[0].data_ptr() if kept else None, kept[1].data_ptr() if len(kept) > 1 else None, width * 4 if kept else 0)
    needed = lib.nk_amd_linear_workspace_size(l)
    workspace = _workspace(torch, needed, device)
    _check(lib.nk_amd_linear_async(l, _address(workspace), needed, mx._stream(like.get_device())), where)
    return (result if out is None else out), kept


def _eight_bits(where, *operands):
    lib, torch, _ = _library()
    if _tracked(torch, *(t for t in operands if not isinstance(t, Mx8Matrix))):
        raise NumKongAmdError(f"{where} with 8-bit weights has no gradient: detach its operands, or call it under torch.no_grad()")


def linear(a, w, bias=None, activation=None, residual=None, out=None, out_dtype=None, sums: bool = False):
    """``activation(a @ w.T + bias) + residual`` in one pass over the results, 32-bit sums. ``a`` (height x depth) and ``w`` (width x depth)
    are bfloat16 or float16 alike, or ``w`` is an ``Mx8Matrix`` and ``a`` is one too, or floats that are quantised on the way exactly as
    ``mx8_quantize`` does. ``activation``: None, "relu", "silu", "gelu" (erf's) or "gelu_tanh"; ``bias`` (width) and ``residual`` (height x
    width) are floats of any type. The result has ``out_dtype`` (or ``out``'s; default: ``a``'s type), 16 bits where ``w`` is 8-bit;
    ``out`` may be the residual itself, and shares memory with no other operand.

    16-bit products have gradients for ``a``, ``w``, ``bias`` and ``residual``, which autograd follows; 8-bit ones have none and refuse
    operands that require one while autograd records. With ``sums`` (16-bit) the result is ``(y, a @ w.T + bias)``, as ``linear_backward`` takes them."""
    lib, torch, dtype_codes = _LIB or _library()
    if _CALLS is not None and out is None:
        if (made := _CALLS.linear(*_parts(a), *_parts(w), None, None, bias, ACTIVATIONS.get(activation), residual, out_dtype, sums)) is not None:
            return made[:2] if sums else made[0]
    w = _matrix(w, "w")
    t = _left(a, w)
    height, width, code = t.shape[0], w.shape[0], _activation(activation)
    bias = _vector(bias, width, "bias")
    if residual is not None:
        residual = _floats(residual, "residual")
        if tuple(residual.shape) != (height, width):
            raise ValueError(f"residual must have shape {(height, width)}, got {tuple(residual.shape)}")
    out_dtype = _product_dtype(t, w, out, out_dtype, sums)
    index = _home(t, w, bias, residual)
    if index is None:
        _check_host_out(out, (height, width), out_dtype)
        found = linear(_to_gpu(t), _to_gpu(w), _to_gpu(bias), activation, _to_gpu(residual), None, out_dtype, sums)
        as_numpy = _is_numpy(a)
        return (_to_host(found[0], as_numpy, out), _to_host(found[1], as_numpy)) if sums else _to_host(found, as_numpy, out)
    if isinstance(w, Mx8Matrix):
        _eight_bits("linear", t, bias, residual)
    elif _tracked(torch, t, w, bias, residual):
        if out is not None or sums:
            raise NumKongAmdError("linear with out= or sums= takes no operands that require a gradient")
        _autograd()
        return _LINEAR.apply(t, w, bias, activation, residual, out_dtype)
    if index != mx._device():
        with torch.cuda.device(index):
            return linear(t, w, bias, activation, residual, out, out_dtype, sums)
    result, kept = _multiply(t, w, None, bias, code, residual, out, out_dtype, sums, "linear")
    return (result, *kept) if sums else result


def gated_linear(a, w_gate, w_up, activation="silu", out=None, out_dtype=None, sums: bool = False):
    """``activation(a @ w_gate.T) * (a @ w_up.T)``, both products in one kernel. Operands, types and gradients as in ``linear``; the two
    matrices have one type and shape. With ``sums`` (16-bit) the result is ``(y, a @ w_gate.T, a @ w_up.T)``, as ``gated_linear_backward`` takes them."""
    lib, torch, dtype_codes = _LIB or _library()
    if _CALLS is not None and out is None and w_up is not None:
        if (made := _CALLS.linear(*_parts(a), *_parts(w_gate), *_parts(w_up), None, ACTIVATIONS.get(activation), None, out_dtype, sums)) is not None:
            return made if sums else made[0]
    gate, up = _matrix(w_gate, "w_gate"), _matrix(w_up, "w_up")
    if gate.shape != up.shape or isinstance(gate, Mx8Matrix) != isinstance(up, Mx8Matrix) or getattr(gate, "dtype", None) != getattr(up, "dtype", None):
        raise ValueError("w_gate and w_up must have the same shape and type")
    t, code = _left(a, gate), _activation(activation)
    out_dtype = _product_dtype(t, gate, out, out_dtype, sums)
    shape = t.shape[0], gate.shape[0]
    index = _home(t, gate, up)
    if index is None:
        _check_host_out(out, shape, out_dtype)
        found = gated_linear(_to_gpu(t), _to_gpu(gate), _to_gpu(up), activation, None, out_dtype, sums)
        as_numpy = _is_numpy(a)
        return (_to_host(found[0], as_numpy, out), *(_to_host(one, as_numpy) for one in found[1:])) if sums else _to_host(found, as_numpy, out)
    if isinstance(gate, Mx8Matrix):
        _eight_bits("gated_linear", t)
    elif _tracked(torch, t, gate, up):
        if out is not None or sums:
            raise NumKongAmdError("gated_linear with out= or sums= takes no operands that require a gradient")
        _autograd()
        return _GATED.apply(t, gate, up, activation, out_dtype)
    if index != mx._device():
        with torch.cuda.device(index):
            return gated_linear(t, gate, up, activation, out, out_dtype, sums)
    result, kept = _multiply(t, gate, up, None, code, None, out, out_dtype, sums, "gated_linear")
    return (result, *kept) if sums else result


def _backward(grad, a, w, w_up, sums, activation, need_a, need_w, need_up, bias_dtype, where):
    """(of a, of w, of w_up, of the bias): the gradients of either product, None where one is not needed."""
    lib, torch, dtype_codes = _LIB or _library()
    if _CALLS is not None and len(sums) <= 2:
        if (made := _CALLS.linear_backward(grad, a, w, w_up, *sums, *[None] * (2 - len(sums)), ACTIVATIONS.get(activation), need_a, need_w, need_up, bias_dtype)) is not None:
            return made
    names = ("w", None) if w_up is None else ("w_gate", "w_up")
    w, w_up = _matrix(w, names[0]), None if w_up is None else _matrix(w_up, names[1])
    if isinstance(a, Mx8Matrix) or isinstance(w, Mx8Matrix) or isinstance(w_up, Mx8Matrix):
        raise TypeError(f"{where} takes 16-bit matrices")
    t, g, code = _left(a, w), _floats(grad, "grad"), _activation(activation)
    if w_up is not None and (w_up.shape != w.shape or w_up.dtype != w.dtype):
        raise ValueError("w_gate and w_up must have the same shape and type")
    (height, depth), width = t.shape, w.shape[0]
    if tuple(g.shape) != (height, width):
        raise ValueError(f"grad must have shape {(height, width)}, got {tuple(g.shape)}")
    if bias_dtype is not None and bias_dtype not in dtype_codes:
        raise TypeError(f"bias_dtype must be float32, bfloat16 or float16, got {bias_dtype}")
    if w_up is None and not code:
        sums = ()
    sums = [_floats(one, "sums") for one in sums]
    if any(one.dtype != torch.float32 or tuple(one.shape) != (height, width) for one in sums):
        raise ValueError(f"sums must be {(height, width)} of float32, as the product gives them")
    _no_tangent(torch, g, t, w, w_up, *sums)
    index = _home(g, t, w, w_up, *sums)
    if index is None:
        found = _backward(_to_gpu(g), _to_gpu(t), _to_gpu(w), _to_gpu(w_up), [_to_gpu(one) for one in sums], activation, need_a, need_w, need_up, bias_dtype, where)
        return tuple(None if one is None else _to_host(one, _is_numpy(a)) for one in found)
    if index != mx._device():
        with torch.cuda.device(index):
            return _backward(g, t, w, w_up, sums, activation, need_a, need_w, need_up, bias_dtype, where)
    if len(sums) == 2 and _row_bytes(sums[0]) != _row_bytes(sums[1]):
        sums = [one.contiguous() for one in sums]
    device = t.device
    of_a = mx._new(torch, height, depth, t.dtype, device) if need_a else None
    of_w = mx._new(torch, width, depth, w.dtype, device) if need_w else None
    of_up = mx._new(torch, width, depth, w.dtype, device) if need_up and w_up is not None else None
    of_bias = torch.empty((width,), dtype=bias_dtype, device=device) if bias_dtype is not None else None
    l = _LinearBackward(height, width, depth, w_up is not None, dtype_codes[t.dtype], t.data_ptr(), _row_bytes(t), w.data_ptr(), _row_bytes(w), _address(w_up),
                        0 if w_up is None else _row_bytes(w_up), code, sums[0].data_ptr() if sums else None, sums[1].data_ptr() if len(sums) > 1 else None,
                        _row_bytes(sums[0]) if sums else 0, dtype_codes[g.dtype], g.data_ptr(), _row_bytes(g), _address(of_a), depth * 2, _address(of_w),
                        depth * 2, _address(of_up), depth * 2, 0 if bias_dtype is None else dtype_codes[bias_dtype], _address(of_bias))
    needed = lib.nk_amd_linear_backward_workspace_size(l)
    workspace = _workspace(torch, needed, device)
    _check(lib.nk_amd_linear_backward_async(l, _address(workspace), needed, mx._stream(index)), where)
    return of_a, of_w, of_up, of_bias


def linear_backward(grad, a, w, sums=None, activation=None, need_a: bool = True, need_w: bool = True, bias_dtype=None):
    """The gradients ``(of a, of w, of bias)`` of a 16-bit ``linear`` from ``grad``, that of its result; that of the residual is ``grad``
    itself. ``sums`` are those that ``linear`` gave (not looked at without an activation). What is not needed is None; the bias's is given
    where ``bias_dtype`` says its type. The gradient of ``a @ w.T`` is rounded to the matrices' type on the way, and has its range: with float16, scale
    ``grad`` so that it fits. Autograd does not follow this call."""
    if activation is not None and sums is None:
        raise ValueError("an activation's gradient needs the sums that linear(..., sums=True) gives")
    of_a, of_w, _, of_bias = _backward(grad, a, w, None, () if sums is None else (sums,), activation, need_a, need_w, False, bias_dtype, "linear_backward")
    return of_a, of_w, of_bias


def gated_linear_backward(grad, a, w_gate, w_up, gate_sums, up_sums, activation="silu", need_a: bool = True, need_gate: bool = True,
                          need_up: bool = True):
    """The gradients ``(of a, of w_gate, of w_up)`` of a 16-bit ``gated_linear`` from ``grad``, that of its result, and the sums that it
    gave. What is not needed is None. Those of the two products are rounded as in ``linear_backward``. Autograd does not follow this call."""
    if w_up is None:
        raise TypeError("w_up must be a matrix")
    return _backward(grad, a, w_gate, w_up, (gate_sums, up_sums), activation, need_a, need_gate, need_up, None, "gated_linear_backward")[:3]
