"""The dense feed-forward operators without a GPU: exports, structures, sizes, and what is refused before anything is queued."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import numkong_amd as nk
from numkong_amd import api
from numkong_amd import dense as binding
from tests import dense_support as ds
from tests import support

HEADER = os.path.join(support.ROOT, "include", "numkong_amd", "dense.h")
F32, BF16, F16, E4M3, I8 = api.NK_F32, api.NK_BF16, api.NK_F16, api.NK_E4M3, api.NK_I8
SOME = 1 << 20  # an address that no refused call reads


def lib():
    return binding._library()[0]


def message(status):
    assert status != 0
    return lib().nk_hip_last_error().decode()


def test_every_declared_function_is_exported_and_bound():
    text = open(HEADER).read()
    declared = set(re.findall(r"NK_DYNAMIC[^;(]*?\b(nk_amd_[a-z0-9_]+)\s*\(", text))
    assert len(declared) == 9
    for name in declared:
        parameters = re.search(name + r"\s*\(([^;]*)\);", text).group(1).count(",") + 1
        assert len(getattr(lib(), name).argtypes) == parameters, name


@pytest.mark.parametrize("name,structure", [("nk_amd_rms_norm_t", binding._RmsNorm), ("nk_amd_rms_norm_backward_t", binding._RmsNormBackward),
                                            ("nk_amd_linear_t", binding._Linear), ("nk_amd_linear_backward_t", binding._LinearBackward)])
def test_structures_are_those_of_the_header(name, structure):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = [part for part in re.findall(r"typedef struct \{(.*?)\} (\w+);", text, flags=re.S) if part[1] == name][0][0]
    kinds = {"nk_size_t": ctypes.c_uint64, "float": ctypes.c_float, "nk_dtype_t": ctypes.c_int, "int": ctypes.c_int}
    fields = []
    for declaration in (" ".join(line.split()) for line in body.split(";") if line.strip()):
        kind, names = re.match(r"((?:\w+ )+(?:const \*|\*)?)(.*)", declaration).groups()
        for field in names.split(","):
            fields.append((field.strip(), ctypes.c_void_p if "*" in kind else kinds[kind.strip()]))
    assert fields == list(structure._fields_)


def norm(**changed):
    fields = dict(rows=4, depth=64, eps=1e-6, dtype=BF16, x=SOME, x_stride=128, residual=SOME, residual_stride=128, total=SOME, total_stride=128,
                  weight_dtype=F32, weight=SOME, y_dtype=BF16, y=SOME, y_stride=128, y_scales=None, y_scales_stride=0) | changed
    return lib().nk_amd_rms_norm_async(binding._RmsNorm(**fields), None)


def test_norm_refuses():
    for field in ("dtype", "weight_dtype", "y_dtype"):
        assert "has to be f32, bf16" in message(norm(**{field: I8}))
    assert "too many" in message(norm(rows=1 << 31)) and "32768" in message(norm(depth=32769))
    for eps in (-1e-9, float("nan"), float("inf")):
        assert "eps" in message(norm(eps=eps))
    for field in ("x", "y", "total"):
        assert "NULL" in message(norm(**{field: None}))
    assert "NULL" in message(norm(y_dtype=E4M3))
    for field in ("x", "residual", "total", "weight", "y"):
        assert "aligned" in message(norm(**{field: SOME + 1}))
    for field in ("x_stride", "residual_stride", "total_stride", "y_stride"):
        assert "aligned" in message(norm(**{field: 129}))
    assert norm(rows=0, x=None, y=None) == 0 and norm(depth=0) == 0
    assert "NULL" in message(lib().nk_amd_rms_norm_async(None, None))


def norm_backward(room=1 << 30, workspace=SOME, **changed):
    fields = dict(rows=4, depth=64, eps=1e-6, dtype=BF16, total=SOME, total_stride=128, weight_dtype=F32, weight=SOME, grad_dtype=F16, grad=SOME,
                  grad_stride=128, grad_total=SOME, grad_total_stride=128, grad_x=SOME, grad_x_stride=128, grad_weight=SOME) | changed
    return lib().nk_amd_rms_norm_backward_async(binding._RmsNormBackward(**fields), workspace, room, None)


def test_norm_backward_refuses():
    for field in ("dtype", "weight_dtype", "grad_dtype"):
        assert "have to be" in message(norm_backward(**{field: I8}))
    assert "too many" in message(norm_backward(rows=1 << 31)) and "32768" in message(norm_backward(depth=32769))
    assert "eps" in message(norm_backward(eps=-1.0))
    for field in ("total", "grad", "grad_x"):
        assert "NULL" in message(norm_backward(**{field: None}))
    for field in ("total", "grad", "grad_total", "grad_x", "weight", "grad_weight"):
        assert "aligned" in message(norm_backward(**{field: SOME + 1}))
    size = lib().nk_amd_rms_norm_backward_workspace_size
    needed = size(binding._RmsNormBackward(rows=4, depth=64, grad_weight=SOME))
    assert needed >= 64 * 4 and size(binding._RmsNormBackward(rows=4, depth=64)) == 0
    assert size(binding._RmsNormBackward(rows=4, depth=32769, grad_weight=SOME)) == 0 and size(None) == 0
    for workspace, room in ((None, needed), (SOME + 16, needed), (SOME, needed - 1)):
        assert "workspace" in message(norm_backward(workspace=workspace, room=room))
    assert norm_backward(depth=0) == 0


def test_quantising_refuses():
    def call(name, dtype=F32, x=SOME, rows=4, depth=64, stride=256, codes=SOME, scales=SOME):
        if name == "mx8_quantize_async":
            return lib().nk_amd_mx8_quantize_async(dtype, x, rows, depth, stride, codes, 64, scales, 2, None)
        return lib().nk_amd_mx8_dequantize_async(dtype, codes, 64, scales, 2, rows, depth, x, stride, None)
    for name in ("mx8_quantize_async", "mx8_dequantize_async"):
        assert "f32, bf16 or f16" in message(call(name, dtype=I8)) and "f32, bf16 or f16" in message(call(name, dtype=E4M3))
        assert all("NULL" in message(call(name, **{field: None})) for field in ("x", "codes", "scales"))
        assert "aligned" in message(call(name, x=SOME + 2)) and "aligned" in message(call(name, stride=254))
        assert "too many" in message(call(name, rows=1 << 31)) and "too many" in message(call(name, depth=1 << 31))
        assert call(name, rows=0, x=None) == 0


LINEAR = dict(height=100, width=64, depth=96, gated=0, a_dtype=BF16, a=SOME, a_stride=192, w_dtype=BF16, w=SOME, w_stride=192, activation=2, bias_dtype=F32,
              bias=SOME, residual_dtype=F16, residual=SOME, residual_stride=128, c_dtype=BF16, c=SOME, c_stride=128)
GATED = dict(LINEAR, gated=1, w_up=SOME, w_up_stride=192, bias=None, residual=None)
EIGHT = dict(LINEAR, w_dtype=E4M3, w_scales=SOME, w_scales_stride=4)


def linear(fields, workspace=SOME, room=1 << 40, **changed):
    return lib().nk_amd_linear_async(binding._Linear(**(fields | changed)), workspace, room, None)


def test_products_refuse():
    for fields in (LINEAR, GATED, EIGHT):
        for field in ("height", "width"):
            assert "dimensions" in message(linear(fields, **{field: 1 << 31}))
        assert "dimensions" in message(linear(fields, depth=1 << 22))
        assert "W has to be" in message(linear(fields, w_dtype=F32)) and "A has to" in message(linear(fields, a_dtype=I8))
        assert "C has to be" in message(linear(fields, c_dtype=I8))
        assert "activation" in message(linear(fields, activation=5)) and "activation" in message(linear(fields, activation=-1))
        for field in ("a", "w", "c"):
            assert "NULL" in message(linear(fields, **{field: None}))
        assert "aligned" in message(linear(fields, c_stride=129)) and "aligned" in message(linear(fields, a=SOME + 1))
        assert linear(fields, height=0, c=None) == 0 and linear(fields, width=0, c=None) == 0
    assert "A has to" in message(linear(LINEAR, a_dtype=F16)) and "A has to" in message(linear(LINEAR, a_dtype=F32))
    assert "have to be" in message(linear(LINEAR, bias_dtype=I8)) and "have to be" in message(linear(LINEAR, residual_dtype=I8))
    for field in ("bias", "residual", "w"):
        assert "aligned" in message(linear(LINEAR, **{field: SOME + 1}))
    assert "aligned" in message(linear(LINEAR, pre=SOME + 2, pre_stride=256)) and "aligned" in message(linear(LINEAR, pre=SOME, pre_stride=258))
    assert "gated" in message(linear(GATED, bias=SOME)) and "gated" in message(linear(GATED, residual=SOME))
    assert "both" in message(linear(GATED, pre=SOME, pre_stride=256)) and "both" in message(linear(LINEAR, pre=SOME, pre_up=SOME, pre_stride=256))
    assert "NULL" in message(linear(GATED, w_up=None))
    assert "C has to be" in message(linear(EIGHT, c_dtype=F32))
    assert "NULL" in message(linear(EIGHT, w_scales=None)) and "NULL" in message(linear(EIGHT, a_dtype=E4M3)) and "NULL" in message(linear(EIGHT, gated=1, bias=None, residual=None, w_up=SOME))
    needed = lib().nk_amd_linear_workspace_size(binding._Linear(**EIGHT))
    assert needed >= 100 * 96 + 100 * 3
    for workspace, room in ((None, needed), (SOME + 16, needed), (SOME, needed - 1)):
        assert "workspace" in message(linear(EIGHT, workspace=workspace, room=room))
    assert lib().nk_amd_linear_workspace_size(None) == 0 and lib().nk_amd_linear_workspace_size(binding._Linear(**(LINEAR | {"depth": 1 << 22}))) == 0


BACKWARD = dict(height=100, width=64, depth=96, gated=0, dtype=BF16, a=SOME, a_stride=192, w=SOME, w_stride=192, activation=2, pre=SOME, pre_stride=256,
                grad_dtype=BF16, grad=SOME, grad_stride=128, grad_a=SOME, grad_a_stride=192, grad_w=SOME, grad_w_stride=192, bias_dtype=F32, grad_bias=SOME)
GATED_BACKWARD = dict(BACKWARD, gated=1, w_up=SOME, w_up_stride=192, pre_up=SOME, grad_w_up=SOME, grad_w_up_stride=192, grad_bias=None)


def backward(fields, workspace=SOME, room=1 << 40, **changed):
    return lib().nk_amd_linear_backward_async(binding._LinearBackward(**(fields | changed)), workspace, room, None)


def test_gradients_refuse():
    for fields in (BACKWARD, GATED_BACKWARD):
        for field in ("height", "width", "depth"):
            assert "dimensions" in message(backward(fields, **{field: 1 << 22}))
        assert "have to be" in message(backward(fields, dtype=F32)) and "have to be" in message(backward(fields, dtype=E4M3)) and "has to be" in message(backward(fields, grad_dtype=I8))
        assert "activation" in message(backward(fields, activation=5))
        for field in ("a", "w", "pre", "grad"):
            assert "NULL" in message(backward(fields, **{field: None}))
        for field in ("a", "w", "grad", "grad_a", "grad_w", "pre"):
            assert "aligned" in message(backward(fields, **{field: SOME + 1}))
        needed = lib().nk_amd_linear_backward_workspace_size(binding._LinearBackward(**fields))
        assert needed >= 100 * 64 * 2 * (2 if fields["gated"] else 1)
        for workspace, room in ((None, needed), (SOME + 16, needed), (SOME, needed - 1)):
            assert "workspace" in message(backward(fields, workspace=workspace, room=room))
    assert "bias has to be" in message(backward(BACKWARD, bias_dtype=I8)) and "no bias" in message(backward(GATED_BACKWARD, grad_bias=SOME))
    assert "second" in message(backward(BACKWARD, grad_w_up=SOME)) and "NULL" in message(backward(GATED_BACKWARD, w_up=None))
    assert "NULL" in message(backward(GATED_BACKWARD, pre_up=None)) and "aligned" in message(backward(GATED_BACKWARD, pre_up=SOME + 2))


def test_python_refuses():
    half = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16)  # noqa: E731
    eight = nk.Mx8Matrix(torch.zeros((8, 64), dtype=torch.uint8), torch.zeros((8, 2), dtype=torch.uint8))
    for wrong in ("x", [1.0], None):
        with pytest.raises(TypeError):
            nk.rms_norm(wrong)
        with pytest.raises(TypeError):
            nk.linear(wrong, half(8, 64))
        with pytest.raises(TypeError):
            nk.linear(half(4, 64), wrong)
    cases = [
        (TypeError, lambda: nk.rms_norm(torch.zeros((2, 4), dtype=torch.float64))), (ValueError, lambda: nk.rms_norm(half(2, 3, 4))),
        (ValueError, lambda: nk.rms_norm(half(2, 8)[:, ::2])), (ValueError, lambda: nk.rms_norm(half(2, 8), half(7))),
        (ValueError, lambda: nk.rms_norm(half(2, 8), half(1, 8))), (TypeError, lambda: nk.rms_norm(half(2, 8), torch.zeros(8, dtype=torch.int32))),
        (ValueError, lambda: nk.rms_norm(half(2, 8), residual=half(2, 7))), (ValueError, lambda: nk.rms_norm(half(2, 8), residual=half(2, 8).float())),
        (ValueError, lambda: nk.rms_norm(half(2, 8), eps=-1.0)), (ValueError, lambda: nk.rms_norm(half(2, 8), eps=float("nan"))), (ValueError, lambda: nk.rms_norm(half(2, 8), eps=1e40)),
        (TypeError, lambda: nk.rms_norm(half(2, 8), out_dtype=torch.float64)), (ValueError, lambda: nk.rms_norm_backward(half(2, 8), half(3, 8))),
        (ValueError, lambda: nk.rms_norm_backward(half(2, 8), half(2, 8), grad_total=half(2, 8).float())),
        (TypeError, lambda: nk.linear(half(4, 64).float(), half(8, 64))), (TypeError, lambda: nk.linear(half(4, 64).half(), half(8, 64))),
        (TypeError, lambda: nk.linear(half(4, 64), half(8, 64).float())), (ValueError, lambda: nk.linear(half(4, 63), half(8, 64))),
        (ValueError, lambda: nk.linear(half(4, 64), half(8, 64), half(9))), (ValueError, lambda: nk.linear(half(4, 64), half(8, 64), residual=half(4, 9))),
        (ValueError, lambda: nk.linear(half(4, 64), half(8, 64), activation="tanh")), (TypeError, lambda: nk.linear(half(4, 64), half(8, 64), out_dtype=torch.int32)),
        (ValueError, lambda: nk.linear(half(4, 64), half(8, 64), out=half(4, 9))), (TypeError, lambda: nk.linear(eight, half(8, 64))),
        (TypeError, lambda: nk.linear(eight, eight, out_dtype=torch.float32)), (ValueError, lambda: nk.linear(half(4, 32), eight)),
        (ValueError, lambda: nk.gated_linear(half(4, 64), half(8, 64), half(9, 64))), (ValueError, lambda: nk.gated_linear(half(4, 64), half(8, 64), half(8, 64).half())),
        (ValueError, lambda: nk.gated_linear(half(4, 64), half(8, 64), eight)),
        (ValueError, lambda: nk.linear_backward(half(4, 8), half(4, 64), half(8, 64), None, "silu")), (TypeError, lambda: nk.linear_backward(half(4, 8), eight, eight)),
        (ValueError, lambda: nk.linear_backward(half(4, 9), half(4, 64), half(8, 64))), (ValueError, lambda: nk.linear_backward(half(4, 8), half(4, 64), half(8, 64), half(4, 8), "silu")),
        (TypeError, lambda: nk.linear_backward(half(4, 8), half(4, 64), half(8, 64), bias_dtype=torch.int8)),
        (TypeError, lambda: nk.gated_linear_backward(half(4, 8), half(4, 64), half(8, 64), None, half(4, 8), half(4, 8))),
        (TypeError, lambda: nk.Mx8Matrix(half(8, 64), torch.zeros((8, 2), dtype=torch.uint8))), (ValueError, lambda: nk.Mx8Matrix(eight.codes, eight.scales[:, :1])),
        (ValueError, lambda: nk.Mx8Matrix(eight.codes[:, ::2], eight.scales[:, :1])), (TypeError, lambda: nk.mx8_dequantize(half(2, 8))),
        (TypeError, lambda: nk.mx8_quantize(torch.zeros((2, 8), dtype=torch.int32))),
    ]
    for error, call in cases:
        with pytest.raises(error):
            call()
    if not torch.cuda.is_available():
        for call in (lambda: nk.rms_norm(half(2, 8)), lambda: nk.linear(half(4, 64), half(8, 64)), lambda: nk.mx8_quantize(np.zeros((2, 8), np.float32)),
                     lambda: nk.mx8_dequantize(eight), lambda: nk.rms_norm_mx8(half(2, 8))):
            with pytest.raises(nk.NumKongAmdError, match="no GPU"):
                call()


def test_the_plain_quantiser():
    """The tests' own form on values that say what it has to give."""
    x = np.zeros((5, 32))
    x[0, :4] = 448, 17, 19, -18  # 17 and 19 lie between 16, 18 and 20
    x[1, :2] = 449, 1
    x[2, 0] = 2.0**-140
    x[3, 5] = np.nan
    codes, scales = ds.quantize(x)
    assert scales[:, 0].tolist() == [127, 128, 0, 255, 0]
    assert ds.values(codes, scales)[0, :4].tolist() == [448, 16, 20, -18]
    assert ds.values(codes, scales)[1, :2].tolist() == [448, 1] and np.isnan(ds.values(codes, scales)[3]).all()
    grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ds.GRID, grid)


@pytest.mark.parametrize("kind", ds.ACTIVATIONS[1:])
def test_the_plain_activations(kind):
    x = torch.linspace(-8, 8, 1001, dtype=torch.float64)
    f = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[kind]
    assert torch.allclose(ds.activate(kind, x), f(x), atol=1e-14)
    s = ds.slope(kind, x)
    assert s.abs().max() <= ds.STEEPEST
    if kind != "relu":
        bends = (s[2:] - s[:-2]) / (x[2:] - x[:-2])
        assert bends.abs().max() <= ds.BEND
