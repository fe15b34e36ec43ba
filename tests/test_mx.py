"""The 4-bit operators and the routing to experts without a GPU: exports, sizes, and what is refused before anything is queued."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import numkong_amd as nk
from numkong_amd import api
from numkong_amd import mx as binding
from tests import mx_support as mx
from tests import support

HEADER = os.path.join(support.ROOT, "include", "numkong_amd", "mx.h")
F32, BF16 = api.NK_F32, api.NK_BF16
I8 = api.NK_I8
SOME = 1 << 20  # an address that no refused call reads


def lib():
    return binding._library()[0]


def refused(name, *arguments):
    """The message of a call that is refused."""
    assert getattr(lib(), "nk_amd_" + name)(*arguments) != 0
    return lib().nk_hip_last_error().decode()


def test_every_declared_function_is_exported_and_bound():
    text = open(HEADER).read()
    declared = set(re.findall(r"NK_DYNAMIC[^;(]*?\b(nk_amd_[a-z0-9_]+)\s*\(", text))
    assert len(declared) == 12
    for name in declared:
        function = getattr(lib(), name)
        parameters = re.search(name + r"\s*\(([^;]*)\);", text).group(1).count(",") + 1
        assert len(function.argtypes) == parameters, name


def test_sizes():
    size = lib().nk_amd_mx_packed_size
    # 64 columns by 512 of depth, half a byte a value and a byte for 32, behind a header of 128 bytes
    assert size(1, 64, 512) == 128 + 64 * 512 // 2 + 64 * 512 // 32
    assert size(3, 1, 1) == 128 + 3 * (64 * 512 // 2 + 64 * 512 // 32)
    assert nk.MxPackedMatrix.packed_size(64, 512) == size(1, 64, 512)
    assert size(1, 1 << 31, 1) == 0 and size(1, 1, 1 << 25) == 0 and size(1 << 20, 1, 1) == 0
    assert size(1, (1 << 31) - 1, (1 << 25) - 1) == 0  # no such amount of memory
    plan = lib().nk_amd_experts_plan_size
    assert plan(0, 1) > 0 and plan(100, 1024) > plan(100, 8) > 100 * 8
    assert plan(1, 0) == 0 and plan(1, 1025) == 0 and plan(1 << 30, 1) == 0
    room = lib().nk_amd_mx_dots_workspace_size
    assert room(0, 8, 8, 0) == 0 and room(8, 0, 8, 0) == 0 and room(1 << 31, 8, 8, 0) == 0
    assert room(1, 8, 64, 0) == 0 < room(1, 8, 64, 1)  # codes have to be laid out, a few floats are not
    assert room(1000, 8, 1000, 0) >= 1000 * (1000 // 2 + 1000 // 32)
    room = lib().nk_amd_mx_experts_workspace_size
    assert room(0, 1, 8, 8, 8, 0, 0) == 0 and room(8, 0, 8, 8, 8, 0, 0) == 0
    assert room(4096, 4, 8, 100, 1000, 0, 1) >= room(4096, 4, 8, 100, 1000, 0, 0) + 4096 * 100 * 4


def test_quantising_refuses():
    call = lambda dtype=F32, x=SOME, rows=4, depth=64, stride=256, codes=SOME, scales=SOME: (  # noqa: E731
        "mx_quantize_async", dtype, x, rows, depth, stride, codes, 32, scales, 2, None)
    assert "f32, bf16 or f16" in refused(*call(dtype=I8))
    assert "NULL" in refused(*call(x=None)) and "NULL" in refused(*call(codes=None)) and "NULL" in refused(*call(scales=None))
    assert "aligned" in refused(*call(x=SOME + 2)) and "aligned" in refused(*call(stride=254))
    assert "too many" in refused(*call(rows=1 << 31)) and "too many" in refused(*call(depth=1 << 31))
    call = lambda dtype=F32, x=SOME, rows=4, depth=64, stride=256, codes=SOME, scales=SOME: (  # noqa: E731
        "mx_dequantize_async", dtype, codes, 32, scales, 2, rows, depth, x, stride, None)
    assert "f32, bf16 or f16" in refused(*call(dtype=I8))
    assert "NULL" in refused(*call(x=None)) and "NULL" in refused(*call(codes=None)) and "NULL" in refused(*call(scales=None))
    assert "aligned" in refused(*call(x=SOME + 2)) and "aligned" in refused(*call(dtype=BF16, stride=129))
    assert "too many" in refused(*call(rows=1 << 31))
    assert lib().nk_amd_mx_quantize_async(F32, None, 0, 64, 0, None, 0, None, 0, None) == 0  # nothing to do


def test_packing_refuses():
    call = lambda codes=SOME, scales=SOME, count=1, width=8, depth=64, image=SOME: (  # noqa: E731
        "mx_pack_async", codes, 32, 0, scales, 2, 0, count, width, depth, image, None)
    assert "dimensions" in refused(*call(depth=1 << 25)) and "dimensions" in refused(*call(width=1 << 31)) and "dimensions" in refused(*call(count=1 << 20))
    assert "16-byte" in refused(*call(image=None)) and "16-byte" in refused(*call(image=SOME + 8))
    assert "NULL" in refused(*call(codes=None)) and "NULL" in refused(*call(scales=None))


def test_products_refuse():
    def call(a_dtype=BF16, a=SOME, a_stride=2000, a_scales=None, packed=SOME, c_dtype=F32, c=SOME, c_stride=400, height=100, width=100,
             depth=1000, workspace=SOME, room=1 << 30):
        return ("mx_dots_packed_async", a_dtype, a, a_stride, a_scales, 32, packed, c_dtype, c, c_stride, height, width, depth, workspace, room, None)
    assert "dimensions" in refused(*call(height=1 << 31)) and "dimensions" in refused(*call(depth=1 << 25))
    assert "A has to be" in refused(*call(a_dtype=I8)) and "C has to be" in refused(*call(c_dtype=I8))
    assert "A is NULL" in refused(*call(a=None)) and "A is NULL" in refused(*call(a=SOME + 1)) and "codes are NULL" in refused(*call(a=None, a_scales=SOME))
    assert "C is NULL" in refused(*call(c=None)) and "C is NULL" in refused(*call(c_stride=402))
    assert "image" in refused(*call(packed=None)) and "image" in refused(*call(packed=SOME + 8))
    needed = lib().nk_amd_mx_dots_workspace_size(100, 100, 1000, 0)
    for workspace, room in ((None, needed), (SOME + 16, needed), (SOME, needed - 1)):
        assert "workspace" in refused(*call(workspace=workspace, room=room))


def test_experts_products_refuse():
    def call(a_dtype=BF16, a=SOME, share=4, packed=SOME, plan=SOME, slots=400, experts=8, top_k=4, weights=None, c_dtype=F32, c=SOME,
             width=100, depth=1000, workspace=SOME, room=1 << 30):
        return ("mx_dots_experts_async", a_dtype, a, 2000, None, 0, share, packed, plan, slots, experts, top_k, weights, c_dtype, c, 400, width,
                depth, workspace, room, None)
    assert "dimensions" in refused(*call(experts=0)) and "dimensions" in refused(*call(experts=1025)) and "dimensions" in refused(*call(slots=1 << 30))
    assert "whole rows" in refused(*call(top_k=0)) and "whole rows" in refused(*call(top_k=3)) and "whole rows" in refused(*call(share=0)) and "whole rows" in refused(*call(share=3))
    assert "A has to be" in refused(*call(a_dtype=I8)) and "C has to be" in refused(*call(c_dtype=I8))
    assert "A is NULL" in refused(*call(a=None)) and "C is NULL" in refused(*call(c=None))
    for pointer in (None, SOME + 4):
        assert "aligned" in refused(*call(packed=pointer)) and "aligned" in refused(*call(plan=pointer))
    for weights in (None, SOME):
        needed = lib().nk_amd_mx_experts_workspace_size(400, 4, 8, 100, 1000, 0, weights is not None)
        for workspace, room in ((None, needed), (SOME + 16, needed), (SOME, needed - 1)):
            assert "workspace" in refused(*call(weights=weights, workspace=workspace, room=room))


def test_products_refuse_before_anything_is_queued():
    """What is too large for the kernels' own counts: no launch for A's rows goes before the refusal."""
    most = (1 << 31) - 1
    call = lambda height, width, depth: ("mx_dots_packed_async", BF16, SOME, 2 * depth, None, 0, SOME, F32, SOME, 4 * width,  # noqa: E731
                                         height, width, depth, SOME, 1 << 62, None)
    assert "too many tiles" in refused(*call(most, most, 32)) and "too large" in refused(*call(most, 100, 1 << 20))
    slots = 1 << 29  # (rows that eight slots share would be quantised first)
    call = lambda width, depth: ("mx_dots_experts_async", BF16, SOME, 2 * depth, None, 0, 8, SOME, SOME, slots, 8, 8, None, F32, SOME, 4 * width,  # noqa: E731
                                 width, depth, SOME, 1 << 62, None)
    assert "too large" in refused(*call(100, 1 << 16)) and "too many tiles" in refused(*call(most, 256))


def test_routing_refuses():
    def how(groups=1, top_groups=1, group_top=1):
        return ctypes.byref(binding._Route(0, 1, 1.0, groups, top_groups, group_top))

    def call(dtype=F32, logits=SOME, stride=256, tokens=4, experts=64, top_k=4, kind=how(), weights=SOME, chosen=SOME):
        return "experts_route_async", dtype, logits, stride, tokens, experts, top_k, None, kind, weights, chosen, None

    def back(chosen=SOME, grad=SOME, result=SOME, stride=256, **others):
        name, dtype, logits, row, tokens, experts, top_k, _, kind, _, _, _ = call(**others)
        return "experts_route_backward_async", dtype, logits, row, tokens, experts, top_k, kind, chosen, grad, result, stride, None

    for of in (call, back):
        assert "f32, bf16 or f16" in refused(*of(dtype=I8))
        for wrong in ({"experts": 0}, {"experts": 1025}, {"top_k": 0}, {"top_k": 65}, {"top_k": 5, "experts": 4}, {"kind": None}, {"logits": None},
                      {"logits": SOME + 2}, {"tokens": 1 << 31}):
            assert refused(*of(**wrong)), wrong
    for wrong in ((0, 1, 1), (5, 1, 1), (128, 1, 1), (8, 9, 1), (8, 0, 1), (8, 2, 3), (8, 2, 0)):
        assert "groups" in refused(*call(kind=how(*wrong))), wrong
    assert "fewer than top_k" in refused(*call(kind=how(32, 1, 1)))
    for wrong in ({"weights": None}, {"chosen": None}):
        assert "NULL" in refused(*call(**wrong))
    for wrong in ({"chosen": None}, {"grad": None}, {"result": None}):
        assert "NULL" in refused(*back(**wrong))
    assert "aligned" in refused(*back(result=SOME + 2)) and "aligned" in refused(*back(stride=258))
    assert "1 to 1024" in refused("experts_plan_async", SOME, 8, 0, SOME, None) and "1 to 1024" in refused("experts_plan_async", SOME, 8, 1025, SOME, None)
    assert "16-byte" in refused("experts_plan_async", SOME, 8, 8, SOME + 4, None) and "chosen" in refused("experts_plan_async", None, 8, 8, SOME, None)


# ---- the Python calls ------------------------------------------------------------------------------------------------

def codes(rows=4, depth=64, count=None):
    shape = (rows,) if count is None else (count, rows)
    return nk.MxMatrix(torch.zeros((*shape, (depth + 1) // 2), dtype=torch.uint8), torch.zeros((*shape, (depth + 31) // 32), dtype=torch.uint8), depth)


def image(count=1, width=8, depth=64):
    return nk.MxPackedMatrix(count, width, depth, torch.zeros(1, dtype=torch.uint8))


def plan(tokens=4, top_k=2, experts=8):
    return nk.ExpertsPlan(tokens, top_k, experts, torch.zeros(1, dtype=torch.uint8))


def test_a_matrix_of_codes_knows_its_shape():
    assert codes(4, 65).shape == (4, 65) and codes(4, 64, 3).shape == (3, 4, 64)
    u8 = lambda *shape: torch.zeros(shape, dtype=torch.uint8)  # noqa: E731
    for wrong in ((u8(4, 32), u8(4, 3), 64), (u8(4, 31), u8(4, 2), 64), (u8(4, 32), u8(5, 2), 64), (u8(32), u8(2), 64), (u8(4, 32), u8(4, 2), -1),
                  (u8(4, 64)[:, ::2], u8(4, 2), 64), (u8(1, 4, 32), u8(4, 2), 64)):
        with pytest.raises(ValueError):
            nk.MxMatrix(*wrong)
    with pytest.raises(TypeError):
        nk.MxMatrix(u8(4, 32).to(torch.int8), u8(4, 2), 64)


@pytest.mark.parametrize("call", [
    lambda: nk.mx_quantize(torch.zeros((4, 64), dtype=torch.float64)),
    lambda: nk.mx_quantize([[1.0]]),
    lambda: nk.mx_dequantize(torch.zeros((4, 64))),
    lambda: nk.mx_dequantize(codes(), torch.int8),
    lambda: nk.mx_dequantize(codes(), out=torch.zeros((4, 64), dtype=torch.float64)),
    lambda: nk.mx_pack(torch.zeros((4, 64), dtype=torch.int32)),
    lambda: nk.mx_dots_packed(torch.zeros((4, 64)), torch.zeros((8, 64))),
    lambda: nk.mx_dots_packed(torch.zeros((4, 64), dtype=torch.int8), image()),
    lambda: nk.mx_dots_packed(torch.zeros((4, 64)), image(), out_dtype=torch.float64),
    lambda: nk.mx_dots_packed(torch.zeros((4, 64)), image(), out=torch.zeros((4, 8)), out_dtype=torch.bfloat16),
    lambda: nk.experts_route(torch.zeros((4, 64), dtype=torch.int32), 2),
    lambda: nk.experts_route_backward(torch.zeros((4, 2)), torch.zeros((4, 64)), torch.zeros((4, 2), dtype=torch.int64)),
    lambda: nk.mx_dots_experts(torch.zeros((4, 64)), image(8), torch.zeros((4, 2), dtype=torch.int32)),
    lambda: nk.mx_dots_experts(torch.zeros((4, 64)), torch.zeros((8, 8, 64)), plan()),
])
def test_wrong_types(call):
    with pytest.raises(TypeError):
        call()


@pytest.mark.parametrize("call", [
    lambda: nk.mx_quantize(torch.zeros(64)),
    lambda: nk.mx_quantize(torch.zeros((64, 4)).T),
    lambda: nk.mx_dequantize(codes(count=2)),
    lambda: nk.mx_dequantize(codes(), out=torch.zeros((4, 63))),
    lambda: nk.mx_pack(torch.zeros(64)),
    lambda: nk.mx_dots_packed(torch.zeros((4, 65)), image()),
    lambda: nk.mx_dots_packed(codes(4, 65), image()),
    lambda: nk.mx_dots_packed(codes(count=2), image()),
    lambda: nk.mx_dots_packed(torch.zeros((4, 64)), image(2)),
    lambda: nk.mx_dots_packed(torch.zeros((4, 64)), image(), out=torch.zeros((4, 9))),
    lambda: nk.experts_route(torch.zeros((4, 64)), 2, "hardmax"),
    lambda: nk.experts_route(torch.zeros((4, 64)), 2, scale=float("nan")),
    lambda: nk.experts_route(torch.zeros((4, 64)), 2, bias=torch.zeros(63)),
    lambda: nk.experts_route(torch.zeros((4, 64)), 2, bias=torch.zeros(64, dtype=torch.float16)),
    lambda: nk.experts_route(torch.zeros(64), 2),
    lambda: nk.experts_route_backward(torch.zeros((4, 2)), torch.zeros((4, 64)), torch.zeros((4, 3), dtype=torch.int32)),
    lambda: nk.experts_route_backward(torch.zeros((5, 2)), torch.zeros((4, 64)), torch.zeros((5, 2), dtype=torch.int32)),
    lambda: nk.experts_plan(torch.zeros((4, 2), dtype=torch.int64), 8),
    lambda: nk.experts_plan(torch.zeros(8, dtype=torch.int32), 8),
    lambda: nk.experts_plan(torch.zeros((4, 2), dtype=torch.int32), 0),
    lambda: nk.experts_plan(torch.zeros((4, 2), dtype=torch.int32), 1025),
    lambda: nk.mx_dots_experts(torch.zeros((4, 64)), image(7), plan()),
    lambda: nk.mx_dots_experts(torch.zeros((5, 64)), image(8), plan()),
    lambda: nk.mx_dots_experts(torch.zeros((4, 65)), image(8), plan()),
    lambda: nk.mx_dots_experts(torch.zeros((4, 64)), image(8), plan(), weights=torch.zeros((4, 3))),
    lambda: nk.mx_dots_experts(torch.zeros((4, 64)), image(8), plan(), weights=torch.zeros((4, 2), dtype=torch.float64)),
    lambda: nk.mx_dots_experts(torch.zeros((4, 64)), image(8), plan(), out=torch.zeros((4, 8))),
    lambda: nk.mx_dots_experts(torch.zeros((4, 64)), image(8), plan(), weights=torch.zeros((4, 2)), out=torch.zeros((4, 2, 8))),
])
def test_wrong_shapes_and_values(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("call", [
    lambda: nk.experts_route(torch.zeros((4, 64)), 2, scale=1e39),
    lambda: nk.experts_route(torch.zeros((4, 64)), 2, groups=(1 << 32) + 1),
    lambda: nk.experts_route(torch.zeros((4, 64)), 2, groups=4, top_groups=(1 << 32) + 1),
    lambda: nk.experts_route(torch.zeros((4, 64)), 2, group_top=-(1 << 32) + 1),
    lambda: nk.experts_route_backward(torch.zeros((4, 2)), torch.zeros((4, 64)), torch.zeros((4, 2), dtype=torch.int32), scale=-1e39),
    lambda: nk.experts_plan(torch.zeros((4, 2), dtype=torch.int32), (1 << 64) + 8),
])
def test_numbers_that_the_library_cannot_hold(call):
    """Refused, and not taken for what is left of them in 32 or 64 bits."""
    with pytest.raises(ValueError):
        call()


@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a GPU")
@pytest.mark.parametrize("call", [
    lambda: nk.mx_quantize(torch.zeros((4, 64))), lambda: nk.mx_quantize(np.zeros((4, 64), np.float32)), lambda: nk.mx_dequantize(codes()),
    lambda: nk.mx_pack(torch.zeros((8, 64))), lambda: nk.mx_dots_packed(torch.zeros((4, 64)), image()), lambda: nk.experts_route(torch.zeros((4, 64)), 2),
    lambda: nk.experts_route_backward(torch.zeros((4, 2)), torch.zeros((4, 64)), torch.zeros((4, 2), dtype=torch.int32)),
    lambda: nk.experts_plan(torch.zeros((4, 2), dtype=torch.int32), 8), lambda: nk.mx_dots_experts(torch.zeros((4, 64)), image(8), plan()),
])
def test_no_gpu_is_an_error(call):
    with pytest.raises(nk.NumKongAmdError, match="no GPU"):
        call()


def test_the_short_way_leaves_the_rest_to_the_general_one():
    """Operands in host memory, other types and shapes, and things that are no tensors: None, and no error."""
    lib()
    calls = binding._CALLS
    assert calls is not None, "numkong_amd/lib/_mx_calls.so is not built"
    x, u8 = torch.zeros((4, 64)), torch.zeros((4, 32), dtype=torch.uint8)
    i32, image_ = torch.zeros((4, 2), dtype=torch.int32), torch.zeros(8, dtype=torch.uint8)
    for a in (x, x.T, x[0], x.double(), x.numpy(), None, "x", 1):
        assert calls.quantize(a) is None
        assert calls.dequantize(u8, a, 64, torch.float32) is None and calls.dequantize(a, u8, 64, torch.float32) is None
        assert calls.dots(a, None, None, image_, 8, 64, torch.float32) is None and calls.dots(x, None, None, a, 8, 64, a) is None
        assert calls.route(a, 2, None, 0, True, 1.0, 1, 1, 1) is None and calls.route(x, 2, a, 0, True, 1.0, 1, 1, 1) is None
        assert calls.route_backward(a, x, i32, 0, True, 1.0) is None and calls.route_backward(x[:, :2], a, i32, 0, True, 1.0) is None
        assert calls.plan(a, 8) is None and calls.plan(i32, a) is None
        assert calls.experts(a, None, None, image_, 8, 8, 64, image_, 4, 2, 8, None, torch.float32) is None
    for name in ("quantize", "dequantize", "dots", "route", "route_backward", "plan", "experts"):
        assert getattr(calls, name)() is None  # (and too few of them)
    with pytest.raises(TypeError):
        calls.bind(1, 2)
    with pytest.raises(ValueError):
        calls.bind(*[0] * 10)


# ---- the plain forms that the GPU's results are compared with ---------------------------------------------------------

def test_plain_quantising():
    """By hand: the largest magnitude of a block goes to [4, 8), ties go to the even code, 6 is the largest."""
    x = np.zeros((1, 64))
    x[0, :8] = [7.9, 5.0, 2.5, 0.25, 0.75, -1.25, -0.0, 6.0]  # scale 1: 6, 4, 2, 0, 1, -1, -0, 6
    x[0, 32] = 2.0**100
    codes, scales = mx.quantize(x)
    assert list(codes[0, :8]) == [7, 6, 4, 0, 2, 10, 8, 7] and list(scales[0]) == [127, 127 + 98] and codes[0, 32] == 6
    assert np.array_equal(mx.values(codes, scales)[0, :8], [6, 4, 2, 0, 1, -1, -0.0, 6]) and mx.values(codes, scales)[0, 32] == 2.0**100
    assert np.array_equal(mx.unpacked(mx.packed(codes[:, :63]), 63), codes[:, :63])
    x[0, 1], x[0, 40] = np.nan, -np.inf
    assert np.isnan(mx.rounded(x)).all()


def test_plain_routing():
    """Renormalised softmax weights are a softmax over the chosen alone; a group that drops out takes its experts with it."""
    logits = np.random.default_rng(1).normal(size=(5, 12))
    chosen = np.argsort(-logits, 1, kind="stable")[:, :3]
    picked = np.take_along_axis(logits, chosen, 1)
    alone = np.exp(picked) / np.exp(picked).sum(1, keepdims=True)
    assert np.allclose(mx.weights(logits, chosen, "softmax", True, 1.0), alone, rtol=1e-12)
    assert np.array_equal(mx.choice(logits, "softmax"), logits)
    grouped = mx.choice(logits, "softmax", groups=4, top_groups=1)
    assert (np.isfinite(grouped).sum(1) == 3).all() and (grouped.argmax(1) == logits.argmax(1)).all()
