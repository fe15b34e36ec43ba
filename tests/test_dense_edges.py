"""The dense feed-forward operators at their edges, without a GPU: waits that the source has to ask for, sizes that few launches hold, refusals."""
import os
import re

import pytest
import torch

import numkong_amd as nk
from numkong_amd import api
from numkong_amd import dense as binding
from tests import support

BF16, F16, E4M3 = api.NK_BF16, api.NK_F16, api.NK_E4M3
SOME = 1 << 20  # an address that no refused call reads
CSRC = os.path.join(support.ROOT, "numkong_amd", "csrc")


def test_tiles_wait_for_every_load_into_lds_before_they_put_sums_there():
    """Behind the loop over the stages loads into LDS (zeros, of stages past the end) are still on their way, into arrays that another wavefront puts
    its sums into: each wavefront has to wait for its own before they meet. A barrier alone does not, by contract."""
    source = open(os.path.join(CSRC, "dense_tiles_gfx950.hpp")).read()
    wait = re.search(r"void arrive_and_meet\(\) \{(.*?)\n\}", source, flags=re.S).group(1)
    assert re.search(r"s_waitcnt\(0x0070\).*s_barrier\(\)", wait, flags=re.S)  # vmcnt(0) and lgkmcnt(0), then the barrier
    kernel = source[source.index("void tile_kernel("):]
    behind = kernel[kernel.index("stage(a1, b1, a0, b0, s + 1"):]
    before_sums = re.sub(r"//.*", "", behind[:behind.index("float *const room")])
    assert "arrive_and_meet();" in before_sums and "__syncthreads" not in before_sums and "s_barrier" not in before_sums


@pytest.mark.skipif(torch.cuda.is_available(), reason="what is not refused would run, on addresses of nothing")
@pytest.mark.parametrize("height,width,depth,gated", [(1 << 30, 8, 64, 0), ((1 << 31) - 1, 1, 64, 0), (1 << 30, 64, 128, 1), (17, (1 << 31) - 128, 64, 1), (70, (1 << 31) - 1, 64, 0)])
def test_many_short_rows_are_not_refused_for_tiles_that_others_hold(height, width, depth, gated):
    """Tiles of 64 rows would be 2^24 or more, which no launch has; those of 128 or 256 fit. (Without a GPU the launch is what fails.)"""
    lib = binding._library()[0]
    l = binding._Linear(height=height, width=width, depth=depth, gated=gated, a_dtype=BF16, a=SOME, a_stride=256, w_dtype=BF16, w=SOME, w_stride=256,
                        w_up=SOME if gated else None, w_up_stride=256, c_dtype=BF16, c=SOME, c_stride=width * 2)
    needed = lib.nk_amd_linear_workspace_size(l)
    assert lib.nk_amd_linear_async(l, SOME, needed, None) != 0
    message = lib.nk_hip_last_error().decode()
    assert "more results" not in message and "tile_kernel" in message


@pytest.mark.parametrize("height,width", [(17, (1 << 31) - 127), (1 << 30, 1 << 20)])
def test_results_of_more_tiles_than_a_launch_has_are_refused(height, width):
    lib = binding._library()[0]
    l = binding._Linear(height=height, width=width, depth=64, gated=1, a_dtype=BF16, a=SOME, a_stride=128, w_dtype=BF16, w=SOME, w_stride=128, w_up=SOME, w_up_stride=128,
                        c_dtype=BF16, c=SOME, c_stride=width * 2)
    assert lib.nk_amd_linear_async(l, SOME, lib.nk_amd_linear_workspace_size(l), None) != 0
    assert "more results" in lib.nk_hip_last_error().decode()


def test_operands_with_a_tangent_are_refused():
    """Forward mode, which torch.no_grad() does not end: the results would carry no tangent on."""
    forward = torch.autograd.forward_ad
    x = torch.ones((2, 8), dtype=torch.bfloat16)
    assert not binding._tracked(torch, x, None) and binding._tracked(torch, x.clone().requires_grad_(), None)
    with forward.dual_level():
        dual = forward.make_dual(x, torch.ones_like(x))
        for operands in ((dual,), (None, x, dual)):
            with pytest.raises(nk.NumKongAmdError, match="forward-mode"):
                binding._tracked(torch, *operands)
            with torch.no_grad(), pytest.raises(nk.NumKongAmdError, match="forward-mode"):
                binding._tracked(torch, *operands)
        assert not binding._tracked(torch, x, forward.unpack_dual(dual).primal)


def test_gradients_with_a_tangent_are_refused():
    forward = torch.autograd.forward_ad
    x, w, v = torch.ones((2, 8), dtype=torch.bfloat16), torch.ones((8, 8), dtype=torch.bfloat16), torch.ones(8)
    weights, chosen = torch.ones((2, 2)), torch.zeros((2, 2), dtype=torch.int32)
    calls = [(lambda t: nk.rms_norm_backward(t, x, v), x), (lambda t: nk.rms_norm_backward(x, t, v), x), (lambda t: nk.rms_norm_backward(x, x, t), v), (lambda t: nk.rms_norm_backward(x, x, v, t), x),
             (lambda t: nk.linear_backward(t, x, w), x), (lambda t: nk.linear_backward(x, t, w), x), (lambda t: nk.linear_backward(x, x, t), w), (lambda t: nk.linear_backward(x, x, w, t, "silu"), x.float()),
             (lambda t: nk.gated_linear_backward(x, x, w, t, x.float(), x.float()), w), (lambda t: nk.experts_route_backward(t, x, chosen), weights), (lambda t: nk.experts_route_backward(weights, t, chosen), x)]
    with forward.dual_level():
        for call, t in calls:
            with pytest.raises(nk.NumKongAmdError, match="forward-mode"):
                call(forward.make_dual(t, torch.ones_like(t)))


def test_8_bit_products_give_no_sums():
    """Results of 8-bit products are 16-bit for the bits that the matrix instruction drops: 32-bit sums would show them, and no backward pass takes them."""
    lib = binding._library()[0]
    fields = dict(height=100, width=64, depth=96, a_dtype=BF16, a=SOME, a_stride=192, w_dtype=E4M3, w=SOME, w_stride=96, w_scales=SOME, w_scales_stride=4, c_dtype=BF16, c=SOME,
                  c_stride=128, pre_stride=256)
    gated = dict(gated=1, w_up=SOME, w_up_stride=96, w_up_scales=SOME, w_up_scales_stride=4)
    for l in (binding._Linear(**fields, pre=SOME), binding._Linear(**fields, **gated, pre=SOME, pre_up=SOME), binding._Linear(**fields, **gated, pre_up=SOME)):
        assert lib.nk_amd_linear_async(l, None, 0, None) != 0 and "16-bit matrices" in lib.nk_hip_last_error().decode()
        assert lib.nk_amd_linear_workspace_size(l) == 0
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    w8 = nk.Mx8Matrix(torch.zeros((8, 64), dtype=torch.uint8), torch.zeros((8, 2), dtype=torch.uint8))
    for call in (lambda: nk.linear(x, w8, sums=True), lambda: nk.linear(w8, w8, sums=True), lambda: nk.gated_linear(x, w8, w8, sums=True)):
        with pytest.raises(TypeError, match="16-bit matrices"):
            call()


def test_results_in_out_are_seen_by_autograd():
    """A tensor that a backward pass has kept, and that a call has written over since, has to be noticed; one that requires a gradient is refused."""
    out = torch.zeros((2, 8))
    version = out._version
    assert binding._result(torch, out, (2, 8), torch.float32, out) is out and out._version > version
    leaf = torch.zeros((2, 8), requires_grad=True)
    kept = (leaf * leaf.sin())  # (keeps the sine)
    for t in (leaf, kept):
        with pytest.raises(nk.NumKongAmdError, match="requires a gradient"):
            binding._result(torch, t, (2, 8), torch.float32, t)
    with torch.no_grad():
        binding._result(torch, leaf, (2, 8), torch.float32, leaf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()
    with torch.inference_mode():
        t = torch.zeros((2, 8))
        assert binding._result(torch, t, (2, 8), torch.float32, t) is t
