"""8-bit blocks and the root mean square norm on a real MI355X, against 64-bit forms (dense_support.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import numkong_amd as nk  # noqa: E402
from tests import dense_support as ds  # noqa: E402
from tests.dense_support import FLOATS, UNIT, normal, strided  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def same_quantized(matrix, x):
    codes, scales = ds.quantize(x)
    got_codes, got_scales = ds.bytes_of(matrix)
    np.testing.assert_array_equal(got_scales, scales)
    np.testing.assert_array_equal(got_codes, codes)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,depth,pad,offset", [(1, 1, 0, 0), (1, 31, 0, 0), (3, 32, 0, 0), (5, 33, 0, 0), (2, 127, 1, 1), (7, 129, 3, 0),
                                                   (16, 4096, 0, 0), (3, 1000, 24, 8), (260, 64, 0, 1), (1, 70000, 0, 0), (0, 8, 0, 0), (4, 0, 0, 0)])
def test_quantize(dtype, rows, depth, pad, offset):
    x = normal(rows, depth, dtype, rows + depth, spread=2.0)
    same_quantized(nk.mx8_quantize(strided(x, pad, offset)), x)


def test_quantize_every_bfloat16():
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).reshape(-1, 1)
    # each value alone in a block, and beside others, which decide the scale of what is smaller
    for other in (0.0, 1.0, 448.0, 449.0):
        block = torch.full((65536, 32), other, dtype=torch.bfloat16)
        block[:, 17:18] = x
        same_quantized(nk.mx8_quantize(block.to(DEV)), block)


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_halfway_and_extreme(dtype):
    info = torch.finfo(dtype)
    middles = torch.tensor((ds.GRID[1:] + ds.GRID[:-1]) / 2)
    x = torch.zeros((len(middles), 32), dtype=torch.float64)
    x[:, 0], x[:, 1], x[:, 2] = 448, middles, -middles
    near = x.clone()
    near[:, 1] *= 1 + 2 * info.eps
    near[:, 2] *= 1 - 2 * info.eps
    ends = torch.zeros((8, 32), dtype=torch.float64)
    for i, value in enumerate((info.max, info.tiny, info.tiny / 8, info.smallest_normal * info.eps, 448.0, 449.0, 448 * (1 + info.eps), 0.0)):
        ends[i, 3], ends[i, 9] = value, -value / 3
    bad = torch.zeros((3, 64), dtype=torch.float64)
    bad[:, 40] = torch.tensor([float("nan"), float("inf"), -float("inf")])
    bad[:, 5] = 2.0
    for t in (x, near, ends, bad):
        t = t.to(dtype)
        same_quantized(nk.mx8_quantize(t.to(DEV)), t)


@pytest.mark.parametrize("dtype", FLOATS)
def test_dequantize_every_code_and_scale(dtype):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 8)
    got = nk.mx8_dequantize(nk.Mx8Matrix(codes.to(DEV), scales.to(DEV)), dtype).cpu()
    with np.errstate(over="ignore"):
        truth = torch.from_numpy(ds.values(codes.numpy(), scales.numpy()))
    expected = truth.float().to(dtype)  # (all are f32 values, so they are rounded once)
    assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), expected.nan_to_num(7.0, 8.0, 9.0))
    assert torch.equal(got.isnan(), expected.isnan()) and torch.equal(got.isinf(), expected.isinf())


def test_dequantize_strided_and_out():
    x = normal(9, 77, torch.float32, 3)
    m = nk.mx8_quantize(x.to(DEV))
    codes, scales = ds.bytes_of(m)
    wide = torch.zeros((9, 90), dtype=torch.uint8, device=DEV)
    wide[:, 5:82] = torch.from_numpy(codes).to(DEV)
    view = nk.Mx8Matrix(wide[:, 5:82], m.scales)
    out = torch.full((9, 100), -1.0, device=DEV)
    assert nk.mx8_dequantize(view, out=out[:, 3:80]) is not None
    assert torch.equal(out[:, 3:80].cpu().double(), torch.from_numpy(ds.values(codes, scales)))
    assert (out[:, :3] == -1).all() and (out[:, 80:] == -1).all()


SHAPES = [(1, 1, 0, 0), (5, 7, 0, 0), (3, 64, 0, 0), (9, 129, 3, 1), (4, 511, 0, 1), (5, 512, 0, 0), (7, 1000, 24, 8), (3, 1024, 0, 0), (2, 1025, 1, 0),
          (16, 4096, 0, 0), (3, 8191, 0, 3), (2, 8200, 0, 0), (1, 16384, 0, 0), (2, 16385, 0, 1), (1, 32768, 0, 0), (700, 96, 0, 0), (0, 64, 0, 0)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,depth,pad,offset", SHAPES)
def test_norm(dtype, rows, depth, pad, offset):
    x, r = normal(rows, depth, dtype, 1), normal(rows, depth, dtype, 2)
    w = (1 + 0.3 * normal(1, depth, torch.float32, 3, 0.0)[0])
    bound = lambda y, out: ds.rounded((depth / 64 + 60) * UNIT * y.abs(), y, out)  # noqa: E731
    for weight_dtype, out, residual in ((dtype, dtype, True), (torch.float32, torch.float32, False), (None, torch.bfloat16, True), (torch.float16, torch.float16, False)):
        weight = None if weight_dtype is None else w.to(weight_dtype)
        gx, gr, gw = strided(x, pad, offset), strided(r, pad, offset), None if weight is None else weight.to(DEV)
        found = nk.rms_norm(gx, gw, gr if residual else None, out_dtype=out)
        total = (x.float() + r.float()).to(dtype) if residual else x
        y = found[0] if residual else found
        if residual:
            assert torch.equal(found[1].cpu(), total)
        truth = ds.norm(total, weight)
        assert y.dtype == out
        ds.assert_within(y, truth, bound(truth, out))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,depth,pad,offset", SHAPES)
def test_norm_mx8(dtype, rows, depth, pad, offset):
    x, r = normal(rows, depth, dtype, 4), normal(rows, depth, dtype, 5)
    w = (1 + 0.3 * normal(1, depth, torch.float32, 6, 0.0)[0]).to(dtype)
    y, total = nk.rms_norm_mx8(strided(x, pad, offset), w.to(DEV), strided(r, pad, offset))
    expected = (x.float() + r.float()).to(dtype)
    assert torch.equal(total.cpu(), expected)
    same_quantized(y, ds.norm(expected, w))
    same_quantized(nk.rms_norm_mx8(strided(x, pad, offset)), ds.norm(x))


def test_norm_mx8_of_a_large_matrix_is_exact():
    """4 M values: some hundred lie so near to a border of the codes that 32-bit arithmetic would put them on its other side."""
    x = torch.randn((1024, 4096), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn((4096,), generator=torch.Generator().manual_seed(9))).to(torch.bfloat16)
    same_quantized(nk.rms_norm_mx8(x.to(DEV), w.to(DEV)), ds.norm(x, w))


@pytest.mark.parametrize("dtype", FLOATS)
def test_norm_of_rows_that_are_zero_or_not_finite(dtype):
    x = normal(8, 200, dtype, 11)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    x[4] = torch.finfo(dtype).smallest_normal
    y = nk.rms_norm(x.to(DEV), eps=1e-6).cpu()
    truth = ds.norm(x)
    truth[3] = torch.where(torch.isinf(x[3].double()), torch.nan, 0.0 * x[3].double())  # x / inf, inf / inf
    ds.assert_within(y, truth, ds.rounded(64 * UNIT * truth.abs(), truth, dtype))
    assert (nk.rms_norm(x[1:2].to(DEV), eps=0.0).cpu().isnan()).all()  # 0 / 0
    m = nk.rms_norm_mx8(x.to(DEV))
    codes, scales = ds.bytes_of(m)
    assert (scales[2] == 255).all() and not codes[1].any() and (scales[1] == 0).all()


def test_norm_of_a_broadcast_residual():
    x, r = normal(33, 100, torch.bfloat16, 12), normal(1, 100, torch.bfloat16, 13)
    y, total = nk.rms_norm(x.to(DEV), residual=r.to(DEV).expand(33, 100))
    expected = (x.float() + r.float()).to(torch.bfloat16)
    assert torch.equal(total.cpu(), expected)
    truth = ds.norm(expected)
    ds.assert_within(y, truth, ds.rounded(64 * UNIT * truth.abs(), truth, torch.bfloat16))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,depth,pad,offset", SHAPES + [(2500, 40, 0, 0), (1030, 513, 1, 0)])
def test_norm_backward(dtype, rows, depth, pad, offset):
    t, g, gt = normal(rows, depth, dtype, 21), normal(rows, depth, dtype, 22), normal(rows, depth, dtype, 23)
    w = (1 + 0.3 * normal(1, depth, torch.float32, 24, 0.0)[0])
    for weight_dtype, with_total, grad_dtype in ((dtype, True, dtype), (torch.float32, False, torch.float32), (None, True, torch.bfloat16)):
        weight = None if weight_dtype is None else w.to(weight_dtype)
        grad = g.to(grad_dtype)
        of_x, of_weight = nk.rms_norm_backward(strided(grad, pad, offset), strided(t, pad, offset), None if weight is None else weight.to(DEV),
                                               strided(gt, pad, offset) if with_total else None)
        (x_truth, x_error), (w_truth, w_error) = ds.norm_gradients(grad, t, weight, gt if with_total else None)
        ds.assert_within(of_x, x_truth, ds.rounded(x_error, x_truth, dtype), "gradient of x")
        if weight is None:
            assert of_weight is None
        else:
            ds.assert_within(of_weight, w_truth, ds.rounded(w_error, w_truth, weight_dtype), "gradient of weight")


def test_norm_gradients_against_differences():
    """Along a direction, the results' difference is what the gradients say: second differences of the 64-bit form bound the rest."""
    x, r, w = (normal(6, 50, torch.float32, s) for s in (31, 32, 33))
    w = w[0]
    g, gt = normal(6, 50, torch.float32, 34), normal(6, 50, torch.float32, 35)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, r)]
    y, total = nk.rms_norm(leaves[0], leaves[1], leaves[2])
    grads = [t.double().cpu() for t in torch.autograd.grad([y, total], leaves, [g.to(DEV), gt.to(DEV)])]
    along = [normal(*(t.shape if t.dim() == 2 else (1, 50)), torch.float64, 36 + i).reshape(t.shape) for i, t in enumerate((x, w, r))]

    def value(step):
        t = x.double() + step * along[0] + r.double() + step * along[2]
        return (ds.norm(t, w.double() + step * along[1]) * g.double() + t * gt.double()).sum()

    h = 1e-4
    slope = (value(h) - value(-h)) / (2 * h)
    third = abs(value(2 * h) - 2 * value(h) + 2 * value(-h) - value(-2 * h)) / (12 * h)  # h^2 f''' / 6
    said = sum((a * b).sum() for a, b in zip(grads, along))
    size = sum((a * b).abs().sum() for a, b in zip(grads, along))
    assert abs(slope - said) <= 2 * third + 1e-10 / h + 200 * UNIT * size
    assert torch.equal(grads[0], grads[2])


def test_norm_autograd_partial_graphs():
    x = normal(5, 64, torch.bfloat16, 41).to(DEV)
    w = normal(1, 64, torch.bfloat16, 42)[0].to(DEV)
    r = normal(5, 64, torch.bfloat16, 43).to(DEV).requires_grad_()
    y, total = nk.rms_norm(x, w, r)
    only_y, = torch.autograd.grad(y.sum(), r, retain_graph=True)  # (an expanded gradient)
    only_total, = torch.autograd.grad(total.float().sum(), r, retain_graph=True)
    assert torch.equal(only_total, torch.ones_like(r))
    expected, _ = nk.rms_norm_backward(torch.ones_like(x), total.detach(), w)
    assert torch.equal(only_y, expected)
    leaf = x.clone().requires_grad_()
    grad, = torch.autograd.grad(nk.rms_norm(leaf).t(), leaf, torch.ones((64, 5), dtype=x.dtype, device=DEV))  # (a transposed one)
    assert torch.equal(grad, nk.rms_norm_backward(torch.ones_like(x), x)[0])
    with pytest.raises(nk.NumKongAmdError, match="no gradient"):
        nk.rms_norm_mx8(x, w, r)
    with torch.no_grad():
        nk.rms_norm_mx8(x, w, r)
