"""Dense products and their gradients on a real MI355X, against 64-bit forms (dense_support.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import numkong_amd as nk  # noqa: E402
from tests import dense_support as ds  # noqa: E402
from tests.dense_support import ACTIVATIONS, FLOATS, HALVES, normal, strided  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def weights(n, k, dtype, seed):
    return (normal(n, k, torch.float32, seed, 0.0) / max(k, 1) ** 0.5).to(dtype)


# height, width, depth, values between rows, values before the first: few rows, tiles and their edges, depths that end inside a step,
# rows that start at odd addresses
SHAPES = [(1, 1, 1, 0, 0), (1, 8, 32, 0, 0), (1, 100, 999, 1, 1), (2, 64, 64, 0, 0), (4, 300, 260, 0, 2), (16, 33, 128, 8, 0), (17, 512, 130, 0, 0),
          (33, 70, 1000, 0, 0), (64, 64, 512, 0, 0), (65, 257, 72, 4, 4), (100, 130, 64, 0, 0), (128, 128, 256, 0, 0), (129, 255, 8, 0, 0), (200, 96, 6, 0, 1),
          (256, 256, 64, 0, 0), (300, 520, 136, 0, 0), (257, 511, 1001, 0, 0), (513, 259, 328, 3, 5), (40, 24, 0, 0, 0), (3, 8, 4100, 0, 0)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k,pad,offset", SHAPES)
def test_linear(dtype, m, n, k, pad, offset):
    a, w = normal(m, k, dtype, m + k), weights(n, k, dtype, n)
    ga, gw = strided(a, pad, offset), strided(w, pad, offset)
    bias, residual = normal(1, n, torch.float32, 5)[0], normal(m, n, torch.float32, 6)
    for i, kind in enumerate(ACTIVATIONS):
        out, other, third = FLOATS[i % 3], FLOATS[(i + 1) % 3], FLOATS[(i + 2) % 3]
        b = bias.to(other) if i % 2 == 0 else None
        r = residual.to(third) if i in (0, 1, 4) else None
        truth = ds.Linear(a.double(), w.double(), None, None if b is None else b.double(), kind, None if r is None else r.double(), dtype)
        y = nk.linear(ga, gw, None if b is None else b.to(DEV), kind, None if r is None else strided(r, pad, offset), out_dtype=out)
        assert y.dtype == out
        truth.check(y, f"{kind}, {out}")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k,pad,offset", SHAPES)
def test_gated(dtype, m, n, k, pad, offset):
    a, gate, up = normal(m, k, dtype, m + k), weights(n, k, dtype, n), weights(n, k, dtype, n + 1)
    for i, kind in enumerate(ACTIVATIONS):
        out = FLOATS[i % 3]
        y = nk.gated_linear(strided(a, pad, offset), strided(gate, pad, offset), strided(up, pad, offset), kind, out_dtype=out)
        ds.Linear(a.double(), gate.double(), up.double(), activation=kind, half=dtype).check(y, f"{kind}, {out}")


def check_mx8(truth, y):
    """Element by element as far as the instruction's own sums let derive, and as a whole, where their errors add up as those of
    many numbers do: 2^-18 of the products' magnitudes, four times what was probed."""
    truth.check(y)
    error = (y.double().cpu() - truth.y).norm()
    size = truth.a.abs() @ truth.w.abs().T
    allowed = 2.0**-18 * size * ds.STEEPEST
    if truth.w_up is not None:
        allowed = allowed * truth.q.abs() + truth.f.abs() * 2.0**-18 * (truth.a.abs() @ truth.w_up.abs().T)
    assert error <= ds.ROUNDING[y.dtype] * truth.y.norm() + allowed.norm() + 1e-30


@pytest.mark.parametrize("m,n,k,pad,offset", SHAPES)
def test_linear_mx8(m, n, k, pad, offset):
    a, w = normal(m, k, torch.bfloat16, m + k), weights(n, k, torch.float32, n)
    bias, residual = normal(1, n, torch.bfloat16, 5)[0], normal(m, n, torch.bfloat16, 6)
    w8 = nk.mx8_quantize(w.to(DEV))
    a8 = nk.mx8_quantize(a.to(DEV))
    for i, (kind, out) in enumerate([(None, torch.bfloat16), ("silu", torch.float16)]):
        b, r = (bias, None) if i else (None, residual)
        truth = ds.Linear(ds.matrix_values(a8), ds.matrix_values(w8), None, None if b is None else b.double(), kind, None if r is None else r.double(), out,
                          ds.mx8_sum_error)
        operands = None if b is None else b.to(DEV), kind, None if r is None else r.to(DEV)
        y = nk.linear(strided(a, pad, offset), w8, *operands, out_dtype=out)
        check_mx8(truth, y)
        assert torch.equal(y, nk.linear(a8, w8, *operands, out_dtype=out))
        # the same matrices as others may hold them: codes and scales side by side, or anywhere
        codes, scales = (torch.from_numpy(t).to(DEV) for t in ds.bytes_of(w8))
        assert torch.equal(y, nk.linear(a8, nk.Mx8Matrix(codes, scales), *operands, out_dtype=out))
        if n and k:
            odd = torch.full((n, k + 7), 0x7F, dtype=torch.uint8, device=DEV)
            odd[:, 3:k + 3] = codes
            odd_scales = torch.full((n, scales.shape[1] + 2), 255, dtype=torch.uint8, device=DEV)
            odd_scales[:, 1:-1] = scales
            assert torch.equal(y, nk.linear(a8, nk.Mx8Matrix(odd[:, 3:k + 3], odd_scales[:, 1:-1]), *operands, out_dtype=out))


@pytest.mark.parametrize("m,n,k,pad,offset", SHAPES)
def test_gated_mx8(m, n, k, pad, offset):
    a, gate, up = normal(m, k, torch.float32, m + k), weights(n, k, torch.float32, n), weights(n, k, torch.float32, n + 1)
    a8, gate8, up8 = (nk.mx8_quantize(t.to(DEV)) for t in (a, gate, up))
    truth = ds.Linear(*(ds.matrix_values(t) for t in (a8, gate8, up8)), activation="gelu_tanh", half=torch.bfloat16, sums=ds.mx8_sum_error)
    y = nk.gated_linear(strided(a, pad, offset), gate8, up8, "gelu_tanh")
    assert y.dtype == torch.bfloat16
    check_mx8(truth, y)
    assert torch.equal(y, nk.gated_linear(a8, gate8, up8, "gelu_tanh"))


@pytest.mark.parametrize("m,n,k", [(5, 48, 200), (130, 260, 520), (300, 64, 96)])
def test_mx8_blocks_of_very_different_scales(m, n, k):
    """Scales over the whole range of exponents that leaves finite results, some blocks zero, some rows NaN."""
    generator = torch.Generator().manual_seed(m)
    a, w = torch.randn((m, k), generator=generator), torch.randn((n, k), generator=generator)
    power = torch.randint(-40, 40, (1, (k + 31) // 32), generator=generator).double().repeat_interleave(32, 1)[:, :k]
    a, w = (a * torch.exp2(power)).float(), (w * torch.exp2(-power)).float()  # products of ordinary size
    a[:, 32:64] = 0
    w[1, 64:96] = 0
    if m > 3:
        a[3, k - 1] = float("nan")
    a8, w8 = nk.mx8_quantize(a.to(DEV)), nk.mx8_quantize(w.to(DEV))
    y = nk.linear(a8, w8)
    truth = ds.Linear(ds.matrix_values(a8), ds.matrix_values(w8), half=torch.bfloat16, sums=ds.mx8_sum_error)
    if m > 3:
        assert y[3].isnan().all()
        keep = torch.arange(m) != 3
        truth = ds.Linear(ds.matrix_values(a8)[keep], ds.matrix_values(w8), half=torch.bfloat16, sums=ds.mx8_sum_error)
        y = y[keep.to(DEV)]
    check_mx8(truth, y)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k,pad,offset", SHAPES)
def test_linear_backward(dtype, m, n, k, pad, offset):
    a, w = normal(m, k, dtype, m + k), weights(n, k, dtype, n)
    ga, gw = strided(a, pad, offset), strided(w, pad, offset)
    for i, (kind, grad_dtype) in enumerate(zip(ACTIVATIONS, (dtype, torch.float32, dtype, torch.bfloat16, torch.float16))):
        grad = normal(m, n, grad_dtype, 9)
        bias = normal(1, n, FLOATS[i % 3], 5)[0]
        truth = ds.Linear(a.double(), w.double(), None, bias.double(), kind, None, dtype)
        y, sums = nk.linear(ga, gw, bias.to(DEV), kind, sums=True)
        ds.assert_within(sums, truth.p, ds.rounded(truth.p_error, truth.p, torch.float32), "sums")
        of_a, of_w, of_bias = nk.linear_backward(strided(grad, pad, offset), ga, gw, sums, kind, bias_dtype=bias.dtype)
        truth.check_gradients(grad, a=of_a, w=of_w, bias=of_bias)
    # any of them alone, without a bias
    alone = [nk.linear_backward(grad.to(DEV), ga, gw, sums, kind, need_a=i == 0, need_w=i == 1, bias_dtype=bias.dtype if i == 2 else None) for i in range(3)]
    assert [[t is not None for t in found] for found in alone] == [[i == j for j in range(3)] for i in range(3)]
    assert torch.equal(alone[0][0], of_a) and torch.equal(alone[1][1], of_w) and torch.equal(alone[2][2], of_bias)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k,pad,offset", SHAPES)
def test_gated_backward(dtype, m, n, k, pad, offset):
    a, gate, up = normal(m, k, dtype, m + k), weights(n, k, dtype, n), weights(n, k, dtype, n + 1)
    ga, gg, gu = (strided(t, pad, offset) for t in (a, gate, up))
    for kind, grad_dtype in zip(ACTIVATIONS, (dtype, torch.float32, dtype, torch.bfloat16, torch.float16)):
        grad = normal(m, n, grad_dtype, 9)
        truth = ds.Linear(a.double(), gate.double(), up.double(), activation=kind, half=dtype)
        y, p, q = nk.gated_linear(ga, gg, gu, kind, sums=True)
        truth.check(y)
        ds.assert_within(p, truth.p, ds.rounded(truth.p_error, truth.p, torch.float32), "gate's sums")
        ds.assert_within(q, truth.q, ds.rounded(truth.q_error, truth.q, torch.float32), "up's sums")
        of_a, of_gate, of_up = nk.gated_linear_backward(strided(grad, pad, offset), ga, gg, gu, p, q, kind)
        truth.check_gradients(grad, a=of_a, w=of_gate, w_up=of_up)
    alone = [nk.gated_linear_backward(grad.to(DEV), ga, gg, gu, p, q, kind, need_a=i == 0, need_gate=i == 1, need_up=i == 2) for i in range(3)]
    assert [[t is not None for t in found] for found in alone] == [[i == j for j in range(3)] for i in range(3)]
    assert torch.equal(alone[0][0], of_a) and torch.equal(alone[1][1], of_gate) and torch.equal(alone[2][2], of_up)


def test_autograd():
    dtype = torch.bfloat16
    a, w, residual = normal(70, 130, dtype, 1), weights(90, 130, dtype, 2), normal(70, 90, torch.float32, 3)
    bias, grad = normal(1, 90, torch.float32, 4)[0], normal(70, 90, torch.bfloat16, 5)
    leaves = [t.to(DEV).requires_grad_() for t in (a, w, bias, residual)]
    y = nk.linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[3])
    truth = ds.Linear(a.double(), w.double(), None, bias.double(), "gelu", residual.double(), dtype)
    truth.check(y.detach())
    of_a, of_w, of_bias, of_residual = torch.autograd.grad(y, leaves, grad.to(DEV))
    truth.check_gradients(grad, a=of_a, w=of_w, bias=of_bias)
    assert of_residual.dtype == torch.float32 and torch.equal(of_residual.cpu(), grad.float())
    # a bias and a residual that were broadcast, a transposed and an expanded gradient
    row = residual[:1].to(DEV).requires_grad_()
    y = nk.linear(leaves[0].detach(), leaves[1], residual=row.expand(70, 90))
    assert torch.equal(torch.autograd.grad(y.t(), row, grad.to(DEV).t())[0], grad.to(DEV).float().sum(0, keepdim=True))
    y = nk.linear(leaves[0], leaves[1])
    ones = torch.ones((70, 90), dtype=dtype, device=DEV)
    assert torch.equal(torch.autograd.grad(y.sum(), leaves[0])[0], nk.linear_backward(ones, a.to(DEV), w.to(DEV))[0])
    # the same matrix as both of a gated product's
    w2 = w.to(DEV).requires_grad_()
    y = nk.gated_linear(a.to(DEV), w2, w2, "silu")
    found, = torch.autograd.grad(y, w2, grad.to(DEV))
    gated = ds.Linear(a.double(), w.double(), w.double(), activation="silu", half=dtype)
    parts = gated.gradients(grad.double())
    value, error = parts["w"][0] + parts["w_up"][0], parts["w"][1] + parts["w_up"][1]
    error = error + ds.ROUNDING[dtype] * (parts["w"][0].abs() + parts["w_up"][0].abs() + error)  # each is rounded before they are added
    ds.assert_within(found, value, ds.rounded(error, value, dtype))


def test_gradients_against_differences():
    """Along a direction, the 64-bit results' difference is what the gradients say, but for the third derivative's share and roundings."""
    dtype = torch.float16
    a, gate, up = normal(20, 40, dtype, 1), weights(30, 40, dtype, 2), weights(30, 40, dtype, 3)
    grad = normal(20, 30, dtype, 4)
    leaves = [t.to(DEV).requires_grad_() for t in (a, gate, up)]
    found = torch.autograd.grad(nk.gated_linear(*leaves, "gelu_tanh"), leaves, grad.to(DEV))
    along = [normal(*t.shape, torch.float64, 7 + i, 0.0) for i, t in enumerate((a, gate, up))]

    def value(step):
        x, g, u = (t.double() + step * v for t, v in zip((a, gate, up), along))
        return (ds.activate("gelu_tanh", x @ g.T) * (x @ u.T) * grad.double()).sum()

    h = 1e-4
    difference = (value(h) - value(-h)) / (2 * h)
    third = abs(value(2 * h) - 2 * value(h) + 2 * value(-h) - value(-2 * h)) / (12 * h)
    said = sum((t.double().cpu() * v).sum() for t, v in zip(found, along))
    truth = ds.Linear(a.double(), gate.double(), up.double(), activation="gelu_tanh", half=dtype).gradients(grad.double())
    allowed = sum((ds.rounded(truth[name][1], truth[name][0], dtype) * v.abs()).sum() for name, v in zip(("a", "w", "w_up"), along))
    assert abs(difference - said) <= 2 * third + 1e-9 / h + allowed


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m", [1, 40, 300])
def test_values_that_are_not_finite_stay_in_their_rows_and_columns(dtype, m):
    a, w = normal(m, 200, dtype, 1), weights(150, 200, dtype, 2)
    a[m // 2, 199] = float("nan")
    w[7, 0] = float("inf")
    y = nk.linear(a.to(DEV), w.to(DEV)).cpu()
    truth = a.double() @ w.double().T
    assert torch.equal(y.isnan(), truth.isnan())
    assert torch.equal(y.isinf(), truth.isinf())
    for kind in ACTIVATIONS[1:]:
        x = torch.tensor([[-float("inf"), float("inf"), float("nan"), -200.0, 200.0, -3e4, 0.0, -0.0]], dtype=dtype).T.contiguous()
        one = torch.ones((1, 1), dtype=dtype)
        got, sums = nk.linear(x.to(DEV), one.to(DEV), activation=kind, sums=True)
        assert got.cpu().flatten()[:2].tolist() == [0.0, float("inf")] and got[2].isnan().all() and got[3:4].abs().item() == 0 and got[4].item() == 200
        of_bias = [nk.linear_backward(torch.ones((1, 1), device=DEV), x[i:i + 1].to(DEV), one.to(DEV), sums[i:i + 1], kind, False, False, torch.float32)[2].item()
                   for i in (0, 1, 3, 4, 5)]
        assert of_bias == [0.0, 1.0, 0.0, 1.0, 0.0]


def test_in_place_and_strided_results():
    dtype = torch.bfloat16
    for m in (3, 100, 400):
        a, w = normal(m, 96, dtype, 1), weights(200, 96, dtype, 2)
        stream = normal(m, 200, dtype, 3).to(DEV)
        expected = nk.linear(a.to(DEV), w.to(DEV), residual=stream)
        store = torch.full((m, 210), 3.0, dtype=dtype, device=DEV)
        out = store[:, 5:205]
        out.copy_(stream)
        assert nk.linear(a.to(DEV), w.to(DEV), residual=out, out=out) is out
        assert torch.equal(out, expected) and (store[:, :5] == 3).all() and (store[:, 205:] == 3).all()
        gated = nk.gated_linear(a.to(DEV), w.to(DEV), w.to(DEV), out=out)
        assert torch.equal(gated, nk.gated_linear(a.to(DEV), w.to(DEV), w.to(DEV)))
        assert (store[:, :5] == 3).all() and (store[:, 205:] == 3).all()


def test_host_operands():
    a, w = normal(20, 64, torch.bfloat16, 1), weights(30, 64, torch.bfloat16, 2)
    y = nk.linear(a, w, activation="relu")
    assert not y.is_cuda and torch.equal(y, nk.linear(a.to(DEV), w.to(DEV), activation="relu").cpu())
    x = np.random.default_rng(0).standard_normal((4, 64)).astype(np.float32)
    found = nk.rms_norm(x)
    assert isinstance(found, np.ndarray) and found.shape == x.shape
    m = nk.mx8_quantize(x)
    assert not m.is_cuda
    assert torch.equal(nk.linear(m, m), nk.linear(*[nk.mx8_quantize(torch.from_numpy(x).to(DEV))] * 2).cpu())
    of_a, of_w, _ = nk.linear_backward(torch.ones((20, 30), dtype=torch.bfloat16), a, w)
    assert not of_a.is_cuda and torch.equal(of_w, nk.linear_backward(torch.ones((20, 30), dtype=torch.bfloat16, device=DEV), a.to(DEV), w.to(DEV))[1].cpu())
