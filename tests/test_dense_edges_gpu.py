"""The dense feed-forward operators at their edges on a real MI355X, against 64-bit forms (dense_support.py)."""
import pytest

torch = pytest.importorskip("torch")

import numkong_amd as nk  # noqa: E402
from tests import dense_support as ds  # noqa: E402
from tests.dense_support import normal  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_more_short_rows_than_one_launch_has_tiles_of_64():
    """2^30 rows of 64 values, a window of one vector each (17 GB of results): tiles of 128 rows."""
    rows, width, depth = 1 << 30, 8, 64
    vector = torch.empty(2 * rows + depth, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(1))
    a, w = vector.as_strided((rows, depth), (2, 1)), normal(width, depth, torch.bfloat16, 2).to(DEV)
    y = nk.linear(a, w, activation="relu")
    some = torch.cat([torch.arange(300, device=DEV), rows - 1 - torch.arange(300, device=DEV), torch.randint(0, rows, (4000,), device=DEV, generator=torch.Generator(DEV).manual_seed(3))])
    ds.Linear(a[some].double().cpu(), w.double().cpu(), activation="relu").check(y[some])


def test_operands_with_a_tangent_are_refused():
    forward = torch.autograd.forward_ad
    x, w, v = (normal(m, 64, torch.bfloat16, m).to(DEV) for m in (5, 64, 1))
    v, w8, logits = v[0], nk.mx8_quantize(w), normal(5, 8, torch.float32, 9).to(DEV)
    packed = nk.mx_pack(nk.mx_quantize(w))
    stack = nk.mx_pack(w.expand(8, 64, 64).contiguous())
    weights, chosen = nk.experts_route(logits, 2)
    plan = nk.experts_plan(chosen, 8)
    calls = [  # every operand that could have a derivative, in turn
        (lambda t: nk.rms_norm(t, v, x), x), (lambda t: nk.rms_norm(x, t), v), (lambda t: nk.rms_norm(x, v, t), x), (lambda t: nk.rms_norm_mx8(t, v), x),
        (lambda t: nk.rms_norm_mx8(x, t), v), (lambda t: nk.linear(t, w), x), (lambda t: nk.linear(x, t, activation="gelu"), w), (lambda t: nk.linear(x, w, t), v),
        (lambda t: nk.linear(x, w, residual=t), x), (lambda t: nk.linear(t, w8), x), (lambda t: nk.linear(x, w8, t), v), (lambda t: nk.gated_linear(t, w, w), x),
        (lambda t: nk.gated_linear(x, t, w), w), (lambda t: nk.gated_linear(x, w, t), w), (lambda t: nk.gated_linear(t, w8, w8), x),
        (lambda t: nk.mx_dots_packed(t, packed), x), (lambda t: nk.experts_route(t, 2), logits), (lambda t: nk.mx_dots_experts(t, stack, plan), x),
        (lambda t: nk.mx_dots_experts(x, stack, plan, t), weights),
    ]
    with forward.dual_level():
        for call, t in calls:
            call(t)
            dual = forward.make_dual(t, torch.ones_like(t))
            with pytest.raises(nk.NumKongAmdError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(nk.NumKongAmdError, match="forward-mode"):
                call(dual)
            with pytest.raises(nk.NumKongAmdError, match="forward-mode"):
                call(forward.make_dual(t.clone().requires_grad_(), torch.ones_like(t)))
        same = forward.make_dual(x, torch.ones_like(x))
        codes = nk.mx8_quantize(same)  # (numbers that no gradient passes)
        assert torch.equal(codes.codes.view(torch.uint8), nk.mx8_quantize(x).codes.view(torch.uint8))


def test_gradients_with_a_tangent_are_refused():
    """Forward mode over a backward pass: the pass's own gradients would carry no tangent on."""
    forward = torch.autograd.forward_ad
    x, w, v = (normal(m, 64, torch.bfloat16, m).to(DEV) for m in (5, 64, 1))
    v, logits = v[0], normal(5, 8, torch.float32, 9).to(DEV)
    leaf, free = x.clone().requires_grad_(), logits.clone().requires_grad_()
    found = [(nk.rms_norm(leaf, v), leaf), (nk.rms_norm(leaf, v, x)[0], leaf), (nk.rms_norm(leaf, v, x)[1], leaf), (nk.linear(leaf, w, activation="silu"), leaf), (nk.gated_linear(leaf, w, w), leaf),
             (nk.experts_route(free, 2)[0], free)]
    with forward.dual_level():
        for y, t in found:
            grad = torch.ones_like(y)
            plain, = torch.autograd.grad(y, t, grad, retain_graph=True)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, t, forward.make_dual(grad, torch.ones_like(grad)), retain_graph=True)
            assert torch.equal(torch.autograd.grad(y, t, grad)[0], plain)
    dual_calls = [(lambda t: nk.rms_norm_backward(t, x, v), x), (lambda t: nk.linear_backward(x, t, w), x), (lambda t: nk.gated_linear_backward(x, x, w, t, x.float(), x.float()), w)]
    with forward.dual_level():
        for call, t in dual_calls:
            call(t)
            with pytest.raises(nk.NumKongAmdError, match="forward-mode"):
                call(forward.make_dual(t, torch.ones_like(t)))


def test_8_bit_products_give_no_sums():
    x, w8 = normal(5, 64, torch.bfloat16, 1).to(DEV), nk.mx8_quantize(normal(8, 64, torch.bfloat16, 2).to(DEV))
    for call in (lambda: nk.linear(x, w8, sums=True), lambda: nk.linear(nk.mx8_quantize(x), w8, sums=True), lambda: nk.gated_linear(x, w8, w8, sums=True)):
        with pytest.raises(TypeError, match="16-bit matrices"):
            call()


def test_results_in_out_are_seen_by_autograd():
    x, w = normal(8, 64, torch.bfloat16, 1).to(DEV), normal(64, 64, torch.bfloat16, 2).to(DEV)
    leaf, buffer, w8, packed = torch.ones_like(x).requires_grad_(), x.clone(), nk.mx8_quantize(w), nk.mx_pack(w)
    calls = (lambda out: nk.linear(x, w, out=out), lambda out: nk.linear(x, w, residual=out, out=out), lambda out: nk.linear(x, w8, out=out), lambda out: nk.gated_linear(x, w, w, out=out),
             lambda out: nk.mx_dots_packed(x, packed, out=out))
    for call in calls:
        loss = (leaf * buffer).sum()  # (keeps the buffer)
        call(buffer)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with pytest.raises(nk.NumKongAmdError, match="requires? a gradient"):
            call(leaf)
    with torch.no_grad():
        assert torch.equal(nk.linear(x, w, out=leaf), nk.linear(x, w))


@pytest.mark.parametrize("kind", ds.ACTIVATIONS[1:])
def test_activations_and_slopes_over_their_whole_range(kind):
    """Every activation and slope of any 32-bit x, through a product of zeros with x as its bias, and through the bias's gradient, both in 32 bits. What may
    be off: roundings (of the exponent z four: z units each), and below 1.1e-36 (silu's end), of slopes 2.6e-27 (gelu_tanh's)."""
    ends = torch.tensor([9.0, 10.0, 13.2, 16.0, 80.0, 87.3, 88.0, 89.0, 92.0, 104.0, 128.0, 129.0, 1e4, 3e38, 1e-20, 1e-38, 1e-44, 0.0])
    x = torch.cat([torch.linspace(-130, 130, 40001), torch.linspace(-12, 12, 20001), ends, -ends, torch.nextafter(ends, ends + 1), -torch.nextafter(ends, ends + 1)])
    n = len(x)
    zeros = torch.zeros((n, 1), dtype=torch.bfloat16, device=DEV)
    got = nk.linear(zeros[:1], zeros, x.to(DEV), kind, out_dtype=torch.float32)[0]
    p = x.double()
    near = p.clamp(-128, 128)  # (what is beyond is at its limit, and its exponent with it)
    z = 1.6 * (near.abs() + 0.045 * near.abs() ** 3) if kind == "gelu_tanh" else near.abs()
    truth = torch.where(p > 128, p, torch.where(p < -128, 0.0, ds.activate(kind, near)))
    ds.assert_within(got, truth, (16 + 4 * z.clamp(max=128)) * ds.UNIT * truth.abs() + 1.1e-36, kind)
    slopes = nk.linear_backward(torch.ones((1, n), device=DEV), zeros[:1], zeros, x.to(DEV)[None], kind, need_a=False, need_w=False, bias_dtype=torch.float32)[2]
    truth = torch.where(p > 128, 1.0, torch.where(p < -128, 0.0, ds.slope(kind, near)))
    if kind == "relu":
        truth = (p > 0).double()  # (0 at 0)
    ds.assert_within(slopes, truth, (16 + 4 * z.clamp(max=128)) * ds.UNIT * ds.STEEPEST + 2.6e-27, f"slope of {kind}")


SEGMENT = 22 << 20  # (the allocator asks the driver for so much by itself: what is behind it is no tensor's)


@pytest.fixture
def at_end():
    """Makes copies of matrices and vectors that end with the last byte of an allocation from the driver, their rows `pad` values further apart, NaN before and between."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    kept = []

    def place(x, pad=0):
        room = torch.empty(SEGMENT, dtype=torch.uint8, device=DEV)
        ends = [s["address"] + s["total_size"] for s in torch.cuda.memory_snapshot()]
        if room.data_ptr() + SEGMENT not in ends:
            pytest.skip("the allocator cuts its segments otherwise")
        values = room.view(x.dtype if x.dtype != torch.float8_e4m3fn else torch.uint8)
        values.fill_(float("nan") if x.dtype.is_floating_point and x.dtype != torch.float8_e4m3fn else 127)
        rows, depth = x.shape if x.dim() == 2 else (1, x.shape[0])
        start = values.numel() - ((rows - 1) * (depth + pad) + depth)
        view = values.view(x.dtype).as_strided(x.shape, (depth + pad, 1) if x.dim() == 2 else (1,), start)
        view.copy_(x)
        kept.append(room)
        assert view.data_ptr() + (view.shape[0] - 1) * view.stride(0) * view.itemsize + view.shape[-1] * view.itemsize == room.data_ptr() + SEGMENT or x.dim() == 1
        return view

    yield place
    torch.cuda.synchronize()
    kept.clear()
    torch.cuda.empty_cache()


# few rows; tiles of 64, 128 and 256; depths that end within 16 bytes and, of rows apart, are read in place; rows at odd addresses, which are moved
@pytest.mark.parametrize("m,n,k,pad", [(1, 100, 999, 0), (3, 64, 1000, 3), (16, 33, 130, 0), (17, 512, 130, 0), (65, 257, 72, 4), (100, 130, 66, 2), (129, 255, 8, 0), (200, 96, 6, 2),
                                       (257, 511, 1001, 0), (300, 520, 1002, 6), (513, 1030, 328, 0)])
def test_products_of_operands_at_the_last_bytes_of_memory(at_end, m, n, k, pad):
    a, w, up = (normal(r, k, torch.bfloat16, s) for r, s in ((m, 1), (n, 2), (n, 3)))
    bias, residual, grad = normal(1, n, torch.float32, 4)[0], normal(m, n, torch.float16, 5), normal(m, n, torch.bfloat16, 6)
    ga, gw, gu = at_end(a, pad), at_end(w, pad), at_end(up, pad)
    truth = ds.Linear(a.double(), w.double(), None, bias.double(), "gelu", residual.double())
    y, sums = nk.linear(ga, gw, at_end(bias), "gelu", at_end(residual, pad), out=at_end(torch.zeros_like(grad), pad), sums=True)
    truth.check(y)
    of_a, of_w, of_bias = nk.linear_backward(at_end(grad, pad), ga, gw, at_end(sums, pad), "gelu", bias_dtype=torch.float32)
    truth.check_gradients(grad, a=of_a, w=of_w, bias=of_bias)
    gated = ds.Linear(a.double(), w.double(), up.double(), None, "silu")
    y, gate_sums, up_sums = nk.gated_linear(ga, gw, gu, sums=True)
    gated.check(y)
    of_a, of_w, of_up = nk.gated_linear_backward(at_end(grad, pad), ga, gw, gu, at_end(gate_sums, pad), at_end(up_sums, pad))
    gated.check_gradients(grad, a=of_a, w=of_w, w_up=of_up)
    a8, w8, up8 = (nk.mx8_quantize(t) for t in (ga, gw, gu))
    placed = [nk.Mx8Matrix(at_end(t.codes, pad), at_end(t.scales, pad)) for t in (a8, w8, up8)]
    assert torch.equal(nk.linear(placed[0], placed[1]), nk.linear(a8, w8)) and torch.equal(nk.linear(ga, placed[1]), nk.linear(a8, w8))
    assert torch.equal(nk.gated_linear(*placed), nk.gated_linear(a8, w8, up8))
    assert torch.equal(nk.mx8_dequantize(placed[0], torch.bfloat16), nk.mx8_dequantize(a8, torch.bfloat16))


@pytest.mark.parametrize("dtype", ds.FLOATS)
@pytest.mark.parametrize("rows,depth,pad", [(1, 1, 0), (5, 7, 0), (9, 129, 3), (5, 513, 0), (3, 2049, 1), (3, 8191, 0), (2, 16385, 1), (1, 32767, 0)])
def test_norms_of_operands_at_the_last_bytes_of_memory(at_end, dtype, rows, depth, pad):
    x, r, g, w = normal(rows, depth, dtype, 1), normal(rows, depth, dtype, 2), normal(rows, depth, dtype, 3), (1 + 0.3 * normal(1, depth, torch.float32, 4, 0.0)[0]).to(dtype)
    operands = [t.to(DEV) for t in (x, w, r)]
    placed = at_end(x, pad), at_end(w), at_end(r, pad)
    for got, want in zip(nk.rms_norm(*placed), nk.rms_norm(*operands)):
        assert torch.equal(got, want)
    (got, total), (want, _) = nk.rms_norm_mx8(*placed), nk.rms_norm_mx8(*operands)
    assert torch.equal(got.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got.scales, want.scales)
    of = nk.rms_norm_backward(at_end(g, pad), at_end(total, pad), placed[1], at_end(r, pad))
    for got, want in zip(of, nk.rms_norm_backward(g.to(DEV), total, operands[1], operands[2])):
        assert torch.equal(got, want)
