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
