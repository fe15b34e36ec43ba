"""Dense products and norms on a real MI355X at the sizes that choose their kernels, as programs use them: together, captured, on other streams, with
operands of every layout. Against 64-bit forms (dense_support.py), on the GPU where they are large."""
import pytest

torch = pytest.importorskip("torch")

import numkong_amd as nk  # noqa: E402
from numkong_amd import dense as binding  # noqa: E402
from tests import dense_support as ds  # noqa: E402
from tests.dense_support import HALVES, normal, strided  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def matrix(rows, depth, dtype, seed, scale=1.0):
    generator = torch.Generator(device=DEV).manual_seed(seed)
    return (scale * torch.randn((rows, depth), device=DEV, generator=generator)).to(dtype)


def weights(n, k, dtype, seed):
    return matrix(n, k, dtype, seed, max(k, 1) ** -0.5)


# Sizes at which tiles of 64, 128 and 256 rows are taken, whole and with edges, with and without splits of the depth; depths that are multiples of a
# stage, of 16 bytes, and of neither.
SIZES = [(100, 700, 4096), (130, 8192, 1000), (520, 2048, 2048), (700, 900, 5000), (1030, 2050, 1024), (1500, 3000, 520), (2048, 2048, 4096), (4100, 4103, 264), (4096, 4096, 1030),
         (2300, 9000, 1001), (5000, 260, 6000)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(dtype, m, n, k):
    a, w, bias, residual = matrix(m, k, dtype, 1), weights(n, k, dtype, 2), matrix(1, n, torch.float32, 3)[0], matrix(m, n, dtype, 4)
    truth = ds.Linear(a.double(), w.double(), None, bias.double(), "gelu", residual.double(), dtype)
    for out in (dtype, torch.float32):
        y, sums = nk.linear(a, w, bias, "gelu", residual, out_dtype=out, sums=True)
        truth.check(y, str(out))
        ds.assert_within(sums, truth.p, ds.rounded(truth.p_error, truth.p, torch.float32), "sums")
        assert torch.equal(y, nk.linear(a, w, bias, "gelu", residual, out_dtype=out))
    grad = matrix(m, n, dtype, 5)
    found = nk.linear_backward(grad, a, w, sums, "gelu", bias_dtype=torch.float32)
    truth.check_gradients(grad, a=found[0], w=found[1], bias=found[2])
    assert all(torch.equal(x, y) for x, y in zip(found, nk.linear_backward(grad, a, w, sums, "gelu", bias_dtype=torch.float32)))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gated(dtype, m, n, k):
    a, gate, up = matrix(m, k, dtype, 1), weights(n, k, dtype, 2), weights(n, k, dtype, 3)
    truth = ds.Linear(a.double(), gate.double(), up.double(), activation="silu", half=dtype)
    y, p, q = nk.gated_linear(a, gate, up, sums=True)
    truth.check(y)
    ds.assert_within(p, truth.p, ds.rounded(truth.p_error, truth.p, torch.float32), "gate's sums")
    ds.assert_within(q, truth.q, ds.rounded(truth.q_error, truth.q, torch.float32), "up's sums")
    assert torch.equal(y, nk.gated_linear(a, gate, up))
    grad = matrix(m, n, dtype, 5)
    of_a, of_gate, of_up = nk.gated_linear_backward(grad, a, gate, up, p, q)
    truth.check_gradients(grad, a=of_a, w=of_gate, w_up=of_up)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_mx8(m, n, k):
    a = matrix(m, k, torch.bfloat16, 1)
    w, up = (nk.mx8_quantize(weights(n, k, torch.float32, seed)) for seed in (2, 3))
    a8 = nk.mx8_quantize(a)
    values = [nk.mx8_dequantize(t).double() for t in (a8, w, up)]
    y = nk.linear(a, w, activation="silu")
    ds.Linear(*values[:2], activation="silu", half=torch.bfloat16, sums=ds.mx8_sum_error).check(y)
    assert torch.equal(y, nk.linear(a8, w, activation="silu"))
    y = nk.gated_linear(a, w, up, out_dtype=torch.float16)
    ds.Linear(*values, activation="silu", half=torch.float16, sums=ds.mx8_sum_error).check(y)
    assert torch.equal(y, nk.gated_linear(a8, w, up, out_dtype=torch.float16))


@pytest.mark.parametrize("m", [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129])
def test_rows_around_the_kernels_borders(m):
    for n, k in ((300, 520), (2048, 2049), (8200, 1024)):
        a, w, up = matrix(m, k, torch.float16, 1), weights(n, k, torch.float16, 2), weights(n, k, torch.float16, 3)
        ds.Linear(a.double(), w.double(), half=torch.float16).check(nk.linear(a, w))
        ds.Linear(a.double(), w.double(), up.double(), activation="gelu_tanh", half=torch.float16).check(nk.gated_linear(a, w, up, "gelu_tanh"))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_rows_far_apart_repeated_or_at_odd_addresses(m):
    dtype, k, n = torch.bfloat16, 200, 130
    a, w = normal(m, k, dtype, 1), normal(n, k, dtype, 2, 0.0)
    expected = nk.linear(a.to(DEV), w.to(DEV))
    for pad, offset in ((1, 0), (0, 1), (7, 3), (8, 0), (56, 8), (2, 2)):
        assert torch.equal(expected, nk.linear(strided(a, pad, offset), strided(w, pad, offset)))
    far = torch.empty((m, (1 << 23) + 64), dtype=dtype, device=DEV)[:, :k]  # more than 2^24 bytes from row to row
    far.copy_(a)
    assert torch.equal(expected, nk.linear(far, w.to(DEV)))
    one = a[:1].to(DEV).expand(m, k)
    assert torch.equal(nk.linear(one, w.to(DEV)), nk.linear(one.contiguous(), w.to(DEV)))
    assert torch.equal(nk.linear(a.to(DEV), w[:1].to(DEV).expand(n, k)), nk.linear(a.to(DEV), w[:1].expand(n, k).contiguous().to(DEV)))
    grad = normal(m, n, dtype, 3).to(DEV)
    found = nk.linear_backward(grad, a.to(DEV), w.to(DEV))
    for x, y in zip(found[:2], nk.linear_backward(strided(grad.cpu(), 3, 1), far, strided(w, 5, 1))[:2]):
        assert torch.equal(x, y)
    row = grad[:1].expand(m, n)
    assert all(torch.equal(x, y) for x, y in zip(nk.linear_backward(row, a.to(DEV), w.to(DEV))[:2], nk.linear_backward(row.contiguous(), a.to(DEV), w.to(DEV))[:2]))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", [(2, 300, 100), (200, 300, 100), (300, 300, 1004)])
def test_what_stands_around_operands_does_not_matter(dtype, m, n, k):
    """NaN before, between and behind the rows (`strided` puts them there), at the last bytes of an allocation too."""
    a, w = normal(m, k, dtype, 1), normal(n, k, dtype, 2, 0.0)
    truth = ds.Linear(a.double(), w.double(), half=dtype)
    for pad, offset in ((4, 0), (3, 1), (8, 8)):
        truth.check(nk.linear(strided(a, pad, offset), strided(w, pad, offset)))
    grad = normal(m, n, dtype, 3)
    truth.check_gradients(grad, **dict(zip("aw", nk.linear_backward(strided(grad, 2, 2), strided(a, 4, 2), strided(w, 8, 0))[:2])))


def test_matrices_beyond_32_bits_of_offsets():
    dtype, n, k = torch.bfloat16, 70000, 32768  # 4.6 GB
    w = torch.empty((n, k), dtype=dtype, device=DEV)
    w.copy_(matrix(1, k, dtype, 1, k**-0.5).expand(n, k))
    w[-50:] = weights(50, k, dtype, 2)
    for m in (2, 70):
        a = matrix(m, k, dtype, 3)
        y = nk.linear(a, w)
        ds.Linear(a.double(), w[-60:].double(), half=dtype).check(y[:, -60:])
        ds.Linear(a.double(), w[:60].double(), half=dtype).check(y[:, :60])
    a8 = nk.mx8_quantize(a)
    w8 = nk.mx8_quantize(w)
    ds.Linear(nk.mx8_dequantize(a8).double(), nk.mx8_dequantize(nk.Mx8Matrix(w8.codes[-60:], w8.scales[-60:])).double(), half=dtype, sums=ds.mx8_sum_error).check(nk.linear(a8, w8)[:, -60:])
    del w8
    # the results and the gradient of A with as many rows: of 64 columns
    small = weights(k, 64, dtype, 4)
    tall = torch.empty((n, 64), dtype=dtype, device=DEV)
    tall.copy_(matrix(1, 64, dtype, 5).expand(n, 64))
    tall[-50:] = matrix(50, 64, dtype, 6)
    y = nk.linear(tall, small, out=w)
    ds.Linear(tall[-60:].double(), small.double(), half=dtype).check(y[-60:])
    of_a, of_w, _ = nk.linear_backward(y, tall, small)
    ds.Linear(tall[-60:].double(), small.double(), half=dtype).check_gradients(y[-60:], a=of_a[-60:])
    assert of_w.isfinite().all()
    normed, total = nk.rms_norm(y[-40000:], residual=y[-40000:])
    ds.assert_within(normed[-3:], ds.norm(total[-3:]), ds.rounded(1e-5 * ds.norm(total[-3:]).abs(), ds.norm(total[-3:]), dtype))


def test_empty_ones_have_gradients():
    dtype = torch.bfloat16
    for m, n, k in ((0, 40, 64), (40, 0, 64), (40, 24, 0), (0, 0, 0)):
        a, w, bias = (t.to(DEV).requires_grad_() for t in (normal(m, k, dtype, 1), normal(n, k, dtype, 2), torch.zeros(n)))
        for y in (nk.linear(a, w, bias, "silu"), nk.linear(a, w, bias)):
            found = torch.autograd.grad(y, (a, w, bias), torch.ones_like(y))
            assert not found[0].any() and not found[1].any() and found[0].shape == a.shape and found[1].shape == w.shape
            assert m or not found[2].any()
        y = nk.gated_linear(a, w, w)
        assert not any(t.any() for t in torch.autograd.grad(y, (a, w), torch.ones_like(y)))
        x, scale = normal(m, k, dtype, 3).to(DEV).requires_grad_(), torch.ones(k, device=DEV, requires_grad=True)
        of_x, of_scale = torch.autograd.grad(nk.rms_norm(x, scale), (x, scale), normal(m, k, dtype, 4).to(DEV))
        assert of_x.shape == x.shape and (m or not of_scale.any())


def test_results_over_operands_are_refused():
    store = torch.zeros((64, 200), dtype=torch.bfloat16, device=DEV)
    a, w = store[:, :64], torch.ones((64, 64), dtype=torch.bfloat16, device=DEV)
    for call in (lambda out: nk.linear(a, w, out=out), lambda out: nk.gated_linear(a, w, w, out=out)):
        for out in (a, store[:, 10:74], store[:, 63:127], w):
            with pytest.raises(ValueError, match="shares memory"):
                call(out)
        call(store[:, 64:128])  # rows between those of A
        assert not store.any()
    with pytest.raises(ValueError, match="residual itself"):
        nk.linear(a, w, residual=store[:, 70:134], out=store[:, 71:135])
    row = torch.zeros(64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="bias"):
        nk.linear(a[:1], w, row, out=row[None])
    m = nk.mx8_quantize(w)
    over = torch.empty(0, dtype=torch.bfloat16, device=DEV).set_(m.codes.untyped_storage(), 0, (32, 64), (64, 1))  # the codes' memory
    with pytest.raises(ValueError, match="shares memory with w"):
        nk.linear(a[:32], m, out=over)


def test_gradients_of_many_rows_without_width():
    m = (1 << 21) + 70000  # more rows than one grid of the kernel that writes the zeros is high
    a, w = torch.ones((m, 24), dtype=torch.float16, device=DEV), torch.empty((0, 24), dtype=torch.float16, device=DEV)
    of_a, of_w, _ = nk.linear_backward(torch.empty((m, 0), dtype=torch.float16, device=DEV), a, w)
    assert of_a.shape == a.shape and not of_a.any() and of_w.shape == w.shape


def test_gradients_have_none_of_their_own_and_say_so():
    x, w = (normal(20, 64, torch.float16, seed).to(DEV).requires_grad_() for seed in (1, 2))
    for y in (nk.linear(x, w, activation="silu"), nk.gated_linear(x, w, w), nk.rms_norm(x, w[0])):
        found, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="gradients"):
            found.sum().backward()


def test_the_general_way_gives_the_same(monkeypatch):
    """What csrc/dense_calls.cpp does not take goes through ctypes: the same results, gradients and refusals."""
    assert binding._library() and binding._CALLS is not None
    dtype = torch.bfloat16
    x, w, up, scale = (t.to(DEV) for t in (normal(70, 96, dtype, 1), normal(50, 96, dtype, 2), normal(50, 96, dtype, 3), torch.linspace(0.5, 2, 96)))
    bias, residual, grad = torch.linspace(-1, 1, 50, device=DEV), normal(70, 50, torch.float32, 4).to(DEV), normal(70, 50, dtype, 5).to(DEV)

    def everything():
        m, m2 = nk.mx8_quantize(x), nk.mx8_quantize(w)
        out = [m.codes.float(), m.scales, nk.mx8_dequantize(m), nk.mx8_dequantize(m, dtype), *nk.rms_norm(x, scale, x), nk.rms_norm(x, out_dtype=torch.float32)]
        q, total = nk.rms_norm_mx8(x, scale, x)
        out += [q.codes.float(), q.scales, total, nk.linear(x, w, bias, "gelu", residual), nk.linear(q, m2, bias), nk.gated_linear(x, m2, m2), *nk.linear(x, w, sums=True)]
        out += [t for t in nk.gated_linear(x, w, up, sums=True)]
        leaves = [t.detach().requires_grad_() for t in (x, w, up, scale, bias, residual)]
        y = nk.linear(*leaves[:2], leaves[4], "silu", leaves[5], out_dtype=dtype)
        out += [y.detach(), *torch.autograd.grad(y, [leaves[0], leaves[1], leaves[4], leaves[5]], grad)]
        y = nk.linear(leaves[0].detach(), leaves[1], leaves[4])
        out += torch.autograd.grad(y, [leaves[1], leaves[4]], grad)
        y = nk.linear(x, w, residual=leaves[5])
        out += torch.autograd.grad(y, [leaves[5]], grad)
        y = nk.gated_linear(*leaves[:3], "gelu_tanh")
        out += [y.detach(), *torch.autograd.grad(y, leaves[:3], grad.t().contiguous().t())]
        y = nk.gated_linear(x, w, leaves[2])
        out += torch.autograd.grad(y, [leaves[2]], grad[:1].expand(70, 50))
        y, total = nk.rms_norm(leaves[0], leaves[3], leaves[0])
        out += torch.autograd.grad([y, total], [leaves[0], leaves[3]], [x, x])
        y, total = nk.rms_norm(leaves[0], leaves[3], x)
        out += torch.autograd.grad(total, [leaves[0], leaves[3]], x, allow_unused=True)
        y = nk.rms_norm(x, leaves[3])
        return out + list(torch.autograd.grad(y, [leaves[3]], x))

    short = everything()
    monkeypatch.setattr(binding, "_CALLS", None)
    long = everything()
    assert len(short) == len(long)
    for i, (a, b) in enumerate(zip(short, long)):
        assert (a is None) == (b is None) and (a is None or (a.dtype == b.dtype and torch.equal(a, b))), i


def test_a_block_in_8_bits():
    """Norm with its residual, gated product, product back with the residual, as a server runs them."""
    generator = torch.Generator().manual_seed(7)
    for tokens, width, inner in ((1, 256, 640), (5, 512, 1000), (70, 512, 1000), (700, 1024, 2050)):
        x, stream = normal(tokens, width, torch.bfloat16, 1), normal(tokens, width, torch.bfloat16, 2)
        scale = 1 + 0.2 * torch.randn(width, generator=generator)
        gate, up, down = (nk.mx8_quantize(ds.normal(r, c, torch.float32, s, 0.0).to(DEV) / c**0.5) for r, c, s in ((inner, width, 3), (inner, width, 4), (width, inner, 5)))
        y, total = nk.rms_norm_mx8(x.to(DEV), scale.to(DEV), stream.to(DEV))
        assert torch.equal(total.cpu(), (x.float() + stream.float()).bfloat16())
        h = nk.gated_linear(y, gate, up)
        ds.Linear(*(ds.matrix_values(t) for t in (y, gate, up)), activation="silu", half=torch.bfloat16, sums=ds.mx8_sum_error).check(h)
        after = nk.linear(h, down, residual=total, out=total.clone())
        ds.Linear(ds.matrix_values(nk.mx8_quantize(h)), ds.matrix_values(down), residual=total.double().cpu(), half=torch.bfloat16, sums=ds.mx8_sum_error).check(after)


def test_a_block_trains():
    """The same in 16 bits with all gradients: each operator's is the formula's for what the others handed it."""
    dtype = torch.bfloat16
    x, stream, scale = (t.to(DEV).requires_grad_() for t in (normal(300, 256, dtype, 1), normal(300, 256, dtype, 2), torch.linspace(0.5, 1.5, 256)))
    gate, up, down = (weights(r, c, dtype, s).requires_grad_() for r, c, s in ((520, 256, 3), (520, 256, 4), (256, 520, 5)))
    y, total = nk.rms_norm(x, scale, stream)
    h = nk.gated_linear(y, gate, up)
    after = nk.linear(h, down, residual=total)
    for t in (y, total, h):
        t.retain_grad()
    grad = matrix(300, 256, dtype, 6)
    after.backward(grad)
    last = ds.Linear(h.detach().double(), down.detach().double(), half=dtype)
    last.check_gradients(grad, a=h.grad, w=down.grad)
    middle = ds.Linear(y.detach().double(), gate.detach().double(), up.detach().double(), activation="silu", half=dtype)
    middle.check_gradients(h.grad, a=y.grad, w=gate.grad, w_up=up.grad)
    (of_x, x_error), (of_scale, scale_error) = ds.norm_gradients(y.grad, total.detach(), scale.detach(), grad)
    ds.assert_within(x.grad, of_x, ds.rounded(x_error, of_x, dtype))
    ds.assert_within(scale.grad, of_scale, ds.rounded(scale_error, of_scale, torch.float32))
    assert torch.equal(x.grad, stream.grad)


def test_captured_and_replayed():
    """Two graphs, each with all operators, replayed in turn on new inputs with eager work between: every replay equals the eager result."""
    dtype = torch.bfloat16
    shapes = [(40, 300, 264), (600, 1030, 520)]
    state = []
    for i, (m, n, k) in enumerate(shapes):
        w, up, scale = weights(n, k, dtype, 1 + i), weights(n, k, dtype, 3 + i), matrix(1, k, torch.float32, 5)[0]
        state.append(dict(x=matrix(m, k, dtype, 6), grad=matrix(m, n, dtype, 7), w=w, up=up, scale=scale, w8=nk.mx8_quantize(w)))

    def everything(s):
        y, total = nk.rms_norm(s["x"], s["scale"], s["x"])
        q = nk.rms_norm_mx8(s["x"], s["scale"])
        h, sums = nk.linear(y, s["w"], activation="gelu", sums=True)
        g, p, u = nk.gated_linear(y, s["w"], s["up"], sums=True)
        back = nk.linear_backward(s["grad"], y, s["w"], sums, "gelu", bias_dtype=torch.float32)
        gated = nk.gated_linear_backward(s["grad"], y, s["w"], s["up"], p, u)
        return [y, total, h, g, *back, *gated, *nk.rms_norm_backward(back[0], total, s["scale"], gated[0]), nk.linear(s["x"], s["w8"]), nk.gated_linear(q, s["w8"], s["w8"]), nk.mx8_dequantize(q)]

    graphs = []
    for s in state:
        everything(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = everything(s)
        graphs.append((graph, out))
    for turn in range(4):
        for s, (graph, out) in zip(state, graphs):
            s["x"].copy_(matrix(*s["x"].shape, dtype, 100 + turn))
            expected = [t.clone() for t in everything(s)]
            torch.cuda.synchronize()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, expected))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, expected))


def test_a_training_step_is_captured():
    """Gradients through autograd in a graph, while no eager graph of the same leaves lives."""
    dtype = torch.float16
    x, grad = matrix(130, 200, dtype, 1), matrix(130, 96, dtype, 2)
    w, up, scale = (t.requires_grad_() for t in (weights(96, 200, dtype, 3), weights(96, 200, dtype, 4), torch.ones(200, device=DEV)))

    def step():
        return torch.autograd.grad(nk.gated_linear(nk.rms_norm(x, scale), w, up), (w, up, scale), grad)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        x.copy_(matrix(130, 200, dtype, 10 + turn))
        expected = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expected))


def test_other_streams_and_calls_side_by_side():
    dtype = torch.bfloat16
    a, w = matrix(500, 1024, dtype, 1), weights(700, 1024, dtype, 2)
    w8 = nk.mx8_quantize(w)
    expected, expected8 = nk.linear(a, w, activation="silu"), nk.linear(a, w8)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(5):
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append((nk.linear(a, w, activation="silu"), nk.linear(a, w8)))
    torch.cuda.synchronize()
    assert all(torch.equal(x, expected) and torch.equal(y, expected8) for x, y in results)
    # the same matrix as both operands
    ds.Linear(a.double(), a.double(), half=dtype).check(nk.linear(a, a))
    ds.Linear(a.double(), a.double(), a.double(), activation="silu", half=dtype).check(nk.gated_linear(a, a, a))
