"""Routing to experts and the experts' products on a real MI355X, against 64-bit forms (mx_support.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import numkong_amd as nk  # noqa: E402
from tests import mx_support as mx  # noqa: E402
from tests.test_mx_gpu import DEV, normal, strided  # noqa: E402

pytestmark = pytest.mark.gpu

# tokens, experts, top_k, score, with a bias, groups, top_groups, group_top
ROUTES = [(1, 1, 1, "softmax", False, 1, 1, 1), (5, 8, 2, "softmax", False, 1, 1, 1), (9, 8, 8, "sigmoid", True, 1, 1, 1),
          (33, 60, 4, "softmax", False, 1, 1, 1), (7, 64, 6, "softmax", True, 1, 1, 1), (64, 65, 8, "sigmoid", False, 1, 1, 1),
          (100, 128, 8, "softmax", False, 1, 1, 1), (50, 256, 8, "sigmoid", True, 8, 4, 2), (50, 160, 6, "softmax", False, 8, 3, 1),
          (20, 96, 4, "sigmoid", True, 12, 5, 2), (20, 30, 5, "softmax", True, 30, 9, 2), (11, 500, 10, "sigmoid", True, 4, 2, 2),
          (6, 1000, 64, "softmax", False, 1, 1, 1), (6, 1024, 16, "sigmoid", True, 64, 20, 2), (4099, 72, 3, "softmax", False, 3, 2, 2),
          (4200, 256, 8, "sigmoid", True, 8, 4, 2), (4100, 200, 4, "softmax", False, 5, 2, 1), (4097, 210, 20, "sigmoid", True, 21, 10, 2)]


def logits_of(tokens, experts, dtype, seed):
    return (2 * normal(tokens, experts, torch.float32, seed, 0.0)).to(dtype)


def check_route(logits, got_weights, got_experts, top_k, score, bias, groups, top_groups, group_top, renormalize, scale):
    """The chosen are among the best: exactly where selection goes by logits; within the rounding of scores otherwise, which
    are made in 32 bits from a sum of `experts` terms and few operations more: 8 + experts / 64 units of 2^-23, of scores
    and biases below 2."""
    experts, found = got_experts.cpu().numpy(), got_weights.double().cpu().numpy()
    x = logits.double().cpu().numpy()
    slack = 0.0 if bias is None and group_top == 1 else (8 + x.shape[1] / 64) * 2.0**-22 * max(1.0, np.abs(x[np.isfinite(x)]).max())
    selection = mx.choice(x, score, None if bias is None else bias.cpu().numpy())
    if groups > 1:  # which groups stay, from the result itself where sums are too near to tell
        exact = mx.choice(x, score, None if bias is None else bias.cpu().numpy(), groups, top_groups, group_top)
        inside = selection.reshape(len(x), groups, -1)
        of_group = np.sort(inside, 2)[:, :, ::-1][:, :, :group_top].sum(2)
        ordered = np.sort(of_group, 1)[:, ::-1]
        clear = np.ones(len(x), bool) if top_groups == groups else ordered[:, top_groups - 1] - ordered[:, top_groups] > slack
        assert clear.mean() > 0.9
        x, selection, experts, found = x[clear], exact[clear], experts[clear], found[clear]
    order = np.argsort(-selection, axis=1, kind="stable")[:, :top_k]
    best = np.take_along_axis(selection, order, 1)
    there = ~np.isneginf(best)
    np.testing.assert_array_equal(experts >= 0, there)
    mine = np.where(there, np.take_along_axis(selection, np.maximum(experts, 0), 1), 0)
    if slack == 0:
        np.testing.assert_array_equal(experts, np.where(there, order, -1))
    assert (np.abs(mine - np.where(there, best, 0)) <= slack).all()
    for row in experts:
        real = row[row >= 0]
        assert len(set(real)) == len(real)
    want = mx.weights(x, experts, score, renormalize, scale)
    np.testing.assert_allclose(found, want, rtol=(16 + x.shape[1] / 32) * 2.0**-23, atol=1e-30)


@pytest.mark.parametrize("tokens,experts,top_k,score,biased,groups,top_groups,group_top", ROUTES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_route(tokens, experts, top_k, score, biased, groups, top_groups, group_top, dtype):
    logits = logits_of(tokens, experts, dtype, tokens + experts)
    logits = strided(logits, 3, 1) if tokens % 2 else logits.to(DEV)
    bias = 0.2 * normal(1, experts, torch.float32, 3, 0.0)[0].to(DEV) if biased else None
    for renormalize, scale in ((True, 1.0), (False, 2.5)):
        weights, chosen = nk.experts_route(logits, top_k, score, bias, groups, top_groups, group_top, renormalize, scale)
        assert weights.dtype == torch.float32 and chosen.dtype == torch.int32 and weights.shape == chosen.shape == (tokens, top_k)
        check_route(logits, weights, chosen, top_k, score, bias, groups, top_groups, group_top, renormalize, scale)


@pytest.mark.parametrize("experts", [6, 70, 300])
def test_ties_go_to_the_lowest(experts):
    generator = torch.Generator().manual_seed(experts)
    logits = torch.randint(-1, 2, (200, experts), generator=generator).float()
    logits[0] = 0.0
    logits[1] = torch.where(torch.arange(experts) % 2 == 0, 0.0, -0.0)
    for score, bias in (("softmax", None), ("sigmoid", None), ("sigmoid", torch.zeros(experts, device=DEV))):
        _, chosen = nk.experts_route(logits.to(DEV), 5, score, bias)
        want = np.argsort(-logits.numpy(), axis=1, kind="stable")[:, :5]
        np.testing.assert_array_equal(chosen.cpu().numpy(), want)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups", [(8, 1, 1), (64, 8, 2), (130, 1, 1)])
def test_masked_logits(score, experts, groups, top_groups):
    logits = logits_of(8, experts, torch.float32, 1)
    logits[0] = -float("inf")
    logits[1, 1:] = -float("inf")
    logits[2, :-2] = -float("inf")
    logits[3] = torch.finfo(torch.float32).min  # the lowest number is a number
    logits[4, 3] = torch.finfo(torch.float32).max
    bias = torch.linspace(-1, 1, experts, device=DEV) if score == "sigmoid" else None
    weights, chosen = nk.experts_route(logits.to(DEV), 4, score, bias, groups, top_groups)
    weights, chosen = weights.cpu().numpy(), chosen.cpu().numpy()
    assert (chosen[0] == -1).all() and (weights[0] == 0).all()
    assert list(chosen[1]) == [0, -1, -1, -1] and (weights[1, 1:] == 0).all() and abs(weights[1, 0] - 1) < 1e-6
    assert sorted(chosen[2][:2]) == [experts - 2, experts - 1] and list(chosen[2][2:]) == [-1, -1]
    assert (chosen[3] >= 0).all() and np.isfinite(weights[3]).all()
    if score == "softmax":
        assert list(chosen[3]) == [0, 1, 2, 3] and np.allclose(weights[3], 0.25) and chosen[4][0] == 3 and weights[4][0] == 1
    grad = nk.experts_route_backward(torch.ones((8, 4), device=DEV), logits.to(DEV), torch.from_numpy(chosen).to(DEV), score, False)
    assert bool(grad.isfinite().all()) and not grad[0].any() and not grad[logits.isneginf().to(DEV)].any()


@pytest.mark.parametrize("experts,groups,top_groups", [(100, 1, 1), (100, 5, 2), (144, 1, 1), (144, 9, 3), (256, 8, 3)])
def test_many_tokens_choose_as_few(experts, groups, top_groups):
    """Masks, ties, NaNs and infinities among as many tokens as share wavefronts: chosen as where a token has its own. (Sigmoid
    scores are those of each logit alone; weights differ by the order of a sum of four.)"""
    logits = logits_of(32, experts, torch.float32, 8)
    logits[0], logits[1, 3:], logits[2, :-2], logits[3] = -float("inf"), -float("inf"), -float("inf"), 0.25
    logits[4, 7], logits[5, 9], logits[6] = float("nan"), float("inf"), torch.finfo(torch.float32).min
    logits[7:12] = logits[7:12].round()
    logits = logits.to(DEV)
    bias = (torch.arange(experts, device=DEV) % 4).float()
    for of in (None, bias):
        weights, chosen = nk.experts_route(logits, 4, "sigmoid", of, groups, top_groups, 2)
        many, many_chosen = nk.experts_route(logits.repeat(160, 1), 4, "sigmoid", of, groups, top_groups, 2)
        assert torch.equal(many_chosen, chosen.repeat(160, 1))
        torch.testing.assert_close(many, weights.repeat(160, 1), rtol=2.0**-21, atol=0.0, equal_nan=True)


def test_nan_and_infinity_show():
    logits = logits_of(3, 16, torch.float32, 2)
    logits[0, 5], logits[1, 6] = float("nan"), float("inf")
    for score in ("softmax", "sigmoid"):
        weights, chosen = nk.experts_route(logits.to(DEV), 2, score)
        assert int(chosen[0, 0]) == 5 and bool(weights[0].isnan().all()) and int(chosen[1, 0]) == 6
        assert bool(weights[1, 0].isnan()) == (score == "softmax")
        assert bool(weights[2].isfinite().all())


@pytest.mark.parametrize("tokens,experts,top_k,score,renormalize,dtype",
                         [(1, 4, 2, "softmax", True, torch.float32), (40, 64, 4, "softmax", True, torch.float32),
                          (40, 100, 4, "softmax", False, torch.bfloat16), (33, 256, 8, "sigmoid", True, torch.float32),
                          (33, 130, 8, "sigmoid", False, torch.float16), (9, 1000, 64, "softmax", True, torch.float32),
                          (5, 300, 1, "sigmoid", False, torch.float32), (4200, 100, 4, "softmax", True, torch.float32),
                          (4200, 160, 20, "sigmoid", True, torch.float32)])
def test_route_gradient(tokens, experts, top_k, score, renormalize, dtype):
    """Against the formula's gradient in 64 bits, from autograd; padding and missing experts among the rows."""
    logits = logits_of(tokens, experts, dtype, tokens)
    logits[tokens // 2] = -float("inf")
    logits[0, : experts - top_k + 1] = -float("inf")
    x = strided(logits, 1, 1)
    _, chosen = nk.experts_route(x, top_k, score, None, 1, 1, 1, renormalize, 1.5)
    grad = normal(tokens, top_k, torch.float32, 5, 0.0)
    got = nk.experts_route_backward(grad.to(DEV), x, chosen, score, renormalize, 1.5)
    assert got.dtype == dtype and got.shape == logits.shape
    there, index = chosen.cpu() >= 0, chosen.cpu().clamp(min=0).long()
    leaf = logits.double().masked_fill(logits.isneginf(), -1e300)
    leaf[tokens // 2] = 0
    leaf.requires_grad_()
    s = torch.softmax(leaf, 1) if score == "softmax" else torch.sigmoid(leaf)
    picked = s.gather(1, index) * there
    weights = 1.5 * (picked / (picked.sum(1, keepdim=True) + 1e-20) if renormalize else picked)
    (weights * grad.double()).sum().backward()
    want = leaf.grad.masked_fill(logits.isneginf(), 0).numpy()
    # sums over the row and over the chosen of terms no larger than |g| / D, in 32 bits, then the rounding of the result
    total = (picked.sum(1, keepdim=True) + 1e-20).detach().numpy() if renormalize else 1.0
    size = 1.5 * np.abs(grad.numpy()).max(1, keepdims=True) / np.maximum(total, 1e-6) * s.detach().numpy()
    allowed = (32 + experts / 8) * 2.0**-23 * size + mx.ROUNDING[dtype] * np.abs(want) + mx.SMALLEST[dtype]
    assert (np.abs(got.double().cpu().numpy() - want) <= allowed).all()


@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_gradient_by_differences(score, renormalize):
    """(f(x + h) - f(x - h)) / 2h of the operator itself, h = 2^-6: off by h^2 / 6 of the third derivative (weights have
    derivatives of at most 6 at these sizes) and by 2^-22 / h of rounding."""
    tokens, experts, top_k = 3, 6, 3
    logits = torch.arange(experts).float().mul(0.7).repeat(tokens, 1) + 0.1 * normal(tokens, experts, torch.float32, 6, 0.0)
    grad = normal(tokens, top_k, torch.float32, 7, 0.0)
    _, chosen = nk.experts_route(logits.to(DEV), top_k, score, renormalize=renormalize)
    got = nk.experts_route_backward(grad.to(DEV), logits.to(DEV), chosen, score, renormalize).cpu().double().numpy()
    h, want = 2.0**-6, np.zeros((tokens, experts))
    for expert in range(experts):
        sides = []
        for sign in (1, -1):
            moved = logits.clone()
            moved[:, expert] += sign * h
            weights, again = nk.experts_route(moved.to(DEV), top_k, score, renormalize=renormalize)
            assert torch.equal(again, chosen)
            sides.append((weights.double().cpu() * grad.double()).sum(1).numpy())
        want[:, expert] = (sides[0] - sides[1]) / (2 * h)
    allowed = np.abs(grad.numpy()).sum(1, keepdims=True) * (h * h + 2.0**-22 / h)
    assert (np.abs(got - want) <= allowed).all()


# ---- the plan and the products ---------------------------------------------------------------------------------------

def routing(tokens, top_k, experts, kind, seed=0):
    rng = np.random.default_rng(seed)
    chosen = np.array([rng.permutation(experts)[:top_k] if top_k <= experts else rng.integers(0, experts, top_k) for _ in range(tokens)])
    chosen = chosen.reshape(tokens, top_k).astype(np.int32)
    if kind == "one":  # everything to one expert
        chosen[:] = experts - 1
    elif kind == "none":
        chosen[:] = -1
    elif kind == "some":  # padding, missing experts, experts of other processes
        chosen[rng.random(tokens) < 0.3] = -1
        chosen[rng.random(chosen.shape) < 0.1] = experts + 5
        chosen[rng.random(chosen.shape) < 0.05] = np.iinfo(np.int32).min
    return chosen


CASES = [(1, 1, 1, "all"), (1, 4, 8, "all"), (3, 2, 60, "some"), (40, 4, 32, "all"), (40, 4, 32, "some"), (130, 2, 8, "all"), (100, 2, 3, "some"),
         (300, 4, 8, "all"), (300, 4, 16, "some"), (1000, 1, 2, "all"), (700, 2, 4, "one"), (50, 3, 128, "none"), (600, 8, 16, "some"),
         (33, 5, 1000, "some"), (2000, 1, 3, "one")]


@pytest.mark.parametrize("tokens,top_k,experts,kind", CASES + [(9000, 4, 77, "some"), (1, 1, 1024, "all"), (0, 4, 8, "all")])
def test_plan(tokens, top_k, experts, kind):
    chosen = routing(tokens, top_k, experts, kind, tokens)
    plan = nk.experts_plan(torch.from_numpy(chosen).to(DEV), experts)
    assert (plan.tokens, plan.top_k, plan.experts) == (tokens, top_k, experts)
    words = plan.buffer.view(torch.int32).cpu().numpy()
    flat = chosen.reshape(-1)
    bucket = np.where((flat >= 0) & (flat < experts), flat, experts)
    counts = np.bincount(bucket, minlength=experts + 1)
    sizes = (counts + 15) // 16 * 16  # an expert's rows start at a multiple of 16; rows between have slot -1
    starts = np.concatenate([[0], np.cumsum(sizes)])[:-1]
    tile_rows, tile_count, zero_tiles, first_zero, end_zero = words[3:8]
    assert (first_zero, end_zero) == (starts[experts], starts[experts] + counts[experts])
    np.testing.assert_array_equal(words[8:8 + experts + 2], np.concatenate([starts, [end_zero]]))
    buckets = min(len(flat), experts + 1)
    first, room = 8 + (experts + 2 + 3) // 4 * 4, (len(flat) + buckets * 15 + 15) // 16 * 16
    order, place = np.full(sizes.sum(), -1), np.full(len(flat), -1)
    for e in range(experts + 1):
        slots = np.flatnonzero(bucket == e)
        order[starts[e]:starts[e] + counts[e]] = slots
        place[slots] = starts[e] + np.arange(counts[e]) if e < experts else -1
    np.testing.assert_array_equal(words[first:first + len(order)], order)
    np.testing.assert_array_equal(words[first + room:first + room + len(flat)], place)
    tiles = words[(first + room + len(flat) + 3) // 4 * 4:][:4 * (tile_count + zero_tiles)].reshape(-1, 4)
    want = [(e, starts[e] + row, min(starts[e] + row + tile_rows, starts[e] + counts[e]))
            for e in range(experts + 1) for row in range(0, counts[e], tile_rows)]
    np.testing.assert_array_equal(tiles[:, :3], np.array(want).reshape(-1, 3))
    assert tile_count == sum(tile[0] < experts for tile in want)


@pytest.mark.parametrize("tokens,top_k,experts,kind", CASES)
@pytest.mark.parametrize("n,k,dtype,out", [(130, 200, torch.bfloat16, torch.bfloat16), (64, 513, torch.float32, torch.float32), (77, 33, torch.float16, torch.float16)])
def test_experts_products(tokens, top_k, experts, kind, n, k, dtype, out):
    if experts > 200 and n != 130:
        pytest.skip("one size is enough of a thousand experts")
    chosen = routing(tokens, top_k, experts, kind, tokens + 1)
    a = normal(tokens, k, dtype, tokens, 0.2)
    stack = normal(experts * n, k, torch.float32, experts, 0.2).reshape(experts, n, k)
    packed = nk.mx_pack(stack.to(DEV))
    assert packed.count == experts
    plan = nk.experts_plan(torch.from_numpy(chosen).to(DEV), experts)
    left, right = mx.rounded(a), mx.rounded(stack.reshape(-1, k)).reshape(experts, n, k)
    truth, magnitude = np.zeros((tokens, top_k, n)), np.zeros((tokens, top_k, n))
    for e in range(experts):
        token, slot = np.nonzero(chosen == e)
        truth[token, slot], magnitude[token, slot] = left[token] @ right[e].T, np.abs(left[token]) @ np.abs(right[e]).T
    got = nk.mx_dots_experts(a.to(DEV), packed, plan, out_dtype=out)
    assert got.shape == (tokens, top_k, n) and got.dtype == out
    mx.close(got, truth, magnitude, k)
    # a row for each slot, quantised beforehand
    slots = nk.mx_quantize(a.repeat_interleave(top_k, 0).to(DEV))
    mx.close(nk.mx_dots_experts(slots, packed, plan, out_dtype=out), truth, magnitude, k)
    # summed by weight; what stands at slots without an expert is not looked at
    weights = torch.rand((tokens, top_k), generator=torch.Generator().manual_seed(2)) - 0.3
    there = torch.from_numpy((chosen >= 0) & (chosen < experts))
    weights[~there] = float("nan")
    weight = np.where(there.numpy(), weights.double().numpy(), 0)
    summed = (truth * weight[..., None]).sum(1)
    magnitudes = (magnitude * np.abs(weight)[..., None]).sum(1)
    sizes = (np.abs(truth * weight[..., None])).sum(1)
    extra = top_k * 2.0**-23 * sizes
    got = nk.mx_dots_experts(a.to(DEV), packed, plan, weights.to(DEV), out_dtype=out)
    assert got.shape == (tokens, n)
    mx.close(got, summed, magnitudes, k, extra)


@pytest.mark.parametrize("tokens,top_k,experts,n,k", [(4200, 8, 16, 130, 513), (3000, 6, 40, 77, 1000), (4200, 8, 16, 600, 700), (6000, 8, 16, 1100, 200)])
def test_rows_that_go_to_many(tokens, top_k, experts, n, k):
    """Rows that several experts have, some as floats and some quantised first, one tile to a workgroup and several."""
    chosen = torch.from_numpy(routing(tokens, top_k, experts, "some", 3))
    a, stack = normal(tokens, k, torch.bfloat16, 1, 0.2).to(DEV), normal(experts * n, k, torch.float32, 2, 0.2).reshape(experts, n, k).to(DEV)
    got = nk.mx_dots_experts(a, nk.mx_pack(stack), nk.experts_plan(chosen.to(DEV), experts))
    left, right = mx.rounded(a.cpu()), mx.rounded(stack.reshape(-1, k).cpu()).reshape(experts, n, k)
    for e in range(experts):
        token, slot = torch.nonzero(chosen == e, as_tuple=True)
        truth, magnitude = left[token] @ right[e].T, np.abs(left[token]) @ np.abs(right[e]).T
        mx.close(got[token, slot], truth, magnitude, k)
    assert not got[((chosen < 0) | (chosen >= experts)).to(DEV)].any()


@pytest.mark.parametrize("tokens,experts", [(3, 8), (200, 8), (900, 4)])  # few rows to an expert, some, many
def test_plan_of_other_sizes_gives_nans(tokens, experts):
    a, packed = torch.ones((tokens, 64), device=DEV), nk.mx_pack(torch.ones((experts, 80, 64), device=DEV))
    right = nk.experts_plan(torch.zeros((tokens, 2), dtype=torch.int32, device=DEV), experts)
    for other in (nk.experts_plan(torch.zeros((tokens + 1, 2), dtype=torch.int32, device=DEV), experts),
                  nk.experts_plan(torch.zeros((tokens, 2), dtype=torch.int32, device=DEV), experts + 1)):
        wrong = nk.ExpertsPlan(tokens, 2, experts, other.buffer)
        assert torch.isnan(nk.mx_dots_experts(a, packed, wrong)).all()
        assert torch.isnan(nk.mx_dots_experts(a, packed, wrong, torch.ones((tokens, 2), device=DEV))).all()
    assert (nk.mx_dots_experts(a, packed, right) == 64).all()


def test_no_tokens():
    packed = nk.mx_pack(torch.ones((4, 64, 64), device=DEV))
    plan = nk.experts_plan(torch.zeros((0, 2), dtype=torch.int32, device=DEV), 4)
    assert nk.mx_dots_experts(torch.ones((0, 64), device=DEV), packed, plan).shape == (0, 2, 64)


def test_layer_replays():
    """Router, plan and both products as one graph; replayed on other tokens, the same as the eager calls bit for bit."""
    tokens, experts, top_k, k, n = 48, 16, 4, 256, 192
    x = [normal(tokens, k, torch.bfloat16, seed, 0.0).to(DEV) for seed in (1, 2)]
    router = nk.dots_pack(normal(experts, k, torch.bfloat16, 3, 0.0).to(DEV), "bf16")
    up = nk.mx_pack(normal(experts * n, k, torch.float32, 4, 0.0).reshape(experts, n, k).to(DEV))
    down = nk.mx_pack(normal(experts * k, n, torch.float32, 5, 0.0).reshape(experts, k, n).to(DEV))
    logits = [nk.dots_packed(one, router) for one in x]

    def layer(tokens_in, scores):
        weights, chosen = nk.experts_route(scores, top_k)
        plan = nk.experts_plan(chosen, experts)
        hidden = torch.relu(nk.mx_dots_experts(tokens_in, up, plan, out_dtype=torch.bfloat16))
        return nk.mx_dots_experts(hidden.reshape(-1, n), down, plan, weights, out_dtype=torch.bfloat16)

    eager = [layer(*pair).clone() for pair in zip(x, logits)]
    held, held_logits = x[0].clone(), logits[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer(held, held_logits)
    for replay in range(4):
        held.copy_(x[replay % 2]), held_logits.copy_(logits[replay % 2])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager[replay % 2]), replay
        assert torch.equal(layer(x[0], logits[0]), eager[0])


def test_example_layer():
    """The layer of the example, from the router's scores to the sum by weight, against 64-bit forms step by step."""
    from numkong_amd.examples import experts_layer

    experts, hidden, depth, top_k, tokens = 12, 160, 224, 3, 50
    layer, (router, up, down) = experts_layer.make(experts, hidden, depth, top_k)
    x = normal(tokens, depth, torch.bfloat16, 9, 0.0).to(DEV)
    logits = layer.scores(x)
    exact = x.double() @ router.double().T
    assert ((logits.double() - exact).abs() <= depth * 2.0**-23 * (x.double().abs() @ router.double().abs().T)).all()
    y = layer(x)
    weights, chosen = nk.experts_route(logits, top_k)
    first = nk.mx_dots_experts(x, layer.up, nk.experts_plan(chosen, experts), out_dtype=torch.bfloat16)
    rows, matrices = mx.rounded(x), [mx.rounded(one) for one in up]
    choice = chosen.cpu().numpy()
    truth = np.stack([[matrices[e] @ rows[t] for e in choice[t]] for t in range(tokens)])
    magnitude = np.stack([[np.abs(matrices[e]) @ np.abs(rows[t]) for e in choice[t]] for t in range(tokens)])
    mx.close(first, truth, magnitude, depth)
    rows = mx.rounded(torch.relu(first).reshape(-1, hidden)).reshape(tokens, top_k, hidden)
    matrices = [mx.rounded(one) for one in down]
    parts = np.stack([[matrices[e] @ rows[t, i] for i, e in enumerate(choice[t])] for t in range(tokens)])
    sizes = np.stack([[np.abs(matrices[e]) @ np.abs(rows[t, i]) for i, e in enumerate(choice[t])] for t in range(tokens)])
    weight = weights.double().cpu().numpy()[..., None]
    mx.close(y, (parts * weight).sum(1), (sizes * weight).sum(1), hidden, top_k * 2.0**-23 * (np.abs(parts) * weight).sum(1))


def test_example_trains_a_router():
    from numkong_amd.examples import experts_layer

    wanted = torch.arange(200, device=DEV) % 10
    x = torch.nn.functional.one_hot(wanted, 16).float()
    first, last = experts_layer.train_router(x, wanted, 10, 3, 30, 5.0)
    assert last < first / 2  # separable tokens: the gradient leads there


def test_the_short_way_and_the_general_one_agree(monkeypatch):
    """Every call in its ordinary form, on the default stream and on another, against the same call the general way."""
    from numkong_amd import mx as binding

    x, b = normal(40, 200, torch.bfloat16, 1).to(DEV), normal(70, 200, torch.float32, 2).to(DEV)
    stack, logits = normal(6 * 33, 200, torch.float32, 3).reshape(6, 33, 200).to(DEV), normal(40, 6, torch.float32, 4, 0.0).to(DEV)
    bias, grad = torch.rand(6, device=DEV), torch.rand((40, 2), device=DEV)
    packed, packed_stack = nk.mx_pack(b), nk.mx_pack(stack)

    def calls():
        q = nk.mx_quantize(x)
        weights, chosen = nk.experts_route(logits, 2, "sigmoid", bias, groups=3, top_groups=2, scale=1.5)
        plan = nk.experts_plan(chosen, 6)
        found = [q.codes, q.scales, nk.mx_dequantize(q), nk.mx_dequantize(q, torch.float16), nk.mx_dots_packed(x, packed),
                 nk.mx_dots_packed(q, packed, out_dtype=torch.bfloat16), nk.mx_dots_packed(x[:, 3:103], nk.mx_pack(b[:, :100])), weights, chosen,
                 nk.experts_route_backward(grad, logits, chosen, "sigmoid", scale=1.5), plan.buffer.view(torch.int32)[:8],
                 nk.mx_dots_experts(x, packed_stack, plan), nk.mx_dots_experts(q, packed_stack, plan, out_dtype=torch.float16),
                 nk.mx_dots_experts(x, packed_stack, plan, weights, out_dtype=torch.bfloat16),
                 nk.mx_dots_experts(x.repeat_interleave(2, 0), packed_stack, plan, weights)]
        assert (plan.tokens, plan.top_k, plan.experts) == (40, 2, 6) and q.shape == (40, 200)
        return found

    assert binding._CALLS is not None
    short = calls()
    with torch.cuda.stream(torch.cuda.Stream()):
        elsewhere = calls()
    torch.cuda.synchronize()
    monkeypatch.setattr(binding, "_CALLS", None)
    for one, other, general in zip(short, elsewhere, calls()):
        assert one.dtype == general.dtype and one.shape == general.shape and one.stride() == general.stride()
        assert torch.equal(one, general) and torch.equal(other, general)
