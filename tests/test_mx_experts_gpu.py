"""What routing and the experts' products do at their edges on a real MI355X: masks in groups, gradients, refusals, nothing to add up."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import numkong_amd as nk  # noqa: E402
from tests.test_experts_gpu import logits_of, routing  # noqa: E402
from tests.test_mx_gpu import DEV, normal  # noqa: E402

pytestmark = pytest.mark.gpu


def choice_of_two(selection, groups, top_groups):
    """64-bit selection scores where groups are picked by the sum of their best two; of one that can be chosen, by that one."""
    inside = selection.reshape(len(selection), groups, -1)
    best = np.sort(inside, 2)[:, :, ::-1]
    low = float(torch.finfo(torch.float32).min)
    second = np.where(np.isneginf(best[:, :, 1]), 0.0, best[:, :, 1])
    of_group = np.where(np.isneginf(best[:, :, 0]), -np.inf, np.maximum(best[:, :, 0] + second, low))
    order = np.argsort(-of_group, axis=1, kind="stable")
    keep = np.zeros_like(of_group, dtype=bool)
    np.put_along_axis(keep, order[:, :top_groups], True, 1)
    return np.where(keep[:, :, None], inside, -np.inf).reshape(selection.shape)


@pytest.mark.parametrize("tokens", [40, 4200])  # a wavefront for a token, and 16 lanes
@pytest.mark.parametrize("experts,groups,top_groups", [(64, 8, 4), (64, 8, 1), (30, 5, 2), (100, 5, 2), (144, 9, 3), (256, 8, 3), (512, 64, 20), (1000, 50, 7)])
def test_masked_experts_in_groups(tokens, experts, groups, top_groups):
    """Whatever is masked, the groups that stay are those that have something to choose, by two best of it. Logits are whole
    numbers, scores with a bias ones and quarters: sums of two are exact, and ties go to the lowest."""
    generator = torch.Generator().manual_seed(experts + groups)
    logits = torch.randint(-20, 21, (tokens, experts), generator=generator).float()
    masked = torch.rand((tokens, experts), generator=generator) < torch.rand((tokens, 1), generator=generator) ** 0.2
    logits[masked] = -float("inf")
    size = experts // groups
    logits[0], logits[0, -4] = -float("inf"), 3.0  # a single expert, in the last group
    logits[1], logits[1, -size:] = -float("inf"), torch.finfo(torch.float32).min  # lowest numbers are numbers, their sum as well
    logits[2], logits[2, -1], logits[2, 0] = -float("inf"), -20.0, -19.0
    logits[3] = -float("inf")
    logits[4], logits[4, -2] = -float("inf"), float("inf")
    logits[4, -size - 1] = 5.0
    bias = torch.randint(-3, 4, (experts,), generator=generator) / 4
    for score, of in (("softmax", None), ("sigmoid", bias)):
        x = logits if of is None else torch.where(logits.isneginf(), logits, 60.0)
        selection = x.double().numpy() if of is None else np.where(np.isneginf(x.numpy()), -np.inf, 1.0 + bias.double().numpy())
        selection = choice_of_two(selection, groups, top_groups)
        order = np.argsort(-selection, axis=1, kind="stable")[:, :4]
        there = ~np.isneginf(np.take_along_axis(selection, order, 1))
        weights, chosen = nk.experts_route(x.to(DEV), 4, score, None if of is None else of.to(DEV), groups, top_groups, 2)
        np.testing.assert_array_equal(chosen.cpu().numpy(), np.where(there, order, -1))
        assert (weights.cpu().numpy()[~there] == 0).all()
        assert chosen[0].tolist() == [experts - 4, -1, -1, -1] and int(chosen[1, 0]) >= experts - size and int(chosen[4, 0]) >= 0


def test_groups_by_scores():
    """Groups by the sum of two scores, not of two logits, are what a bias of zeros gives."""
    logits = torch.tensor([[6.0, -6.0, 0.1, 0.1], [0.0, 9.0, 4.0, 4.5], [-3.0, 2.0, 0.0, 0.0]])
    s = torch.sigmoid(logits.double()).reshape(3, 2, 2).sum(2)
    _, chosen = nk.experts_route(logits.to(DEV), 2, "sigmoid", torch.zeros(4, device=DEV), 2, 1, 2)
    assert torch.equal(chosen.cpu() // 2, s.argmax(1, keepdim=True).expand(3, 2))
    _, chosen = nk.experts_route(logits.to(DEV), 2, "sigmoid", None, 2, 1, 2)
    assert torch.equal(chosen.cpu() // 2, logits.reshape(3, 2, 2).sum(2).argmax(1, keepdim=True).expand(3, 2))


@pytest.mark.parametrize("short_way", [True, False])
def test_what_routing_refuses(monkeypatch, short_way):
    """Before room is made for it, and by both ways."""
    from numkong_amd import mx as binding

    if not short_way:
        monkeypatch.setattr(binding, "_CALLS", None)
    logits = torch.zeros((1000, 64), device=DEV)
    for top_k in (0, 65, 1 << 40, -1):
        with pytest.raises(nk.NumKongAmdError, match="1 to 1024 experts"):
            nk.experts_route(logits, top_k)
    for scale in (1e39, -float("inf"), float("nan")):
        with pytest.raises(ValueError, match="finite"):
            nk.experts_route(logits, 2, scale=scale)
    with pytest.raises(ValueError, match="32-bit"):
        nk.experts_route(logits, 2, groups=(1 << 32) + 1)
    with pytest.raises(nk.NumKongAmdError, match="groups"):
        nk.experts_route(logits, 2, groups=-1)


@pytest.mark.parametrize("short_way", [True, False])
@pytest.mark.parametrize("score,biased,groups,renormalize,dtype", [("softmax", False, 1, True, torch.float32), ("sigmoid", True, 4, True, torch.bfloat16),
                                                                   ("sigmoid", False, 1, False, torch.float16), ("softmax", True, 2, False, torch.float32)])
def test_autograd_follows_the_weights(monkeypatch, score, biased, groups, renormalize, dtype, short_way):
    """Weights that a loss is made of hand their gradient on to whatever made the logits, by experts_route_backward."""
    from numkong_amd import mx as binding

    if not short_way:
        monkeypatch.setattr(binding, "_CALLS", None)
    source, grad = logits_of(30, 24, torch.float32, 1).to(DEV).requires_grad_(), normal(30, 3, torch.float32, 2, 0.0).to(DEV)
    bias = torch.rand(24, device=DEV).requires_grad_() if biased else None
    kind = dict(bias=bias, groups=groups, top_groups=max(1, groups // 2), group_top=2 if groups > 1 else 1)
    logits = (2 * source).to(dtype)
    weights, chosen = nk.experts_route(logits, 3, score, renormalize=renormalize, scale=1.5, **kind)
    with torch.no_grad():
        plain, plain_chosen = nk.experts_route(logits, 3, score, renormalize=renormalize, scale=1.5, **kind)
    assert weights.requires_grad and not chosen.requires_grad and not plain.requires_grad
    assert torch.equal(weights, plain) and torch.equal(chosen, plain_chosen)
    (weights * grad).sum().backward()
    want = nk.experts_route_backward(grad, logits.detach(), chosen, score, renormalize, 1.5)
    assert torch.equal(source.grad, 2 * want.float()) and (not biased or bias.grad is None)
    again = nk.experts_route(logits.detach().requires_grad_(), 3, score)[0].sum()  # (its gradient is one number for all)
    again.backward()
    host = logits.detach().cpu().requires_grad_()
    (nk.experts_route(host, 3, score, renormalize=renormalize, scale=1.5, **{**kind, "bias": bias.detach().cpu() if biased else None})[0] * grad.cpu()).sum().backward()
    assert torch.equal(host.grad, want.cpu())
    leaf = logits.detach().requires_grad_()
    first, = torch.autograd.grad(nk.experts_route(leaf, 3, score)[0].square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()


@pytest.mark.parametrize("short_way", [True, False])
def test_products_say_that_they_have_no_gradient(monkeypatch, short_way):
    from numkong_amd import mx as binding

    if not short_way:
        monkeypatch.setattr(binding, "_CALLS", None)
    a, packed, stack = normal(6, 64, torch.float32, 1).to(DEV), nk.mx_pack(torch.ones((8, 64), device=DEV)), nk.mx_pack(torch.ones((4, 8, 64), device=DEV))
    plan, weights = nk.experts_plan(torch.zeros((6, 2), dtype=torch.int32, device=DEV), 4), torch.rand((6, 2), device=DEV)
    leaf, weight = a.clone().requires_grad_(), weights.clone().requires_grad_()
    for name, tracked, plain in (("mx_dots_packed", lambda **o: nk.mx_dots_packed(leaf, packed, **o), lambda: nk.mx_dots_packed(a, packed)),
                                 ("mx_dots_experts", lambda **o: nk.mx_dots_experts(leaf, stack, plan, **o), lambda: nk.mx_dots_experts(a, stack, plan)),
                                 ("mx_dots_experts", lambda **o: nk.mx_dots_experts(a, stack, plan, weight, **o), lambda: nk.mx_dots_experts(a, stack, plan, weights))):
        want, got = plain(), tracked()
        assert torch.equal(got, want) and got.requires_grad and not want.requires_grad
        with pytest.raises(nk.NumKongAmdError, match=name + " has no gradient"):
            got.sum().backward()
        with pytest.raises(nk.NumKongAmdError, match="out="):
            tracked(out=torch.empty_like(want))
        with torch.no_grad():
            assert not tracked().requires_grad and torch.equal(tracked(out=torch.empty_like(want)), want)
    assert leaf.grad is None and weight.grad is None
    array = nk.mx_dots_experts(a.cpu().numpy(), stack, plan, weights.cpu().requires_grad_())  # (an array holds no gradient)
    np.testing.assert_array_equal(array, nk.mx_dots_experts(a, stack, plan, weights).cpu().numpy())


@pytest.mark.parametrize("short_way", [True, False])
def test_images_and_plans_are_as_large_as_their_sizes_say(monkeypatch, short_way):
    """Parts of an image or a plan, and buffers that are not in one piece, are refused before a kernel looks for the rest."""
    from numkong_amd import mx as binding

    a, packed, stack = torch.ones((6, 64), device=DEV), nk.mx_pack(torch.ones((80, 64), device=DEV)), nk.mx_pack(torch.ones((8, 80, 64), device=DEV))
    plan = nk.experts_plan(torch.zeros((6, 2), dtype=torch.int32, device=DEV), 8)
    if not short_way:
        monkeypatch.setattr(binding, "_CALLS", None)

    def parts(buffer):
        twice = torch.zeros(2 * buffer.numel(), dtype=torch.uint8, device=DEV)
        return buffer[:0], buffer[:1], buffer[:-1], buffer[:64].clone(), twice[::2]

    for part in parts(packed.buffer):
        with pytest.raises(ValueError, match="packed image"):
            nk.mx_dots_packed(a, nk.MxPackedMatrix(1, 80, 64, part))
    for width in (1 << 30, 1 << 31, 1 << 40):
        with pytest.raises(ValueError, match="packed image"):
            nk.mx_dots_packed(a, nk.MxPackedMatrix(1, width, 64, packed.buffer))
    for weights in (None, torch.ones((6, 2), device=DEV)):
        for part in parts(stack.buffer):
            with pytest.raises(ValueError, match="packed image"):
                nk.mx_dots_experts(a, nk.MxPackedMatrix(8, 80, 64, part), plan, weights)
        for part in parts(plan.buffer):
            with pytest.raises(ValueError, match="the plan"):
                nk.mx_dots_experts(a, stack, nk.ExpertsPlan(6, 2, 8, part), weights)
        larger = [torch.cat([one, one.new_zeros(100)]) for one in (stack.buffer, plan.buffer)]
        got = nk.mx_dots_experts(a, nk.MxPackedMatrix(8, 80, 64, larger[0]), nk.ExpertsPlan(6, 2, 8, larger[1]), weights)
        assert bool((got == (64 if weights is None else 128)).all())


@pytest.mark.parametrize("tokens,experts", [(3, 8), (200, 8), (900, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_depth_and_other_images(tokens, experts, dtype):
    """Few rows to an expert, some, many; some without an expert, the sums by weight as well."""
    chosen = torch.from_numpy(routing(tokens, 2, experts, "some", 1)).to(DEV)
    there = (chosen >= 0) & (chosen < experts)
    plan, weights = nk.experts_plan(chosen, experts), torch.ones((tokens, 2), device=DEV)
    empty = nk.mx_pack(torch.ones((experts, 300, 0), device=DEV))
    other = nk.MxPackedMatrix(experts, 300, 60, nk.mx_pack(torch.ones((experts, 300, 64), device=DEV)).buffer)
    for k, packed in ((0, empty), (60, other)):
        a = torch.ones((tokens, k), device=DEV)
        rows = nk.mx_dots_experts(a, packed, plan, out_dtype=dtype)
        sums = nk.mx_dots_experts(a, packed, plan, weights, out_dtype=dtype)
        if k:
            assert bool(rows[there].isnan().all()) and bool(sums[there.any(1)].isnan().all()) and not sums[~there.any(1)].any()
        else:
            assert rows.shape == (tokens, 2, 300) and not rows.any() and not sums.any()
