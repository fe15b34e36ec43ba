"""More than one launch takes, and plans of many slots, on a real MI355X: tens of gigabytes each."""
import pytest

torch = pytest.importorskip("torch")

import numkong_amd as nk  # noqa: E402
from tests.test_experts_gpu import logits_of  # noqa: E402
from tests.test_mx_gpu import DEV, normal  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_is_given_back():
    """What these tests have held of the GPU's memory is not what later ones, some of which take times, find."""
    yield
    torch.cuda.empty_cache()


def test_more_rows_than_one_launch_takes():
    """2^28 rows of A, as floats and as codes: quantised pairs of values give sums that 32 bits hold."""
    rows, k, n = (1 << 28) + 37, 2, 3
    generator = torch.Generator(device=DEV).manual_seed(1)
    a = torch.randint(-40, 41, (rows, k), device=DEV, generator=generator, dtype=torch.int8).to(torch.bfloat16)
    b = torch.tensor([[1.0, -3.0], [0.5, 6.0], [4.0, 1.5]], device=DEV)
    packed, codes = nk.mx_pack(b), nk.mx_quantize(a)
    values = nk.mx_dequantize(codes)
    for left in (a, codes):
        got = nk.mx_dots_packed(left, packed)
        for column in range(n):
            assert torch.equal(got[:, column], values[:, 0] * b[column, 0] + values[:, 1] * b[column, 1])
        del got
    torch.cuda.empty_cache()


def test_more_columns_than_one_launch_takes():
    """A matrix of 2^28 columns against one row, and as an expert's against two: sums of quarters below 2^13, which 32 bits hold."""
    n, k = (1 << 28) + 100, 32
    generator = torch.Generator(device=DEV).manual_seed(2)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=generator)
    matrix = nk.MxMatrix(codes, torch.full((n, 1), 127, dtype=torch.uint8, device=DEV), k)
    a = normal(2, k, torch.float32, 3).to(DEV)
    left = nk.mx_dequantize(nk.mx_quantize(a))
    packed = nk.mx_pack(matrix)
    one = nk.mx_dots_packed(a[:1], packed)
    for first in (0, (1 << 26) - 500, (1 << 27) - 500, (1 << 27) + 12345, n - 1000):
        part = nk.MxMatrix(codes[first:first + 1000], matrix.scales[first:first + 1000], k)
        assert torch.equal(one[:, first:first + 1000], left[:1] @ nk.mx_dequantize(part).T.contiguous()), first
    chosen = torch.zeros((2, 1), dtype=torch.int32, device=DEV)
    both = nk.mx_dots_experts(a, nk.MxPackedMatrix(1, n, k, packed.buffer), nk.experts_plan(chosen, 1))
    assert torch.equal(both[0], one)
    for first in (0, (1 << 26) - 500, (1 << 27) - 500, (1 << 27) + 12345, n - 1000):
        part = nk.MxMatrix(codes[first:first + 1000], matrix.scales[first:first + 1000], k)
        assert torch.equal(both[1:, 0, first:first + 1000], left[1:] @ nk.mx_dequantize(part).T.contiguous()), first
    del one, both, packed, codes, matrix
    torch.cuda.empty_cache()


def test_more_tokens_than_one_launch_takes():
    """2^26 rows of logits, a wavefront each: the choices and the gradients of those at the ends of the launches and between are
    those of the same rows alone, bit for bit."""
    tokens, experts, top_k = (1 << 26) + 37, 257, 2
    rows = torch.tensor([0, 1, (1 << 25) - 1, 1 << 25, (1 << 25) + 1, (1 << 26) - 1, 1 << 26, tokens - 1], device=DEV)
    logits = torch.zeros((tokens, experts), dtype=torch.bfloat16, device=DEV)
    logits[rows] = logits_of(len(rows), experts, torch.bfloat16, 1).to(DEV)
    grad = torch.zeros((tokens, top_k), device=DEV)
    grad[rows] = normal(len(rows), top_k, torch.float32, 2, 0.0).to(DEV)
    weights, chosen = nk.experts_route(logits, top_k)
    few, few_chosen = nk.experts_route(logits[rows], top_k)
    assert torch.equal(weights[rows], few) and torch.equal(chosen[rows], few_chosen)
    assert int((chosen != torch.arange(top_k, device=DEV)).any(1).sum()) <= len(rows)  # (equal logits: the first two)
    got = nk.experts_route_backward(grad, logits, chosen)
    assert torch.equal(got[rows], nk.experts_route_backward(grad[rows], logits[rows], few_chosen))
    del logits, got
    torch.cuda.empty_cache()


def large_routing(slots, experts, popular):
    """One expert's share of all slots is `popular`; some slots have no expert."""
    generator = torch.Generator(device=DEV).manual_seed(slots)
    chosen = torch.randint(-1, experts, (slots,), dtype=torch.int32, device=DEV, generator=generator)
    chosen[torch.rand((slots,), device=DEV, generator=generator) < popular] = experts // 2
    return chosen.reshape(-1, 8)


@pytest.mark.parametrize("slots,experts,popular", [(1 << 16, 1024, 0.0), (66 << 10, 100, 0.5), ((1 << 17) + 8, 15, 0.0), (1 << 20, 128, 0.9), (1 << 20, 1024, 0.1),
                                                   (1 << 27, 8, 0.3)])
def test_plan_of_many_slots(slots, experts, popular):
    """The whole plan, by torch's own sort: more workgroups than add up one another's counts, tiles written by several of them."""
    chosen = large_routing(slots, experts, popular)
    words = nk.experts_plan(chosen, experts).buffer.view(torch.int32)
    flat = chosen.reshape(-1)
    bucket = torch.where((flat >= 0) & (flat < experts), flat, experts)
    counts = torch.bincount(bucket, minlength=experts + 1)
    sizes = (counts + 15) // 16 * 16
    starts = sizes.cumsum(0) - sizes
    tile_rows, tile_count, zero_tiles, first_zero, end_zero = words[3:8].tolist()
    assert (first_zero, end_zero) == (int(starts[-1]), int(starts[-1] + counts[-1]))
    assert torch.equal(words[8:8 + experts + 1], starts.int()) and int(words[9 + experts]) == end_zero
    by_bucket, slot_at = torch.sort(bucket, stable=True)
    row_of = starts[by_bucket] + torch.arange(slots, device=DEV) - (counts.cumsum(0) - counts)[by_bucket]
    order = torch.full((int(sizes.sum()),), -1, dtype=torch.int32, device=DEV)
    order[row_of] = slot_at.int()
    place = torch.empty(slots, dtype=torch.int32, device=DEV)
    place[slot_at] = torch.where(by_bucket < experts, row_of, -1).int()
    first, room = 8 + (experts + 2 + 3) // 4 * 4, (slots + min(slots, experts + 1) * 15 + 15) // 16 * 16
    assert torch.equal(words[first:first + len(order)], order)
    assert torch.equal(words[first + room:first + room + slots], place)
    tiles = words[(first + room + slots + 3) // 4 * 4:][:4 * (tile_count + zero_tiles)].reshape(-1, 4)
    of_bucket = (counts + tile_rows - 1) // tile_rows
    expert = torch.repeat_interleave(torch.arange(experts + 1, device=DEV), of_bucket)
    row = starts[expert] + tile_rows * (torch.arange(len(expert), device=DEV) - (of_bucket.cumsum(0) - of_bucket)[expert])
    want = torch.stack([expert, row, torch.minimum(row + tile_rows, (starts + counts)[expert])], 1).int()
    assert torch.equal(tiles[:, :3], want) and tile_count == int(of_bucket[:-1].sum())


def test_a_plan_takes_time_by_its_slots():
    """32 times the slots: about 32 times the work, where a thousand times would be work that grows with their square."""
    def milliseconds(slots):
        chosen = large_routing(slots, 8, 0.9)
        nk.experts_plan(chosen, 8)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        nk.experts_plan(chosen, 8)
        end.record()
        end.synchronize()
        return start.elapsed_time(end)

    assert milliseconds(1 << 27) < 4 * 32 * milliseconds(1 << 22)
