"""Microscaled 4-bit floats on a real MI355X: quantising, going back, products, against 64-bit forms (mx_support.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import numkong_amd as nk  # noqa: E402
from tests import mx_support as mx  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
FLOATS = [torch.float32, torch.bfloat16, torch.float16]


def normal(rows, depth, dtype, seed, spread=1.0):
    generator = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, depth), generator=generator) * torch.exp(spread * torch.randn((rows, 1), generator=generator))
    return x.to(dtype)


def strided(x, pad, offset=0):
    """The same matrix on the GPU, its rows `pad` values further apart and its start `offset` values into the allocation."""
    rows, depth = x.shape
    store = torch.full((rows * (depth + pad) + offset,), float("nan"), dtype=x.dtype, device=DEV)
    view = store[offset:].reshape(rows, depth + pad)[:, :depth]
    view.copy_(x)
    return view


def same_quantized(matrix, x):
    codes, scales = mx.quantize(x)
    np.testing.assert_array_equal(matrix.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(mx.unpacked(matrix.codes, x.shape[1]), codes)
    if x.shape[1] % 2:
        assert not (matrix.codes[:, -1].cpu().numpy() >> 4).any()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,depth,pad,offset", [(1, 1, 0, 0), (1, 31, 0, 0), (3, 32, 0, 0), (5, 33, 0, 0), (2, 127, 1, 1), (7, 129, 3, 0),
                                                   (16, 4096, 0, 0), (3, 1000, 24, 8), (260, 64, 0, 1), (1, 70000, 0, 0)])
def test_quantize(dtype, rows, depth, pad, offset):
    x = normal(rows, depth, dtype, rows + depth)
    same_quantized(nk.mx_quantize(strided(x, pad, offset)), x)


def test_quantize_every_bfloat16():
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16).reshape(-1, 1)
    # each value alone in a block, and beside a one, which decides the scale of what is smaller
    alone = torch.cat([x, torch.zeros((65536, 31), dtype=torch.bfloat16)], 1)
    same_quantized(nk.mx_quantize(alone.to(DEV)), alone)
    beside = alone.clone()
    beside[:, 17] = 1
    same_quantized(nk.mx_quantize(beside.to(DEV)), beside)


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_halfway_and_extreme(dtype):
    info = torch.finfo(dtype)
    halves = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.9, 6.0, -0.25, -0.75, -5.0, 0.0, -0.0, 4.0]).repeat(2)
    rows = [halves, halves * 2.0**-10, halves * info.tiny, torch.full((32,), info.max), torch.full((32,), -info.tiny / 2), torch.zeros(32)]
    for special in (float("nan"), float("inf"), -float("inf")):
        row = halves.clone()
        row[5] = special
        rows.append(row)
    x = torch.stack([row.to(dtype) for row in rows])
    x = torch.cat([x, x.flip(0)], 1)  # a bad block beside a good one
    matrix = nk.mx_quantize(x.to(DEV))
    same_quantized(matrix, x)
    back = nk.mx_dequantize(matrix).cpu().numpy()
    np.testing.assert_array_equal(back, mx.rounded(x).astype(np.float32))


def test_nothing_to_quantize():
    for shape in ((0, 64), (5, 0), (0, 0)):
        matrix = nk.mx_quantize(torch.zeros(shape, device=DEV))
        assert matrix.shape == shape and nk.mx_dequantize(matrix).shape == shape


@pytest.mark.parametrize("dtype", FLOATS)
def test_dequantize_every_code_and_scale(dtype):
    scales = np.arange(256, dtype=np.uint8).reshape(-1, 1)
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    matrix = nk.MxMatrix(torch.from_numpy(mx.packed(codes)).to(DEV), torch.from_numpy(scales).to(DEV), 32)
    got = nk.mx_dequantize(matrix, dtype).cpu()
    with np.errstate(over="ignore"):
        want = torch.from_numpy(mx.values(codes, scales)).to(dtype)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0, 9, -9), want.nan_to_num(0, 9, -9))
    assert torch.equal(torch.signbit(got[:255]), torch.signbit(want[:255]))


@pytest.mark.parametrize("depth,pad", [(1, 0), (7, 3), (33, 0), (1000, 1), (64, 16)])
def test_dequantize_rows_of_any_kind(depth, pad):
    rng = np.random.default_rng(depth)
    codes, scales = rng.integers(0, 16, (9, depth), dtype=np.uint8), rng.integers(100, 150, (9, (depth + 31) // 32), dtype=np.uint8)
    codes[:, depth:] = 0
    inside = torch.from_numpy(mx.packed(codes)).to(DEV)
    store = torch.full((9, inside.shape[1] + pad), 0xFF, dtype=torch.uint8, device=DEV)
    view = store[:, :inside.shape[1]]
    view.copy_(inside)
    out = strided(torch.zeros((9, depth)), pad, 1)
    result = nk.mx_dequantize(nk.MxMatrix(view, torch.from_numpy(scales).to(DEV), depth), out=out)
    assert result is out
    np.testing.assert_array_equal(out.cpu().numpy(), mx.values(codes, scales).astype(np.float32))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,depth,pad", [(8192, 4096, 0), (8300, 4093, 3), (8300, 4090, 22)])
def test_dequantize_past_the_caches(dtype, rows, depth, pad):
    """64 MiB and more at addresses of 16 bytes: rows in one piece, cut, and apart; nothing beside them written."""
    generator = torch.Generator(device=DEV).manual_seed(depth)
    codes = torch.randint(0, 256, (rows, depth // 2 + depth % 2), dtype=torch.uint8, device=DEV, generator=generator)
    scales = torch.randint(115, 135, (rows, (depth + 31) // 32), dtype=torch.uint8, device=DEV, generator=generator)
    scales[77, 5] = 255
    store = torch.full((rows, depth + pad), 77.0, dtype=dtype, device=DEV)
    out = store[:, :depth]
    assert out.data_ptr() % 16 == 0 and out.stride(0) * out.itemsize % 16 == 0 and rows * depth * out.itemsize >= 64 << 20
    nk.mx_dequantize(nk.MxMatrix(codes, scales, depth), dtype, out)
    one_each = torch.stack([codes & 15, codes >> 4], -1).flatten(1)[:, :depth]
    powers = torch.exp2(scales.double() - 127).masked_fill(scales == 255, float("nan"))
    want = (torch.tensor(mx.GRID, device=DEV)[one_each.long()] * powers.repeat_interleave(32, 1)[:, :depth]).to(dtype)
    torch.testing.assert_close(out, want, rtol=0.0, atol=0.0, equal_nan=True)
    out.fill_(77.0)
    assert bool((store == 77.0).all())


def product_of(a, b):
    left, right = mx.rounded(a), mx.rounded(b)
    return left @ right.T, np.abs(left) @ np.abs(right).T


SHAPES = [(1, 1, 1), (1, 17, 31), (2, 64, 32), (1, 256, 4096), (3, 65, 129), (15, 200, 512), (16, 130, 640), (17, 33, 127), (31, 100, 384),
          (32, 64, 1000), (33, 257, 96), (64, 192, 513), (65, 64, 128), (65, 300, 1), (129, 255, 500), (200, 131, 1024), (257, 129, 2100),
          (300, 1000, 160), (1030, 520, 700), (1030, 2100, 700), (8200, 300, 260), (2050, 8200, 130), (2049, 8001, 641)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k):
    for index, (dtype, out) in enumerate([(torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16), (torch.float32, torch.float16)]):
        a, b = normal(m, k, dtype, m + index, 0.3), normal(n, k, torch.float32, n + 7, 0.3)
        packed = nk.mx_pack(b.to(DEV))
        truth, magnitude = product_of(a, b)
        got = nk.mx_dots_packed(a.to(DEV), packed, out_dtype=out)
        assert got.dtype == out
        mx.close(got, truth, magnitude, k)
        # quantised beforehand: the same, bit for bit where the same kernel runs, and as near otherwise
        mx.close(nk.mx_dots_packed(nk.mx_quantize(a.to(DEV)), packed, out_dtype=out), truth, magnitude, k)


@pytest.mark.parametrize("m,n", [(1, 77), (9, 77), (40, 77), (100, 77), (300, 77), (1100, 2077), (2100, 8003)])
def test_product_of_views(m, n):
    """Rows that start anywhere, a result inside a larger matrix, nothing beside it written."""
    k = 333
    a, b = normal(m, k, torch.bfloat16, 1), normal(n, k, torch.bfloat16, 2)
    truth, magnitude = product_of(a, b)
    packed = nk.mx_pack(strided(b, 5, 1))
    for out_dtype in FLOATS:
        store = torch.full((m + 2, n + 9), 77.0, dtype=out_dtype, device=DEV)
        out = store[1:-1, 3:3 + n]
        assert nk.mx_dots_packed(strided(a, 1, 1), packed, out=out) is out
        mx.close(out, truth, magnitude, k)
        store[1:-1, 3:3 + n] = 77.0
        assert bool((store == 77.0).all())


def test_results_whose_rows_share_memory_are_refused():
    a, packed, matrix = torch.ones((4, 64), device=DEV), nk.mx_pack(torch.ones((8, 64), device=DEV)), nk.mx_quantize(torch.ones((4, 64), device=DEV))
    stack, plan = nk.mx_pack(torch.ones((2, 8, 64), device=DEV)), nk.experts_plan(torch.zeros((4, 1), dtype=torch.int32, device=DEV), 2)
    weights = torch.ones((4, 1), device=DEV)
    row = torch.zeros(100, device=DEV)
    for step in (0, 1, 7):
        out = row.as_strided((4, 8), (step, 1))
        with pytest.raises(ValueError, match="share memory"):
            nk.mx_dots_packed(a, packed, out=out)
        with pytest.raises(ValueError, match="share memory"):
            nk.mx_dots_experts(a, stack, plan, weights, out=out)
        with pytest.raises(ValueError, match="share memory"):
            nk.mx_dequantize(matrix, out=row.as_strided((4, 64), (step, 1)))
    out = row.as_strided((4, 8), (8, 1))
    assert bool((nk.mx_dots_packed(a, packed, out=out) == 64).all()) and bool((nk.mx_dots_packed(a[:1], packed, out=row.as_strided((1, 8), (0, 1))) == 64).all())


@pytest.mark.parametrize("m,n", [(1, 90), (20, 90), (70, 90), (260, 90), (1100, 2100), (2100, 8200)])
def test_special_values_stay_in_their_rows(m, n):
    k = 200
    a, b = normal(m, k, torch.float32, 3), normal(n, k, torch.float32, 4)
    a[m // 2, 77], b[5, 199], b[60, 0] = float("inf"), float("nan"), -float("inf")
    a[0, 32:64] = 0  # a NaN of the other side meets zeros only
    truth, magnitude = product_of(a, b)
    got = nk.mx_dots_packed(a.to(DEV), nk.mx_pack(b.to(DEV))).double().cpu().numpy()
    nans = np.zeros((m, n), dtype=bool)
    nans[m // 2], nans[:, 5], nans[:, 60] = True, True, True
    np.testing.assert_array_equal(np.isnan(got), nans)
    np.testing.assert_array_equal(np.isnan(truth), nans)
    assert (np.abs(got - truth)[~nans] <= mx.sum_bound(k, np.nan_to_num(magnitude))[~nans] + 2.0**-24 * np.abs(truth[~nans])).all()


def test_deep_products_in_whole_rounds():
    """Two tiles of 256 x 256 to a compute unit, the last ones cut on both sides; rows that start anywhere, a NaN among them, a
    result inside a larger matrix. (The 64-bit products of the plain form's values are made on the GPU.)"""
    m, n, k = 8100, 4050, 6200
    a, b = normal(m, k, torch.bfloat16, 1, 0.3), normal(n, k, torch.bfloat16, 2, 0.3)
    a[4000, 6199], b[77, 0] = float("nan"), float("inf")
    left, right = torch.from_numpy(mx.rounded(a)).to(DEV), torch.from_numpy(mx.rounded(b)).to(DEV).T.contiguous()
    truth, magnitude = (left @ right).cpu().numpy(), (left.abs() @ right.abs()).cpu().numpy()
    packed = nk.mx_pack(b.to(DEV))
    for out_dtype in FLOATS:
        store = torch.full((m + 2, n + 9), 77.0, dtype=out_dtype, device=DEV)
        out = store[1:-1, 3:3 + n]
        nk.mx_dots_packed(strided(a, 1, 1), packed, out=out)
        mx.close(out, truth, magnitude, k)
        again = nk.mx_dots_packed(a.to(DEV), packed, out_dtype=out_dtype)
        assert torch.equal(again.nan_to_num(0.0), out.nan_to_num(0.0))
        store[1:-1, 3:3 + n] = 77.0
        assert bool((store == 77.0).all())


def test_scales_of_every_size():
    """Products of scales past the range of 32-bit floats overflow and vanish as the products of the values do."""
    scale_pairs = [(127, 127), (0, 254), (0, 127), (60, 67), (254, 126), (200, 180), (1, 100), (0, 0)]
    codes = np.full((1, 32), 2, dtype=np.uint8)  # ones
    for left, right in scale_pairs:
        matrices = [nk.MxMatrix(torch.from_numpy(mx.packed(codes)).to(DEV), torch.tensor([[s]], dtype=torch.uint8, device=DEV), 32)
                    for s in (left, right)]
        got = float(nk.mx_dots_packed(matrices[0], nk.mx_pack(matrices[1]))[0, 0])
        with np.errstate(over="ignore"):
            want = float(np.float32(32 * 2.0 ** (left + right - 254)))
        assert got == want, (left, right)


@pytest.mark.parametrize("m,n", [(8, 40), (30, 700), (64, 700), (1100, 2100)])
def test_scales_of_every_pair(m, n):
    """The same of all pairs of some scales, in each kernel's instruction; the blocks of a row differ, and one is left of each sum:
    32 equal products, whose sums in 32 bits are exact in any order unless a product is below the smallest number, 2^-149; then
    each of 32 additions may be off by half of that."""
    some = np.array([0, 1, 2, 60, 67, 100, 126, 127, 128, 180, 200, 252, 253, 254], dtype=np.int64)
    left, right = some[np.arange(m) * 5 % len(some)], some[np.arange(n) * 3 % len(some)]
    codes, scales = np.zeros((m, 640), dtype=np.uint8), np.full((m, 20), 127, dtype=np.uint8)
    block = np.arange(m) * 7 % 20
    for row in range(m):
        codes[row, 32 * block[row]:32 * block[row] + 32] = 2  # ones
        scales[row, block[row]] = left[row]
    b_codes, b_scales = np.full((n, 640), 2, dtype=np.uint8), np.repeat(right.astype(np.uint8)[:, None], 20, 1)
    make = lambda c, e: nk.MxMatrix(torch.from_numpy(mx.packed(c)).to(DEV), torch.from_numpy(e).to(DEV), 640)  # noqa: E731
    got = nk.mx_dots_packed(make(codes, scales), nk.mx_pack(make(b_codes, b_scales))).cpu().numpy()
    power = (left[:, None] + right[None, :] - 254).astype(np.float64)
    with np.errstate(over="ignore"):
        want = (32 * 2.0 ** power).astype(np.float32)
    held = power >= -149
    np.testing.assert_array_equal(got[held], want[held])
    assert (np.abs(got.astype(np.float64) - 32 * 2.0 ** power)[~held] <= 32 * 2.0**-150).all()


@pytest.mark.parametrize("out", FLOATS)
@pytest.mark.parametrize("m,n", [(40, 700), (1100, 2100), (2100, 8200)])
def test_no_depth_and_other_images_of_many_rows(m, n, out):
    """Zeros where there is nothing to add up, NaNs where the image is one of something else, and nothing beside them."""
    for k, packed, right in ((0, nk.mx_pack(torch.ones((n, 0), device=DEV)), 0.0),
                             (200, nk.MxPackedMatrix(1, n, 200, nk.mx_pack(torch.ones((n, 256), device=DEV)).buffer), float("nan"))):
        store = torch.full((m + 2, n + 9), 77.0, dtype=out, device=DEV)
        view = store[1:-1, 3:3 + n]
        nk.mx_dots_packed(torch.ones((m, k), device=DEV), packed, out=view)
        assert torch.equal(view.isnan(), torch.full_like(view, right).isnan()) and not view.nan_to_num(0.0).any()
        view.fill_(77.0)
        assert bool((store == 77.0).all())


def test_no_depth_and_no_rows():
    for m, n, k in ((3, 5, 0), (0, 5, 64), (3, 0, 64), (100, 5, 0)):
        got = nk.mx_dots_packed(torch.ones((m, k), device=DEV), nk.mx_pack(torch.ones((n, k), device=DEV)))
        assert got.shape == (m, n) and not got.any()


@pytest.mark.parametrize("shape", [(3, 4, 0), (0, 4, 64), (3, 0, 64), (0, 0, 0)])
def test_stacks_of_nothing(shape):
    packed = nk.mx_pack(torch.ones(shape, device=DEV))
    assert (packed.count, packed.width, packed.depth) == shape
    if shape[0]:
        plan = nk.experts_plan(torch.zeros((5, 2), dtype=torch.int32, device=DEV), shape[0])
        got = nk.mx_dots_experts(torch.ones((5, shape[2]), device=DEV), packed, plan)
        assert got.shape == (5, 2, shape[1]) and not got.any()
        got = nk.mx_dots_experts(torch.ones((5, shape[2]), device=DEV), packed, plan, torch.ones((5, 2), device=DEV))
        assert got.shape == (5, shape[1]) and not got.any()


def test_image_of_other_sizes_gives_nans():
    lib = nk.library()
    packed = nk.mx_pack(torch.ones((64, 256), device=DEV))
    wrong = nk.MxPackedMatrix(1, 64, 200, packed.buffer)
    for m in (1, 100):
        assert bool(nk.mx_dots_packed(torch.ones((m, 200), device=DEV), wrong).isnan().all())
    assert lib is not None


def test_image_moves():
    a, b = normal(5, 100, torch.float32, 5).to(DEV), normal(50, 100, torch.float32, 6).to(DEV)
    packed = nk.mx_pack(b)
    moved = nk.MxPackedMatrix(packed.count, packed.width, packed.depth, packed.buffer.cpu().to(DEV))
    assert torch.equal(nk.mx_dots_packed(a, packed), nk.mx_dots_packed(a, moved))


def test_host_operands():
    a, b = normal(5, 100, torch.float32, 5), normal(50, 100, torch.float32, 6)
    packed = nk.mx_pack(b.numpy())
    device = nk.mx_dots_packed(a.to(DEV), packed)
    host, array = nk.mx_dots_packed(a, packed), nk.mx_dots_packed(a.numpy(), packed)
    assert host.device.type == "cpu" and isinstance(array, np.ndarray)
    np.testing.assert_array_equal(array, device.cpu().numpy())
    np.testing.assert_array_equal(host.numpy(), array)
    out = np.zeros((5, 50), np.float32)
    assert nk.mx_dots_packed(a.numpy(), packed, out=out) is out
    np.testing.assert_array_equal(out, array)
    matrix = nk.mx_quantize(a.numpy())
    np.testing.assert_array_equal(mx.unpacked(np.asarray(matrix.codes), 100), mx.quantize(a)[0])
    np.testing.assert_array_equal(nk.mx_dots_packed(matrix, packed), array)
    np.testing.assert_array_equal(nk.mx_dequantize(matrix), mx.rounded(a).astype(np.float32))


@pytest.mark.parametrize("m,n", [(4, 200), (50, 200), (300, 200), (1100, 2100), (2100, 8200)])
def test_streams_and_replays(m, n):
    """Work follows the current stream; a captured call is replayed on new values, with eager work between."""
    a, b = normal(m, 640, torch.bfloat16, 8).to(DEV), normal(n, 640, torch.bfloat16, 9).to(DEV)
    packed = nk.mx_pack(b)
    eager = nk.mx_dots_packed(a, packed).clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        moved = torch.empty_like(a)
        moved.copy_(a)
        apart = nk.mx_dots_packed(moved, packed)
    side.synchronize()
    assert torch.equal(apart, eager)
    graph, held = torch.cuda.CUDAGraph(), a.clone()
    with torch.cuda.graph(graph):
        captured = nk.mx_dots_packed(held, packed)
    for replay in range(4):
        held.copy_(a if replay % 2 == 0 else -a)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager if replay % 2 == 0 else -eager), replay
        nk.mx_dots_packed(a, packed)


def test_offsets_past_32_bits():
    """Images and operands of more than 4 GiB: the last rows and columns are where they belong."""
    n, k = 70000, 131072  # 4.6 GB of codes
    generator = torch.Generator(device=DEV).manual_seed(1)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=generator)
    scales = torch.full((n, k // 32), 120, dtype=torch.uint8, device=DEV)
    matrix = nk.MxMatrix(codes, scales, k)
    small = normal(3, k, torch.bfloat16, 10)
    rows = [0, 1, 32767, 65535, 69999]
    picked = mx.values(mx.unpacked(codes[rows], k), scales[rows].cpu().numpy())
    left = mx.rounded(small)
    truth, magnitude = left @ picked.T, np.abs(left) @ np.abs(picked).T
    mx.close(nk.mx_dots_packed(small.to(DEV), nk.mx_pack(matrix))[:, rows], truth, magnitude, k)
    mx.close(nk.mx_dots_packed(matrix, nk.mx_pack(small.to(DEV)))[rows].T, truth, magnitude, k)
