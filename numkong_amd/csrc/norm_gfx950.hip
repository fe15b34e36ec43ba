/**
 *  @brief 8-bit blocks and the root mean square norm with its gradients on gfx950.
 *  @file numkong_amd/csrc/norm_gfx950.hip
 *
 *  Implements the first half of <numkong_amd/dense.h>. The norm of a row t is y = t w s, s = 1 / sqrt(mean(t^2) + eps); with g the
 *  gradient of y, that of t is s (g w - t s^2 mean(g w t)) and that of w the sum over the rows of g t s.
 */
#include "dense_gfx950.hpp"

namespace nk_gfx950 {
namespace {

/** Calls `launch(first row, rows)` for pieces of `rows` that one launch holds, `threads` for each row. */
template <class Launch>
int in_pieces(uint64_t rows, uint64_t threads, char const *what, Launch launch) {
    uint64_t const most = threads < kMostThreads ? kMostThreads / threads / 4 * 4 : 1;
    for (uint64_t first = 0; first < rows; first += most) {
        launch(first, rows - first < most ? rows - first : most);
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, what);
    }
    return 0;
}

// ---- 8-bit blocks --------------------------------------------------------------------------------------------------

__global__ __launch_bounds__(256) void mx8_quantize_kernel(QuantizeArgs p) { quantize_stretches(p, blockIdx.x); }

__global__ __launch_bounds__(256) void mx8_dequantize_kernel(uint8_t const *codes, uint64_t codes_stride, uint8_t const *scales, uint64_t scales_stride,
                                                             uint64_t stretches, uint32_t each, uint32_t k, uint32_t kind, uint8_t *x, uint64_t x_stride) {
    uint64_t const at = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= stretches) return;
    uint64_t const row = at / each;
    uint32_t const col = (uint32_t)(at - row * each) * 512 + (threadIdx.x & 63) * 8;
    if (col >= k) return;
    uint8_t const *const from = codes + row * codes_stride + col;
    v2u words = {0, 0};
    if (col + 8 <= k) {
        typedef v2u __attribute__((aligned(1))) v2u_anywhere;
        words = *(v2u_anywhere const *)from;
    } else
        for (uint32_t i = 0; i < k - col; ++i) words[i / 4] |= (uint32_t)from[i] << 8 * (i % 4);
    float const power = scale_of(scales[row * scales_stride + col / 32]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float four[4];
        widen_e4m3(words[i], four);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = four[j] * power;
    }
    store_8(kind, x + row * x_stride, col, v, k - col);
}

// ---- the norm ------------------------------------------------------------------------------------------------------

/** The sum of a value over the threads of a row, in all of them; `sums` has room for 16 wavefronts of each row of the workgroup. The
 *  order is fixed: lanes by halves, then wavefronts in turn. */
template <class V>
__device__ __forceinline__ V row_sum(V v, V *sums) {
#pragma unroll
    for (int step = 32; step; step >>= 1) v += __shfl_xor(v, step);
    if (blockDim.x > 64) { // (then the workgroup has one row)
        if (!(threadIdx.x & 63)) sums[threadIdx.x >> 6] = v;
        __syncthreads();
        v = sums[0];
        for (uint32_t i = 1; i < blockDim.x / 64; ++i) v += sums[i];
    }
    return v;
}

struct NormArgs {
    uint8_t const *x, *residual;
    uint8_t *total;
    uint64_t x_stride, residual_stride, total_stride;
    void const *weight;
    uint8_t *y, *scales;
    uint64_t y_stride, scales_stride;
    uint64_t rows;
    uint32_t k, weight_kind, y_kind;
    float eps;
};

/** A number of 64 bits as 32: of its two neighbours the odd one where it is neither of them. What is then rounded to fewer bits comes
 *  out as if it had been in one step. */
__device__ __forceinline__ float to_odd(double v) {
    float const near = (float)v;
    double const back = (double)near;
    uint32_t bits = __float_as_uint(near);
    if (back != v && !(bits & 1)) bits += fabs(back) < fabs(v) ? 1u : ~0u; // an even neighbour: the odd one is on the other side of v
    return __uint_as_float(bits);
}

template <bool MX8>
struct WideOf {
    typedef double type;
};
template <>
struct WideOf<false> {
    typedef float type;
};

/**
 *  Threads (x) share a row, P times eight values each; rows of at most 64 x 8 P values take a wavefront each, four a
 *  workgroup (y). A row is read once and stays in registers between the sum and the result; memory is what bounds it.
 *  With mx8 results everything behind the total is in 64 bits, and the codes are those of the exact y: they depend on which side of a
 *  border a value is, and 32 bits would put some of a large matrix's on the wrong one.
 */
template <class T, int P, bool MX8>
__global__ __launch_bounds__(1024) void rms_norm_kernel(NormArgs p) {
    typedef typename WideOf<MX8>::type Wide;
    __shared__ Wide sums[16];
    uint64_t const row = (uint64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= p.rows) return; // (a whole wavefront, and only where rows are not shared between wavefronts)
    float t[P][8];
    Wide sum = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        uint32_t const col = (i * blockDim.x + threadIdx.x) * 8;
        load_adjacent((T const *)(p.x + row * p.x_stride), col, p.k, t[i]);
        if (p.residual) {
            float r[8];
            load_adjacent((T const *)(p.residual + row * p.residual_stride), col, p.k, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[i][j] = (float)(T)(t[i][j] + r[j]);
            if (col < p.k) store_some((T *)(p.total + row * p.total_stride) + col, t[i], p.k - col);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += (Wide)t[i][j] * (Wide)t[i][j];
    }
    sum = row_sum(sum, sums);
    Wide const scale = (Wide)1 / sqrt(sum / (Wide)p.k + (Wide)p.eps);
#pragma unroll
    for (int i = 0; i < P; ++i) {
        uint32_t const col = (i * blockDim.x + threadIdx.x) * 8;
        float w[8], y[8];
        if (p.weight) load_adjacent(p.weight_kind, p.weight, col, p.k, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            Wide const v = p.weight ? (Wide)t[i][j] * scale * (Wide)w[j] : (Wide)t[i][j] * scale;
            if constexpr (MX8) y[j] = to_odd(v);
            else y[j] = v;
        }
        if constexpr (MX8) {
            uint32_t exponent;
            v2u const codes = quantize_8(y, exponent);
            if (col < p.k) {
                store_codes(p.y + row * p.y_stride + col, codes, p.k - col);
                if (!(threadIdx.x & 3)) p.scales[row * p.scales_stride + col / 32] = (uint8_t)exponent;
            }
        } else if (col < p.k) store_8(p.y_kind, p.y + row * p.y_stride, col, y, p.k - col);
    }
}

struct NormBackwardArgs {
    uint8_t const *total, *grad, *grad_total;
    uint8_t *grad_x;
    uint64_t total_stride, grad_stride, grad_total_stride, grad_x_stride;
    void const *weight;
    float *partial; // (grid, k): each workgroup's part of the weight's gradient, or NULL
    uint64_t rows;
    uint32_t k, weight_kind, grad_kind;
    float eps;
};

/** Eight adjacent values as they lie in memory, so that a row can be on its way while the one before is worked on; HALF: of 16 bits for certain. */
template <bool HALF>
struct Raw {
    v4u low, high; // (high: of f32 only)
    __device__ __forceinline__ void load(uint32_t kind, uint8_t const *row, uint32_t col, uint32_t k) {
        uint32_t const size = HALF ? 2 : bytes_of(kind);
        uint8_t const *const at = row + (uint64_t)col * size;
        if (col + 8 <= k) {
            low = *(v4u_anywhere const *)at;
            if (size == 4) high = *(v4u_anywhere const *)(at + 16);
            return;
        }
        uint32_t words[8] = {};
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (col + i < k) {
                if (size == 4) words[i] = ((uint32_t const *)at)[i];
                else words[i / 2] |= (uint32_t)((uint16_t const *)at)[i] << 16 * (i % 2);
            }
        low = v4u {words[0], words[1], words[2], words[3]}, high = v4u {words[4], words[5], words[6], words[7]};
    }
    __device__ __forceinline__ void widen_to(uint32_t kind, float (&v)[8]) const {
        if (!HALF && kind == kF32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(low[i]), v[4 + i] = __uint_as_float(high[i]);
        } else if (kind == kBF16) widen<__bf16>(low, v);
        else widen<_Float16>(low, v);
    }
};

/**
 *  Threads (x) share a row, rows (y) a workgroup, as forward; a workgroup has every gridDim.x-th of such groups and keeps its part of the weight's
 *  gradient in registers until the last. Where a thread has eight values of a row (P = 1: rows of at most 512 values, and of 1025 to 8192) a row is asked for before
 *  the one before is worked on; of others a row is read twice, the second time out of the caches. HALF: all operands are of 16 bits.
 *  Memory is what bounds it up to there (with the weight's and the total's gradient: 8192 x 4096 bf16 56 to 60 us, 4.5 to 4.8 TB/s, f32 110, 4.9; 8192 x 8192 bf16 104, 5.2;
 *  16384 x 1024 bf16 37, 3.7). Rows of more than 8192 values do not fit the 128 registers of 1024 threads: with P = 2 some 16 to 19 of f32 or mixed types go to
 *  scratch memory (4096 x 16384 bf16 147 us, 3.6 TB/s, f32 339, 3.2), with P = 4 109 to 221 of every type (2000 x 32768 bf16 396 us, 1.3 TB/s; f32 694), which bounds these.
 */
template <class T, int P, bool HALF>
__global__ __launch_bounds__(1024) void rms_norm_backward_kernel(NormBackwardArgs p) {
    constexpr uint32_t kKind = sizeof(T) == 4 ? kF32 : __is_same(T, __bf16) ? kBF16 : kF16;
    __shared__ float sums[2][16][2];
    extern __shared__ float parts[]; // rows of a workgroup but the first: theirs of the weight's gradient
    float of_weight[P][8] = {};
    Raw<HALF> w, ahead[3];
    auto const load_weight = [&](uint32_t col) { if (p.weight) w.load(p.weight_kind, (uint8_t const *)p.weight, col, p.k); };
    auto const load_row = [&](uint64_t row, uint32_t col, Raw<HALF> (&raw)[3], bool rest) { // total, gradient, the total's gradient
        raw[0].load(kKind, p.total + row * p.total_stride, col, p.k);
        raw[1].load(p.grad_kind, p.grad + row * p.grad_stride, col, p.k);
        if (rest && p.grad_total) raw[2].load(kKind, p.grad_total + row * p.grad_total_stride, col, p.k);
    };
    if (P == 1) load_weight(threadIdx.x * 8); // (of longer rows it comes out of the caches each time, and so do their values for the second loop)
    uint64_t const step = (uint64_t)gridDim.x * blockDim.y;
    uint64_t row = (uint64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (P == 1 && row < p.rows) load_row(row, threadIdx.x * 8, ahead, true);
    for (uint32_t turn = 0; row < p.rows; row += step, turn ^= 1) { // (two sets of sums: no wavefront writes what another still reads)
        float square = 0, inner = 0;
        Raw<HALF> now[3];
        if (P == 1) now[0] = ahead[0], now[1] = ahead[1], now[2] = ahead[2];
        if (P == 1 && row + step < p.rows) load_row(row + step, threadIdx.x * 8, ahead, true);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            uint32_t const col = (i * blockDim.x + threadIdx.x) * 8;
            float x[8], y[8], z[8];
            if (P > 1) load_weight(col), load_row(row, col, now, false);
            now[0].widen_to(kKind, x), now[1].widen_to(p.grad_kind, y);
            if (p.weight) w.widen_to(p.weight_kind, z);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                square += x[j] * x[j];
                inner += (p.weight ? y[j] * z[j] : y[j]) * x[j];
            }
        }
#pragma unroll
        for (int half = 32; half; half >>= 1) square += __shfl_xor(square, half), inner += __shfl_xor(inner, half);
        if (blockDim.x > 64) { // (then the workgroup has one row, and all its threads are here)
            if (!(threadIdx.x & 63)) sums[turn][threadIdx.x >> 6][0] = square, sums[turn][threadIdx.x >> 6][1] = inner;
            __syncthreads();
            square = sums[turn][0][0], inner = sums[turn][0][1];
            for (uint32_t i = 1; i < blockDim.x / 64; ++i) square += sums[turn][i][0], inner += sums[turn][i][1];
        }
        float const scale = 1.0f / sqrtf(square / (float)p.k + p.eps), shift = inner / (float)p.k * scale * scale;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            uint32_t const col = (i * blockDim.x + threadIdx.x) * 8;
            float x[8], y[8], z[8], of_x[8];
            if (P > 1) load_weight(col), load_row(row, col, now, true);
            now[0].widen_to(kKind, x), now[1].widen_to(p.grad_kind, y);
            if (p.weight) w.widen_to(p.weight_kind, z);
            if (p.grad_total) now[2].widen_to(kKind, of_x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float const v = scale * ((p.weight ? y[j] * z[j] : y[j]) - x[j] * shift);
                of_x[j] = p.grad_total ? of_x[j] + v : v;
                of_weight[i][j] += y[j] * (x[j] * scale);
            }
            if (col < p.k) store_some((T *)(p.grad_x + row * p.grad_x_stride) + col, of_x, p.k - col);
        }
    }
    if (!p.partial) return;
    if (blockDim.y > 1) { // rows of at most 1024 values: those of the workgroup are added up in their order
        uint32_t const width = blockDim.x * 8 * P;
        if (threadIdx.y) {
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) parts[(threadIdx.y - 1) * width + (i * blockDim.x + threadIdx.x) * 8 + j] = of_weight[i][j];
        }
        __syncthreads();
        if (threadIdx.y) return;
        for (uint32_t y = 1; y < blockDim.y; ++y)
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) of_weight[i][j] += parts[(y - 1) * width + (i * blockDim.x + threadIdx.x) * 8 + j];
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
        uint32_t const col = (i * blockDim.x + threadIdx.x) * 8;
        if (col < p.k) store_some(p.partial + (uint64_t)blockIdx.x * p.k + col, of_weight[i], p.k - col);
    }
}

/** out[col] = the sum over `rows` rows of 32-bit values: 32 halves of wavefronts take every 32nd row of 32 columns each. */
__global__ __launch_bounds__(1024) void column_sum_kernel(float const *values, uint32_t rows, uint32_t k, uint32_t kind, void *out) {
    __shared__ float sums[32][33];
    uint32_t const x = threadIdx.x & 31, col = blockIdx.x * 32 + x, part = threadIdx.x >> 5;
    float sum = 0;
    if (col < k) {
#pragma unroll 4
        for (uint32_t row = part; row < rows; row += 32) sum += values[(uint64_t)row * k + col];
    }
    sums[part][x] = sum;
    __syncthreads();
    if (part || col >= k) return;
#pragma unroll 8
    for (int i = 1; i < 32; ++i) sum += sums[i][x];
    store_1(kind, out, col, sum);
}

constexpr uint64_t kMaxNormDepth = 32768; // (1024 threads of 32 values, which the forward kernels hold; those of the backward pass spill)

/** Threads for a row and how many times eight values one has. */
struct NormShape {
    uint32_t threads, passes, rows;
};
/** (Forward rows of over 2048 values have 16 a thread: more workgroups are at different places of their rows then. 16384 x 8192 bf16 to 8 bits 248 us with 8 and 220 with 16,
 *  222 with 32; without the residual to 16 bits 126, 99 and 101; 8192 x 4096 51 and 44.) */
NormShape norm_shape(uint64_t k, bool forward = false) {
    NormShape s = {64, 1, 4};
    uint64_t const eights = (k + 7) / 8;
    if (eights <= 64) return s;
    if (eights <= 128) return s.passes = 2, s;
    s.rows = 1;
    s.passes = eights <= (forward ? 256 : 1024) ? 1 : eights <= 2048 ? 2 : 4;
    s.threads = (uint32_t)((eights + s.passes * 64 - 1) / (s.passes * 64) * 64);
    return s;
}
template <class Call>
int with_passes(uint32_t passes, Call call) {
    return passes == 1 ? call(Number<1>()) : passes == 2 ? call(Number<2>()) : call(Number<4>());
}
template <class Call>
int with_float(int dtype, Call call) {
    return dtype == nk_f32_k ? call(float()) : dtype == nk_bf16_k ? call(__bf16()) : call(_Float16());
}

/** Workgroups of a backward pass: as many as run at once, with 1024 threads a compute unit, or groups of rows, if there are fewer. */
uint32_t norm_backward_workgroups(uint64_t rows, uint64_t k) {
    NormShape const shape = norm_shape(k);
    uint64_t const groups = (rows + shape.rows - 1) / shape.rows, most = 256 * (1024 / (shape.threads * shape.rows));
    return (uint32_t)(groups < most ? groups : most);
}

} // namespace

int launch_column_sum(float const *values, uint64_t rows, uint64_t k, uint32_t kind, void *out, hipStream_t stream) {
    hipLaunchKernelGGL(column_sum_kernel, dim3((uint32_t)((k + 31) / 32)), dim3(1024), 0, stream, values, (uint32_t)rows, (uint32_t)k, kind, out);
    hipError_t const e = hipGetLastError();
    return e == hipSuccess ? 0 : mx_fail(e, "column_sum_kernel");
}

} // namespace nk_gfx950

using namespace nk_gfx950;

extern "C" {

int nk_amd_mx8_quantize_async(nk_dtype_t dtype, void const *x, nk_size_t rows, nk_size_t depth, nk_size_t x_stride, void *codes,
                              nk_size_t codes_stride, void *scales, nk_size_t scales_stride, void *stream) {
    int const bytes = float_bytes(dtype);
    if (!bytes) return mx_fail("mx8_quantize: x has to be f32, bf16 or f16");
    if (rows >= (1ull << 31) || depth >= (1ull << 31)) return mx_fail("mx8_quantize: too many rows or columns");
    if (!rows || !depth) return 0;
    if (!x || !codes || !scales) return mx_fail("mx8_quantize: NULL operand");
    if (!aligned_to(x, x_stride, bytes)) return mx_fail("mx8_quantize: x is not aligned to its elements");
    uint64_t const each = (depth + 511) / 512;
    return in_pieces(rows, each * 64, "mx8_quantize_kernel", [&](uint64_t first, uint64_t here) {
        QuantizeArgs const p = {(uint8_t const *)x + first * x_stride, x_stride, here * each, (uint8_t *)codes + first * codes_stride, (uint8_t *)scales + first * scales_stride, codes_stride,
                                scales_stride, nullptr, 0, kind_of(dtype), (uint32_t)each, (uint32_t)depth, (uint32_t)depth};
        hipLaunchKernelGGL(mx8_quantize_kernel, dim3((uint32_t)((here * each + 3) / 4)), dim3(256), 0, (hipStream_t)stream, p);
    });
}

int nk_amd_mx8_dequantize_async(nk_dtype_t dtype, void const *codes, nk_size_t codes_stride, void const *scales, nk_size_t scales_stride,
                                nk_size_t rows, nk_size_t depth, void *x, nk_size_t x_stride, void *stream) {
    int const bytes = float_bytes(dtype);
    if (!bytes) return mx_fail("mx8_dequantize: x has to be f32, bf16 or f16");
    if (rows >= (1ull << 31) || depth >= (1ull << 31)) return mx_fail("mx8_dequantize: too many rows or columns");
    if (!rows || !depth) return 0;
    if (!x || !codes || !scales) return mx_fail("mx8_dequantize: NULL operand");
    if (!aligned_to(x, x_stride, bytes)) return mx_fail("mx8_dequantize: x is not aligned to its elements");
    uint64_t const each = (depth + 511) / 512;
    return in_pieces(rows, each * 64, "mx8_dequantize_kernel", [&](uint64_t first, uint64_t here) {
        hipLaunchKernelGGL(mx8_dequantize_kernel, dim3((uint32_t)((here * each + 3) / 4)), dim3(256), 0, (hipStream_t)stream,
                           (uint8_t const *)codes + first * codes_stride, codes_stride, (uint8_t const *)scales + first * scales_stride, scales_stride,
                           here * each, (uint32_t)each, (uint32_t)depth, kind_of(dtype), (uint8_t *)x + first * x_stride, x_stride);
    });
}

int nk_amd_rms_norm_async(nk_amd_rms_norm_t const *n, void *stream) {
    if (!n) return mx_fail("rms_norm: NULL operand");
    int const bytes = float_bytes(n->dtype), weight_bytes = float_bytes(n->weight_dtype);
    bool const mx8 = n->y_dtype == nk_e4m3_k;
    if (!bytes) return mx_fail("rms_norm: x has to be f32, bf16 or f16");
    if (n->weight && !weight_bytes) return mx_fail("rms_norm: weight has to be f32, bf16 or f16");
    if (!mx8 && !float_bytes(n->y_dtype)) return mx_fail("rms_norm: y has to be f32, bf16, f16 or mx8");
    if (n->rows >= (1ull << 31) || n->depth > kMaxNormDepth) return mx_fail("rms_norm: too many rows or columns (at most 32768)");
    if (!(n->eps >= 0) || n->eps == __builtin_inff()) return mx_fail("rms_norm: eps has to be a finite number that is not negative");
    if (!n->rows || !n->depth) return 0;
    if (!n->x || !n->y || (mx8 && !n->y_scales) || (n->residual && !n->total)) return mx_fail("rms_norm: NULL operand");
    if (!aligned_to(n->x, n->x_stride, bytes) || (n->residual && (!aligned_to(n->residual, n->residual_stride, bytes) || !aligned_to(n->total, n->total_stride, bytes))) ||
        (n->weight && !aligned_to(n->weight, 0, weight_bytes)) || (!mx8 && !aligned_to(n->y, n->y_stride, float_bytes(n->y_dtype))))
        return mx_fail("rms_norm: an operand is not aligned to its elements");
    NormShape const shape = norm_shape(n->depth, true);
    return with_float(n->dtype, [&](auto value) {
        typedef decltype(value) T;
        return with_passes(shape.passes, [&](auto number) {
            constexpr int P = decltype(number)::value;
            return in_pieces(n->rows, shape.threads, "rms_norm_kernel", [&](uint64_t first, uint64_t here) {
                NormArgs const p = {(uint8_t const *)n->x + first * n->x_stride, n->residual ? (uint8_t const *)n->residual + first * n->residual_stride : nullptr,
                                    n->residual ? (uint8_t *)n->total + first * n->total_stride : nullptr, n->x_stride, n->residual_stride, n->total_stride,
                                    n->weight, (uint8_t *)n->y + first * n->y_stride, mx8 ? (uint8_t *)n->y_scales + first * n->y_scales_stride : nullptr,
                                    n->y_stride, n->y_scales_stride, here, (uint32_t)n->depth, kind_of(n->weight_dtype), kind_of(n->y_dtype), n->eps};
                dim3 const grid((uint32_t)((here + shape.rows - 1) / shape.rows)), block(shape.threads, shape.rows);
                if (mx8) hipLaunchKernelGGL((rms_norm_kernel<T, P, true>), grid, block, 0, (hipStream_t)stream, p);
                else hipLaunchKernelGGL((rms_norm_kernel<T, P, false>), grid, block, 0, (hipStream_t)stream, p);
            });
        });
    });
}

nk_size_t nk_amd_rms_norm_backward_workspace_size(nk_amd_rms_norm_backward_t const *n) {
    if (!n || !n->grad_weight || n->rows >= (1ull << 31) || n->depth > kMaxNormDepth) return 0;
    return (norm_backward_workgroups(n->rows, n->depth) * n->depth * 4 + 255) / 256 * 256;
}

int nk_amd_rms_norm_backward_async(nk_amd_rms_norm_backward_t const *n, void *workspace, nk_size_t workspace_bytes, void *stream) {
    if (!n) return mx_fail("rms_norm_backward: NULL operand");
    int const bytes = float_bytes(n->dtype), weight_bytes = float_bytes(n->weight_dtype), grad_bytes = float_bytes(n->grad_dtype);
    if (!bytes || !grad_bytes || ((n->weight || n->grad_weight) && !weight_bytes)) return mx_fail("rms_norm_backward: operands have to be f32, bf16 or f16");
    if (n->rows >= (1ull << 31) || n->depth > kMaxNormDepth) return mx_fail("rms_norm_backward: too many rows or columns (at most 32768)");
    if (!(n->eps >= 0) || n->eps == __builtin_inff()) return mx_fail("rms_norm_backward: eps has to be a finite number that is not negative");
    if (!n->depth) return 0;
    if (n->rows && (!n->total || !n->grad || !n->grad_x)) return mx_fail("rms_norm_backward: NULL operand");
    if (!aligned_to(n->total, n->total_stride, bytes) || !aligned_to(n->grad, n->grad_stride, grad_bytes) || !aligned_to(n->grad_x, n->grad_x_stride, bytes) ||
        (n->grad_total && !aligned_to(n->grad_total, n->grad_total_stride, bytes)) || (n->weight && !aligned_to(n->weight, 0, weight_bytes)) ||
        (n->grad_weight && !aligned_to(n->grad_weight, 0, weight_bytes)))
        return mx_fail("rms_norm_backward: an operand is not aligned to its elements");
    nk_size_t const needed = nk_amd_rms_norm_backward_workspace_size(n);
    if (needed && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < needed)) return mx_fail("rms_norm_backward: the workspace is too small or not 256-byte aligned");
    NormShape const shape = norm_shape(n->depth);
    uint32_t const workgroups = norm_backward_workgroups(n->rows, n->depth);
    NormBackwardArgs const p = {(uint8_t const *)n->total, (uint8_t const *)n->grad, (uint8_t const *)n->grad_total, (uint8_t *)n->grad_x, n->total_stride, n->grad_stride,
                                n->grad_total_stride, n->grad_x_stride, n->weight, n->grad_weight ? (float *)workspace : nullptr, n->rows, (uint32_t)n->depth,
                                kind_of(n->weight_dtype), kind_of(n->grad_dtype), n->eps};
    if (workgroups) {
        int const status = with_float(n->dtype, [&](auto value) {
            typedef decltype(value) T;
            return with_passes(shape.passes, [&](auto number) {
                constexpr int P = decltype(number)::value;
                dim3 const grid(workgroups), block(shape.threads, shape.rows);
                uint32_t const room = (shape.rows - 1) * shape.threads * shape.passes * 32;
                bool const half = sizeof(T) == 2 && grad_bytes == 2 && (!n->weight || weight_bytes == 2);
                if (half) hipLaunchKernelGGL((rms_norm_backward_kernel<T, P, sizeof(T) == 2>), grid, block, room, (hipStream_t)stream, p);
                else hipLaunchKernelGGL((rms_norm_backward_kernel<T, P, false>), grid, block, room, (hipStream_t)stream, p);
                hipError_t const e = hipGetLastError();
                return e == hipSuccess ? 0 : mx_fail(e, "rms_norm_backward_kernel");
            });
        });
        if (status) return status;
    }
    return n->grad_weight ? launch_column_sum((float const *)workspace, workgroups, n->depth, kind_of(n->weight_dtype), n->grad_weight, (hipStream_t)stream) : 0;
}

} // extern "C"
