/**
 *  @brief Dense products with everything around them in one pass, and their gradients, on gfx950.
 *  @file numkong_amd/csrc/dense_gfx950.hip
 *
 *  Implements the second half of <numkong_amd/dense.h>. With p = A W^T + bias, C = f(p) + residual and g the gradient of C:
 *
 *      d = g f'(p);   of A: d W;   of W: d^T A;   of the bias: the sum of d over the rows; of the residual: g
 *
 *  and gated, with q = A W_up^T and C = f(p) q:  d = g q f'(p), e = g f(p);  of A: d W + e W_up;  of W: d^T A;  of W_up: e^T A.
 */
#include "dense_gfx950.hpp"

namespace nk_gfx950 {

int launch_mx8_quantize(uint32_t kind, void const *x, uint64_t x_stride, uint64_t rows, uint64_t k, uint8_t *codes, uint64_t codes_stride,
                        uint8_t *scales, uint64_t scales_stride, hipStream_t stream); // norm_gfx950.hip
int launch_column_sum(float const *values, uint64_t rows, uint64_t k, uint32_t kind, void *out, hipStream_t stream);

namespace {

/** What becomes of a product's sums. */
struct Epilogue {
    void const *bias;
    uint8_t const *residual;
    uint8_t *c;
    float *pre, *pre_up;
    uint64_t residual_stride, c_stride, pre_stride;
    uint32_t bias_kind, residual_kind, c_kind, activation;
};
__device__ __forceinline__ void finish_one(Epilogue const &e, uint64_t row, uint32_t col, float p, float q, bool gated) {
    if (e.bias) p += load_1(e.bias_kind, e.bias, col);
    if (e.pre) {
        *((float *)((uint8_t *)e.pre + row * e.pre_stride) + col) = p;
        if (gated) *((float *)((uint8_t *)e.pre_up + row * e.pre_stride) + col) = q;
    }
    float v = activate(e.activation, p);
    if (gated) v *= q;
    if (e.residual) v += load_1(e.residual_kind, e.residual + row * e.residual_stride, col);
    store_1(e.c_kind, e.c + row * e.c_stride, col, v);
}

/** An operand: rows of the result (or columns) by `row` bytes, the depth by `step` bytes; with scales mx8. */
struct Side {
    uint8_t const *values;
    uint64_t row, step;
    uint8_t const *scales;
    uint64_t scales_stride;
};
template <class T>
__device__ __forceinline__ T value_of(Side const &s, uint64_t row, uint32_t k) {
    uint8_t const *const at = s.values + row * s.row + k * s.step;
    if (!s.scales) return *(T const *)at;
    float four[4];
    widen_e4m3(*at, four);
    return (T)(four[0] * scale_of(s.scales[row * s.scales_stride + k / 32]));
}

struct SimpleArgs {
    Side a[2], b[2]; // of sums over two depths: both pairs; gated: the second b
    uint32_t m, n, k, pairs;
    Epilogue e;
};
template <class T>
struct Vector8;
template <>
struct Vector8<__bf16> {
    typedef __bf16 type __attribute__((ext_vector_type(8)));
};
template <>
struct Vector8<_Float16> {
    typedef _Float16 type __attribute__((ext_vector_type(8)));
};
template <class T>
__device__ __forceinline__ v16f multiply(typename Vector8<T>::type a, typename Vector8<T>::type b, v16f c) {
#ifdef NK_MX_DEVICE_BUILTINS
    if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
#else
    return c;
#endif
}

/** The plainest form: 64 x 64 results a workgroup, 32 x 32 a wavefront, operands one value at a time into LDS. */
template <class T, bool GATED>
__global__ __launch_bounds__(256) void simple_kernel(SimpleArgs p) {
    typedef typename Vector8<T>::type V;
    __shared__ __attribute__((aligned(16))) T as[64][40], bs[GATED ? 2 : 1][64][40];
    uint32_t const row0 = blockIdx.y * 64, col0 = blockIdx.x * 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v16f sum = {}, sum_up = {};
    for (uint32_t pair = 0; pair < p.pairs; ++pair)
        for (uint32_t k0 = 0; k0 < p.k; k0 += 32) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < 64 * 32; i += 256) {
                uint32_t const row = i / 32, k = i % 32;
                as[row][k] = row0 + row < p.m && k0 + k < p.k ? value_of<T>(p.a[pair], row0 + row, k0 + k) : (T)0;
                bool const there = col0 + row < p.n && k0 + k < p.k;
                bs[0][row][k] = there ? value_of<T>(p.b[pair], col0 + row, k0 + k) : (T)0;
                if (GATED) bs[GATED][row][k] = there ? value_of<T>(p.b[1], col0 + row, k0 + k) : (T)0;
            }
            __syncthreads();
            for (uint32_t k = 0; k < 32; k += 16) {
                uint32_t const at = k + 8 * (lane / 32), row = (wave & 1) * 32 + lane % 32, col = (wave >> 1) * 32 + lane % 32;
                V const a = *(V const *)&as[row][at];
                sum = multiply<T>(a, *(V const *)&bs[0][col][at], sum);
                if (GATED) sum_up = multiply<T>(a, *(V const *)&bs[GATED][col][at], sum_up);
            }
        }
    for (uint32_t i = 0; i < 16; ++i) {
        uint32_t const row = row0 + (wave & 1) * 32 + i % 4 + 8 * (i / 4) + 4 * (lane / 32), col = col0 + (wave >> 1) * 32 + lane % 32;
        if (row < p.m && col < p.n) finish_one(p.e, row, col, sum[i], sum_up[i], GATED);
    }
}
template <class T>
int launch_simple(SimpleArgs const &p, bool gated, hipStream_t stream) {
    dim3 const grid((p.n + 63) / 64, (p.m + 63) / 64);
    if (gated) hipLaunchKernelGGL((simple_kernel<T, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((simple_kernel<T, false>), grid, dim3(256), 0, stream, p);
    hipError_t const e = hipGetLastError();
    return e == hipSuccess ? 0 : mx_fail(e, "simple_kernel");
}
int launch_simple(int dtype, SimpleArgs const &p, bool gated, hipStream_t stream) {
    return dtype == nk_f16_k ? launch_simple<_Float16>(p, gated, stream) : launch_simple<__bf16>(p, gated, stream);
}

// ---- the gradient of the sums --------------------------------------------------------------------------------------

struct SlopeArgs {
    uint8_t const *grad;
    float const *pre, *pre_up;
    uint8_t *d; // rows of d and, `up_at` values further on, e; or NULL
    float *partial; // (workgroups of rows, n): sums of d, or NULL
    uint64_t grad_stride, pre_stride, d_stride;
    uint32_t m, n, padded, up_at, grad_kind, activation, rows_each;
    bool gated;
};
/** 512 columns of `rows_each` rows a workgroup, four rows at a time, eight columns a lane. Columns from n to `padded` of d get zeros. */
template <class T>
__global__ __launch_bounds__(256) void slope_kernel(SlopeArgs p) {
    __shared__ float sums[4][512];
    uint32_t const lane = threadIdx.x & 63, col = blockIdx.x * 512 + lane * 8;
    float sum[8] = {};
    if (col < p.padded)
        for (uint32_t i = threadIdx.x >> 6; i < p.rows_each; i += 4) {
            uint64_t const row = (uint64_t)blockIdx.y * p.rows_each + i;
            if (row >= p.m) break;
            float g[8], x[8], up[8], d[8], e[8];
            load_8(p.grad_kind, p.grad + row * p.grad_stride, col, p.n, g);
            if (p.pre) load_8((float const *)((uint8_t const *)p.pre + row * p.pre_stride), col, p.n, x);
            if (p.gated) load_8((float const *)((uint8_t const *)p.pre_up + row * p.pre_stride), col, p.n, up);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                d[j] = p.pre ? g[j] * slope(p.activation, x[j]) : g[j];
                if (p.gated) d[j] *= up[j], e[j] = g[j] * activate(p.activation, x[j]);
                sum[j] += d[j];
            }
            if (p.d) {
                T *const to = (T *)(p.d + row * p.d_stride) + col;
                store_some(to, d, p.padded - col);
                if (p.gated) store_some(to + p.up_at, e, p.padded - col);
            }
        }
    if (!p.partial) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[threadIdx.x >> 6][lane * 8 + j] = sum[j];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 512; i += 256) {
        uint32_t const at = blockIdx.x * 512 + i;
        if (at < p.n) p.partial[(uint64_t)blockIdx.y * p.n + at] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
    }
}

constexpr uint64_t kMaxDepth = 1ull << 22, kMaxRows = 1ull << 31;
inline uint64_t up_to(uint64_t n, uint64_t step) { return (n + step - 1) / step * step; }

// ---- what calls ask for --------------------------------------------------------------------------------------------

int check_linear(nk_amd_linear_t const *l) {
    if (!l) return mx_fail("linear: NULL operand");
    bool const mx8 = l->w_dtype == nk_e4m3_k, codes = l->a_dtype == nk_e4m3_k;
    if (l->height >= kMaxRows || l->width >= kMaxRows || l->depth >= kMaxDepth) return mx_fail("linear: unsupported dimensions");
    if (!mx8 && l->w_dtype != nk_bf16_k && l->w_dtype != nk_f16_k) return mx_fail("linear: W has to be bf16, f16 or mx8");
    if (mx8 ? !codes && !float_bytes(l->a_dtype) : l->a_dtype != l->w_dtype) return mx_fail("linear: A has to have W's type, or floats or mx8 where W is mx8");
    if (!float_bytes(l->c_dtype) || (mx8 && l->c_dtype == nk_f32_k)) return mx_fail("linear: C has to be f32, bf16 or f16, where W is mx8 bf16 or f16");
    if (l->activation < nk_amd_no_activation || l->activation > nk_amd_gelu_tanh) return mx_fail("linear: there is no such activation");
    if (l->gated && (l->bias || l->residual)) return mx_fail("linear: a gated product takes no bias and no residual");
    if ((l->bias && !float_bytes(l->bias_dtype)) || (l->residual && !float_bytes(l->residual_dtype))) return mx_fail("linear: bias and residual have to be f32, bf16 or f16");
    if (l->gated ? !l->pre != !l->pre_up : l->pre_up != nullptr) return mx_fail("linear: a gated product leaves both sums or none, another has one");
    return 0;
}
/** Of calls that have results to write. */
int check_linear_operands(nk_amd_linear_t const *l) {
    bool const mx8 = l->w_dtype == nk_e4m3_k, codes = l->a_dtype == nk_e4m3_k;
    uint64_t const a_bytes = codes ? 1 : float_bytes(l->a_dtype), w_bytes = mx8 ? 1 : 2;
    if (!l->c || !aligned_to(l->c, l->c_stride, float_bytes(l->c_dtype))) return mx_fail("linear: C is NULL or not aligned to its elements");
    if (l->depth && (!l->a || !l->w || (l->gated && !l->w_up) || (codes && !l->a_scales) || (mx8 && (!l->w_scales || (l->gated && !l->w_up_scales))))) return mx_fail("linear: NULL operand");
    if (!aligned_to(l->a, l->a_stride, a_bytes) || !aligned_to(l->w, l->w_stride, w_bytes) || !aligned_to(l->w_up, l->w_up_stride, w_bytes) ||
        (l->bias && !aligned_to(l->bias, 0, float_bytes(l->bias_dtype))) || (l->residual && !aligned_to(l->residual, l->residual_stride, float_bytes(l->residual_dtype))) ||
        !aligned_to(l->pre, l->pre ? l->pre_stride : 0, 4) || !aligned_to(l->pre_up, 0, 4))
        return mx_fail("linear: an operand is not aligned to its elements");
    return 0;
}
int check_workspace(char const *what, void const *workspace, uint64_t bytes, uint64_t needed) {
    return needed && (!workspace || ((uintptr_t)workspace & 255) || bytes < needed) ? mx_fail(what) : 0;
}

/** Where a product's workspace has A's codes, if they are made on the way. */
struct LinearLayout {
    uint64_t codes_stride, scales_stride, scales_at, bytes;
    bool quantises;
};
LinearLayout linear_layout(nk_amd_linear_t const *l) {
    LinearLayout y = {};
    y.quantises = l->w_dtype == nk_e4m3_k && l->a_dtype != nk_e4m3_k && l->height && l->width && l->depth;
    if (!y.quantises) return y;
    y.codes_stride = up_to(l->depth, 128), y.scales_stride = y.codes_stride / 32;
    y.scales_at = up_to(l->height * y.codes_stride, 256);
    y.bytes = up_to(y.scales_at + l->height * y.scales_stride, 256);
    return y;
}

/** Where a backward pass's workspace has d (and e behind it in each row), and the sums of d. */
struct BackwardLayout {
    uint64_t padded, d_stride, partial_at, partials, rows_each, bytes;
    bool writes_d, sums;
};
BackwardLayout backward_layout(nk_amd_linear_backward_t const *l) {
    BackwardLayout y = {};
    bool const gated = l->gated, products = l->grad_a || l->grad_w || l->grad_w_up;
    y.writes_d = products && (gated || l->activation || l->grad_dtype != l->dtype);
    y.sums = l->grad_bias != nullptr;
    y.padded = up_to(l->width, 64), y.d_stride = y.padded * 2 * (gated ? 2 : 1);
    y.rows_each = l->height <= 1u << 21 ? 64 : 128, y.partials = (l->height + y.rows_each - 1) / y.rows_each;
    y.partial_at = y.writes_d ? up_to(l->height * y.d_stride, 256) : 0;
    y.bytes = y.partial_at + (y.sums ? up_to(y.partials * l->width * 4, 256) : 0);
    return y;
}
int check_backward(nk_amd_linear_backward_t const *l) {
    if (!l) return mx_fail("linear_backward: NULL operand");
    bool const gated = l->gated;
    if (l->height >= kMaxDepth || l->width >= kMaxDepth || l->depth >= kMaxDepth) return mx_fail("linear_backward: unsupported dimensions");
    if (l->dtype != nk_bf16_k && l->dtype != nk_f16_k) return mx_fail("linear_backward: A and W have to be bf16 or f16");
    if (!float_bytes(l->grad_dtype)) return mx_fail("linear_backward: the gradient has to be f32, bf16 or f16");
    if (l->activation < nk_amd_no_activation || l->activation > nk_amd_gelu_tanh) return mx_fail("linear_backward: there is no such activation");
    if (gated && l->grad_bias) return mx_fail("linear_backward: a gated product has no bias");
    if (!gated && l->grad_w_up) return mx_fail("linear_backward: only a gated product has a second matrix");
    if (l->grad_bias && !float_bytes(l->bias_dtype)) return mx_fail("linear_backward: bias has to be f32, bf16 or f16");
    return 0;
}

} // namespace
} // namespace nk_gfx950

using namespace nk_gfx950;

extern "C" {

nk_size_t nk_amd_linear_workspace_size(nk_amd_linear_t const *l) {
    return check_linear(l) ? 0 : linear_layout(l).bytes;
}

int nk_amd_linear_async(nk_amd_linear_t const *l, void *workspace, nk_size_t workspace_bytes, void *stream) {
    if (int const status = check_linear(l)) return status;
    if (!l->height || !l->width) return 0;
    if (int const status = check_linear_operands(l)) return status;
    LinearLayout const y = linear_layout(l);
    if (check_workspace("linear: the workspace is too small or not 256-byte aligned", workspace, workspace_bytes, y.bytes)) return -1;
    bool const mx8 = l->w_dtype == nk_e4m3_k, gated = l->gated;
    uint64_t const bytes = mx8 ? 1 : 2;
    SimpleArgs p = {};
    p.m = (uint32_t)l->height, p.n = (uint32_t)l->width, p.k = (uint32_t)l->depth, p.pairs = 1;
    p.a[0] = {(uint8_t const *)l->a, l->a_stride, bytes, (uint8_t const *)(mx8 ? l->a_scales : nullptr), l->a_scales_stride};
    if (y.quantises) {
        uint8_t *const codes = (uint8_t *)workspace, *const scales = codes + y.scales_at;
        if (int const status = launch_mx8_quantize(kind_of(l->a_dtype), l->a, l->a_stride, l->height, l->depth, codes, y.codes_stride, scales, y.scales_stride, (hipStream_t)stream)) return status;
        p.a[0] = {codes, y.codes_stride, bytes, scales, y.scales_stride};
    }
    p.b[0] = {(uint8_t const *)l->w, l->w_stride, bytes, (uint8_t const *)(mx8 ? l->w_scales : nullptr), l->w_scales_stride};
    p.b[1] = {(uint8_t const *)l->w_up, l->w_up_stride, bytes, (uint8_t const *)(mx8 ? l->w_up_scales : nullptr), l->w_up_scales_stride};
    p.e = {l->bias, (uint8_t const *)l->residual, (uint8_t *)l->c, l->pre, l->pre_up, l->residual_stride, l->c_stride, l->pre_stride, kind_of(l->bias_dtype),
           kind_of(l->residual_dtype), kind_of(l->c_dtype), (uint32_t)l->activation};
    return launch_simple(l->w_dtype, p, gated, (hipStream_t)stream);
}

nk_size_t nk_amd_linear_backward_workspace_size(nk_amd_linear_backward_t const *l) {
    return check_backward(l) ? 0 : backward_layout(l).bytes;
}

int nk_amd_linear_backward_async(nk_amd_linear_backward_t const *l, void *workspace, nk_size_t workspace_bytes, void *raw_stream) {
    if (int const status = check_backward(l)) return status;
    hipStream_t const stream = (hipStream_t)raw_stream;
    bool const gated = l->gated, some = l->height && l->width;
    if ((l->grad_a && (!aligned_to(l->grad_a, l->grad_a_stride, 2))) || (l->grad_w && !aligned_to(l->grad_w, l->grad_w_stride, 2)) ||
        (l->grad_w_up && !aligned_to(l->grad_w_up, l->grad_w_up_stride, 2)) || (l->grad_bias && !aligned_to(l->grad_bias, 0, float_bytes(l->bias_dtype))))
        return mx_fail("linear_backward: a gradient is not aligned to its elements");
    if (some) {
        if (!l->grad || ((gated || l->activation) && (!l->pre || (gated && !l->pre_up))) || (l->depth && l->grad_a && (!l->w || (gated && !l->w_up))) || (l->depth && (l->grad_w || l->grad_w_up) && !l->a))
            return mx_fail("linear_backward: NULL operand");
        if (!aligned_to(l->grad, l->grad_stride, float_bytes(l->grad_dtype)) || !aligned_to(l->a, l->a_stride, 2) || !aligned_to(l->w, l->w_stride, 2) ||
            !aligned_to(l->w_up, l->w_up_stride, 2) || !aligned_to(l->pre, l->pre_stride, 4) || !aligned_to(l->pre_up, 0, 4))
            return mx_fail("linear_backward: an operand is not aligned to its elements");
    }
    BackwardLayout const y = backward_layout(l);
    if (check_workspace("linear_backward: the workspace is too small or not 256-byte aligned", workspace, workspace_bytes, y.bytes)) return -1;
    uint8_t *const d = (uint8_t *)workspace;
    float *const partial = (float *)(d + y.partial_at);
    if (some && (y.writes_d || y.sums)) {
        SlopeArgs const s = {(uint8_t const *)l->grad, gated || l->activation ? l->pre : nullptr, l->pre_up, y.writes_d ? d : nullptr, y.sums ? partial : nullptr, l->grad_stride,
                             l->pre_stride, y.d_stride, (uint32_t)l->height, (uint32_t)l->width, (uint32_t)y.padded, (uint32_t)y.padded, kind_of(l->grad_dtype), (uint32_t)l->activation,
                             (uint32_t)y.rows_each, gated};
        dim3 const grid((uint32_t)((y.padded + 511) / 512), (uint32_t)y.partials);
        if (l->dtype == nk_f16_k) hipLaunchKernelGGL(slope_kernel<_Float16>, grid, dim3(256), 0, stream, s);
        else hipLaunchKernelGGL(slope_kernel<__bf16>, grid, dim3(256), 0, stream, s);
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, "slope_kernel");
    }
    if (y.sums && l->width)
        if (int const status = launch_column_sum(partial, y.partials, l->width, kind_of(l->bias_dtype), l->grad_bias, stream)) return status;
    uint8_t const *const of_p = y.writes_d ? d : (uint8_t const *)l->grad, *const of_q = d + y.padded * 2;
    uint64_t const d_stride = y.writes_d ? y.d_stride : l->grad_stride;
    auto const kind = kind_of(l->dtype);
    if (l->grad_a && l->height && l->depth) { // rows of d times columns of W
        SimpleArgs p = {};
        p.m = (uint32_t)l->height, p.n = (uint32_t)l->depth, p.k = (uint32_t)l->width, p.pairs = gated ? 2 : 1;
        p.a[0] = {of_p, d_stride, 2, nullptr, 0}, p.a[1] = {of_q, d_stride, 2, nullptr, 0};
        p.b[0] = {(uint8_t const *)l->w, 2, l->w_stride, nullptr, 0}, p.b[1] = {(uint8_t const *)l->w_up, 2, l->w_up_stride, nullptr, 0};
        p.e.c = (uint8_t *)l->grad_a, p.e.c_stride = l->grad_a_stride, p.e.c_kind = kind;
        if (int const status = launch_simple(l->dtype, p, false, stream)) return status;
    }
    for (int i = 0; i < 2; ++i) { // columns of d times columns of A
        void *const to = i ? l->grad_w_up : l->grad_w;
        if (!to || !l->width || !l->depth) continue;
        SimpleArgs p = {};
        p.m = (uint32_t)l->width, p.n = (uint32_t)l->depth, p.k = (uint32_t)l->height, p.pairs = 1;
        p.a[0] = {i ? of_q : of_p, 2, d_stride, nullptr, 0}, p.b[0] = {(uint8_t const *)l->a, 2, l->a_stride, nullptr, 0};
        p.e.c = (uint8_t *)to, p.e.c_stride = i ? l->grad_w_up_stride : l->grad_w_stride, p.e.c_kind = kind;
        if (int const status = launch_simple(l->dtype, p, false, stream)) return status;
    }
    return 0;
}

} // extern "C"
