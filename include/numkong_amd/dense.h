/**
 *  @brief The dense feed-forward layer on one MI355X (gfx950): norm, product, gated product, with their gradients.
 *  @file include/numkong_amd/dense.h
 *
 *  Additions without a counterpart in the reference, next to the packed dots of <numkong_amd/dots.h> and the 4-bit products of
 *  <numkong_amd/mx.h>, whose manner they follow:
 *
 *      rms_norm   y = t w / sqrt(mean(t^2) + eps) of each row, t = x + residual; results in floats or in 8 bits with scales
 *      linear     C[m x n] = activation(A[m x k] * W[n x k]^T + bias) + residual, everything in one pass over the results
 *      gated      C[m x n] = activation(A * W^T) x (A * W_up^T), element by element, both products in one kernel
 *
 *  Matrices of weights are plain rows, as training leaves them: nothing is packed, a program may change them between calls. Types are
 *  bf16 or f16, with gradients, or microscaled 8-bit floats ("mx8"): e4m3 codes, one to a byte, with one E8M0 scale (an exponent of two
 *  biased by 127; 255 makes the block NaN) for each 32 values of a row. Rows of mx8 take `depth` bytes, of scales (depth + 31) / 32.
 *
 *  Every call queues its work on `stream` (a hipStream_t, NULL = the default stream), touches device memory only, neither
 *  allocates nor synchronises, may be captured into a HIP graph (after one eager call, which loads the kernels), and returns 0
 *  or a status that `nk_hip_last_error()` explains; a refused call has queued nothing. Strides are in bytes; results share memory
 *  neither with one another nor with operands, unless it says so. A workspace is device memory, 256-byte aligned, of the
 *  bytes that the call's `*_workspace_size` says of the very same structure (addresses and strides count; 0: NULL will do), and belongs to
 *  the call until the stream has run it. Sums are held in 32 bits; no result depends on the order in which workgroups run.
 */
#ifndef NUMKONG_AMD_DENSE_H
#define NUMKONG_AMD_DENSE_H

#include "numkong_amd/dots.h"

#ifdef __cplusplus
extern "C" {
#endif

/**
 *  x[rows x depth] (`dtype`: nk_f32_k, nk_bf16_k or nk_f16_k) to codes and scales, and back. A block's scale is the smallest power of two,
 *  at least 2^-127, that keeps its largest magnitude within 448; codes are rounded to nearest, ties to the even code. A block
 *  that holds a NaN or an infinity becomes NaN as a whole (scale 255, codes 0).
 */
NK_DYNAMIC int nk_amd_mx8_quantize_async(nk_dtype_t dtype, void const *x, nk_size_t rows, nk_size_t depth, nk_size_t x_stride,
                                         void *codes, nk_size_t codes_stride, void *scales, nk_size_t scales_stride, void *stream);
NK_DYNAMIC int nk_amd_mx8_dequantize_async(nk_dtype_t dtype, void const *codes, nk_size_t codes_stride, void const *scales,
                                           nk_size_t scales_stride, nk_size_t rows, nk_size_t depth, void *x, nk_size_t x_stride,
                                           void *stream);

/** A norm's operands. Depth is at most 32768. */
typedef struct {
    nk_size_t rows, depth;
    float eps;                 /* not negative */
    nk_dtype_t dtype;          /* of x, residual and total: nk_f32_k, nk_bf16_k or nk_f16_k */
    void const *x;
    nk_size_t x_stride;
    void const *residual;      /* added to x, or NULL */
    nk_size_t residual_stride;
    void *total;               /* x + residual, rounded to `dtype`, which is what is normed; NULL without a residual. May be x or */
    nk_size_t total_stride;    /* the residual themselves (the same address and stride) */
    nk_dtype_t weight_dtype;   /* nk_f32_k, nk_bf16_k or nk_f16_k */
    void const *weight;        /* depth values side by side, or NULL: ones */
    nk_dtype_t y_dtype;        /* nk_f32_k, nk_bf16_k, nk_f16_k, or nk_e4m3_k: mx8, quantised from the exact values (64 bits) */
    void *y;
    nk_size_t y_stride;
    void *y_scales;            /* mx8 only */
    nk_size_t y_scales_stride;
} nk_amd_rms_norm_t;
NK_DYNAMIC int nk_amd_rms_norm_async(nk_amd_rms_norm_t const *norm, void *stream);

/** The gradients of a norm. */
typedef struct {
    nk_size_t rows, depth;
    float eps;
    nk_dtype_t dtype;          /* of total and grad_x */
    void const *total;         /* what was normed: x, or x + residual as the norm has left it */
    nk_size_t total_stride;
    nk_dtype_t weight_dtype;   /* of weight and grad_weight */
    void const *weight;        /* or NULL: ones */
    nk_dtype_t grad_dtype;     /* of grad: nk_f32_k, nk_bf16_k or nk_f16_k */
    void const *grad;          /* of y */
    nk_size_t grad_stride;
    void const *grad_total;    /* of total, from elsewhere (`dtype`), or NULL */
    nk_size_t grad_total_stride;
    void *grad_x;              /* of x and the residual alike */
    nk_size_t grad_x_stride;
    void *grad_weight;         /* depth values, or NULL: not wanted */
} nk_amd_rms_norm_backward_t;
NK_DYNAMIC nk_size_t nk_amd_rms_norm_backward_workspace_size(nk_amd_rms_norm_backward_t const *norm);
NK_DYNAMIC int nk_amd_rms_norm_backward_async(nk_amd_rms_norm_backward_t const *norm, void *workspace, nk_size_t workspace_bytes,
                                              void *stream);

/** What a product applies to its sums: erf's gelu, and the one by tanh. */
enum { nk_amd_no_activation = 0, nk_amd_relu = 1, nk_amd_silu = 2, nk_amd_gelu = 3, nk_amd_gelu_tanh = 4 };

/**
 *  A product's operands. Height and width are below 2^31 (gated, of more than 16 rows: width at most 2^31 - 128), depth below 2^22.
 *  With `w_dtype` nk_e4m3_k matrices are mx8; A then has scales as well, or is floats (f32, bf16 or f16), quantised on the way exactly as
 *  nk_amd_mx8_quantize_async does, and C is bf16 or f16: the 8-bit matrix instruction's sums keep 13 bits below a lane's largest
 *  product, about 1e-5 of the norm of all results at a depth of 8192. Single results that are much smaller than their products show it.
 */
typedef struct {
    nk_size_t height, width, depth;
    int gated;                 /* with w_up, else linear */
    nk_dtype_t a_dtype;        /* nk_bf16_k or nk_f16_k as w's; of mx8: nk_e4m3_k (with a_scales), nk_f32_k, nk_bf16_k or nk_f16_k */
    void const *a;
    nk_size_t a_stride;
    void const *a_scales;
    nk_size_t a_scales_stride;
    nk_dtype_t w_dtype;        /* nk_bf16_k, nk_f16_k or nk_e4m3_k */
    void const *w;             /* width rows of `depth` values; of a gated product the gate's */
    nk_size_t w_stride;
    void const *w_scales;
    nk_size_t w_scales_stride;
    void const *w_up;          /* gated: the other matrix */
    nk_size_t w_up_stride;
    void const *w_up_scales;
    nk_size_t w_up_scales_stride;
    int activation;            /* nk_amd_no_activation and so on */
    nk_dtype_t bias_dtype;     /* nk_f32_k, nk_bf16_k or nk_f16_k */
    void const *bias;          /* width values, or NULL; not gated */
    nk_dtype_t residual_dtype; /* nk_f32_k, nk_bf16_k or nk_f16_k */
    void const *residual;      /* height x width, or NULL; not gated. May be C itself (the same address, stride and type) */
    nk_size_t residual_stride;
    nk_dtype_t c_dtype;        /* nk_f32_k, nk_bf16_k or nk_f16_k */
    void *c;
    nk_size_t c_stride;
    float *pre;                /* for the gradients, of 16-bit matrices: A * W^T + bias before the activation, height x width, or NULL */
    float *pre_up;             /* and A * W_up^T, gated only; both or none */
    nk_size_t pre_stride;
} nk_amd_linear_t;
NK_DYNAMIC nk_size_t nk_amd_linear_workspace_size(nk_amd_linear_t const *linear);
NK_DYNAMIC int nk_amd_linear_async(nk_amd_linear_t const *linear, void *workspace, nk_size_t workspace_bytes, void *stream);

/**
 *  The gradients of a product of 16-bit matrices, those of them that have an address. The gradient of A * W^T (+ bias) is rounded
 *  to the matrices' type, as an operand of the matrix instructions; that of the bias is summed before that. With f16 it has f16's range as
 *  well, whatever the types of `grad` and the sums: beyond 65504 it is infinite, below 2^-25 zero (gradients are scaled to fit, as f16 asks for).
 */
typedef struct {
    nk_size_t height, width, depth; /* of the product: all below 2^22 */
    int gated;
    nk_dtype_t dtype;          /* of A, W, and their gradients: nk_bf16_k or nk_f16_k */
    void const *a;
    nk_size_t a_stride;
    void const *w;
    nk_size_t w_stride;
    void const *w_up;          /* gated */
    nk_size_t w_up_stride;
    int activation;
    float const *pre;          /* as the product has left it; NULL without an activation, if not gated */
    float const *pre_up;
    nk_size_t pre_stride;
    nk_dtype_t grad_dtype;     /* nk_f32_k, nk_bf16_k or nk_f16_k */
    void const *grad;          /* of C */
    nk_size_t grad_stride;
    void *grad_a;              /* height x depth */
    nk_size_t grad_a_stride;
    void *grad_w;              /* width x depth */
    nk_size_t grad_w_stride;
    void *grad_w_up;           /* gated */
    nk_size_t grad_w_up_stride;
    nk_dtype_t bias_dtype;
    void *grad_bias;           /* width values; not gated */
} nk_amd_linear_backward_t;
NK_DYNAMIC nk_size_t nk_amd_linear_backward_workspace_size(nk_amd_linear_backward_t const *linear);
NK_DYNAMIC int nk_amd_linear_backward_async(nk_amd_linear_backward_t const *linear, void *workspace, nk_size_t workspace_bytes,
                                            void *stream);

#ifdef __cplusplus
}
#endif

#endif // NUMKONG_AMD_DENSE_H
