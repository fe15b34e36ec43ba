/**
 *  @brief Microscaled 4-bit floats on one MI355X (gfx950), and what a layer of experts needs around their products.
 *  @file include/numkong_amd/mx.h
 *
 *  Additions without a counterpart in the reference, next to the packed dots of <numkong_amd/dots.h> and in their manner:
 *
 *      quantise      rows of f32, bf16 or f16 to e2m1 codes with one E8M0 scale for each 32 values of a row, and back
 *      pack, dots    C[m x n] = A[m x k] * B[n x k]^T with B packed once, A quantised by the call (or quantised already)
 *      route         scores to the experts of each token and their weights, and the gradient of the scores
 *      plan, experts the products of each token's row with the matrices of its experts, in one launch
 *
 *  An element is sign, two bits of exponent (bias 1), one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6. Two share a byte, the
 *  even column in the low half. A scale is the exponent of a power of two, biased by 127; 255 makes the whole block NaN.
 *  Rows of codes take (depth + 1) / 2 bytes, rows of scales (depth + 31) / 32.
 *
 *  Every call queues its work on `stream` (a hipStream_t, NULL = the default stream), touches device memory only, neither
 *  allocates nor synchronises, may be captured into a HIP graph (after one eager call, which loads the kernels), and returns 0
 *  or a status that `nk_hip_last_error()` explains. Strides are in bytes; results share memory neither with one another's rows nor
 *  with operands. Sums are held in 32 bits (of products below 2^-149 nothing may be left); no result depends on the order in which
 *  workgroups run.
 */
#ifndef NUMKONG_AMD_MX_H
#define NUMKONG_AMD_MX_H

#include "numkong_amd/dots.h"

#ifdef __cplusplus
extern "C" {
#endif

/**
 *  x[rows x depth] (`dtype`: nk_f32_k, nk_bf16_k or nk_f16_k) to codes and scales. The scale of a block is
 *  2^(floor(log2 max|x|) - 2), at least 2^-127; elements are rounded to nearest, ties to the even code, and stop at 6.
 *  A block that holds a NaN or an infinity gets scale 255 and zero codes. No alignment beyond the elements' own is asked for.
 */
NK_DYNAMIC int nk_amd_mx_quantize_async(nk_dtype_t dtype, void const *x, nk_size_t rows, nk_size_t depth,
                                        nk_size_t x_stride, void *codes, nk_size_t codes_stride, void *scales,
                                        nk_size_t scales_stride, void *stream);
/** The values that codes and scales stand for, in f32, bf16 (both exact) or f16 (rounded). */
NK_DYNAMIC int nk_amd_mx_dequantize_async(nk_dtype_t dtype, void const *codes, nk_size_t codes_stride,
                                          void const *scales, nk_size_t scales_stride, nk_size_t rows, nk_size_t depth,
                                          void *x, nk_size_t x_stride, void *stream);

/** Bytes of the packed image of `count` matrices of width x depth (0: no such image; width has to be below 2^31, depth below
 *  2^25, count below 2^20). The image is this library's own format (the operand order of the matrix instructions),
 *  relocatable, and must be 16-byte aligned. */
NK_DYNAMIC nk_size_t nk_amd_mx_packed_size(nk_size_t count, nk_size_t width, nk_size_t depth);
/** Packs `count` matrices, matrix i at codes + i * codes_matrix and scales + i * scales_matrix bytes. */
NK_DYNAMIC int nk_amd_mx_pack_async(void const *codes, nk_size_t codes_stride, nk_size_t codes_matrix,
                                    void const *scales, nk_size_t scales_stride, nk_size_t scales_matrix,
                                    nk_size_t count, nk_size_t width, nk_size_t depth, void *packed, void *stream);

/**
 *  C[height x width] = A * B^T. A: floats of `a_dtype`, quantised on the way (exactly as nk_amd_mx_quantize_async does), or,
 *  where `a_scales` is not NULL, codes at `a` and scales (then `a_dtype` is not looked at). C: f32, bf16 or f16 by `c_dtype`.
 *  `workspace`: device memory, 256-byte aligned, of nk_amd_mx_dots_workspace_size bytes (which may be 0, then NULL will do);
 *  it belongs to the call until the stream has run it. An image whose header does not say width x depth gives NaNs. A block
 *  of NaN (scale 255) makes every result NaN that it goes into, also where the other operand's values are zero.
 */
NK_DYNAMIC nk_size_t nk_amd_mx_dots_workspace_size(nk_size_t height, nk_size_t width, nk_size_t depth, int a_is_codes);
NK_DYNAMIC int nk_amd_mx_dots_packed_async(nk_dtype_t a_dtype, void const *a, nk_size_t a_stride, void const *a_scales,
                                           nk_size_t a_scales_stride, void const *packed, nk_dtype_t c_dtype, void *c,
                                           nk_size_t c_stride, nk_size_t height, nk_size_t width, nk_size_t depth,
                                           void *workspace, nk_size_t workspace_bytes, void *stream);

/** How experts_route picks and weighs. */
typedef struct {
    int sigmoid;      /* scores: 0 softmax over the row, 1 sigmoid of each logit */
    int renormalize;  /* weights are divided by the sum of the chosen scores (+ 1e-20) */
    float scale;      /* and multiplied by this */
    int groups;       /* experts stand in so many groups of equal size (1: no groups) */
    int top_groups;   /* of which so many stay, those whose */
    int group_top;    /* best so many (1 or 2) selection scores have the largest sum; a masked expert adds nothing to it */
} nk_amd_route_t;

/**
 *  For each of `tokens` rows of logits (f32, bf16 or f16) the `top_k` experts of largest selection score, in descending
 *  order, ties to the lowest index: `chosen` (tokens x top_k, i32), and their weights (tokens x top_k, f32). The selection
 *  score is the logit, or score + bias[expert] (f32) where a bias is given; weights never contain the bias. A logit of
 *  -inf is never chosen: where a row (the groups of it that stay) has too few others, the expert is -1 and its weight 0. Groups
 *  with an expert that can be chosen stand before those without. A NaN ranks above all numbers.
 *  At most 1024 experts, top_k at most 64, 64 groups.
 */
NK_DYNAMIC int nk_amd_experts_route_async(nk_dtype_t dtype, void const *logits, nk_size_t logits_stride,
                                          nk_size_t tokens, nk_size_t experts, nk_size_t top_k, float const *bias,
                                          nk_amd_route_t const *how, float *weights, nk_i32_t *chosen, void *stream);
/** The gradient of the logits (same type and shape) from that of the weights, for the experts that were chosen. */
NK_DYNAMIC int nk_amd_experts_route_backward_async(nk_dtype_t dtype, void const *logits, nk_size_t logits_stride,
                                                   nk_size_t tokens, nk_size_t experts, nk_size_t top_k,
                                                   nk_amd_route_t const *how, nk_i32_t const *chosen,
                                                   float const *grad_weights, void *grad_logits,
                                                   nk_size_t grad_stride, void *stream);

/**
 *  Which rows each expert gets: `slots` entries of `chosen` (tokens x top_k in a row) sorted by expert, in the order in
 *  which they stand there; entries outside [0, experts) go to no expert. The plan is read by the products, any number of
 *  them; 16-byte aligned device memory.
 */
NK_DYNAMIC nk_size_t nk_amd_experts_plan_size(nk_size_t slots, nk_size_t experts);
NK_DYNAMIC int nk_amd_experts_plan_async(nk_i32_t const *chosen, nk_size_t slots, nk_size_t experts, void *plan,
                                         void *stream);

/**
 *  y[slot] = A[slot / a_share] * B[expert of slot]^T for every slot, zeros where there is no expert: A has
 *  ceil(slots / a_share) rows (a_share = top_k: a row for each token; 1: a row for each slot). With `weights` (slots, f32)
 *  the `top_k` rows of a token are summed by weight into C[slots / top_k x width] instead, slots without an expert left
 *  out, in 32 bits and in the order of the slots. A, C and workspace as in nk_amd_mx_dots_packed_async; the image holds
 *  `experts` matrices, and the plan is one of nk_amd_experts_plan_async for these slots and experts (another gives NaNs).
 */
NK_DYNAMIC nk_size_t nk_amd_mx_experts_workspace_size(nk_size_t slots, nk_size_t a_share, nk_size_t experts,
                                                      nk_size_t width, nk_size_t depth, int a_is_codes,
                                                      int weighted);
NK_DYNAMIC int nk_amd_mx_dots_experts_async(nk_dtype_t a_dtype, void const *a, nk_size_t a_stride, void const *a_scales,
                                            nk_size_t a_scales_stride, nk_size_t a_share, void const *packed,
                                            void const *plan, nk_size_t slots, nk_size_t experts, nk_size_t top_k,
                                            float const *weights, nk_dtype_t c_dtype, void *c, nk_size_t c_stride,
                                            nk_size_t width, nk_size_t depth, void *workspace,
                                            nk_size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif // NUMKONG_AMD_MX_H
