/**
 *  @brief What the norm's and the dense products' kernels share: 8-bit blocks, activations, values of any float type.
 *  @file numkong_amd/csrc/dense_gfx950.hpp
 */
#ifndef NUMKONG_AMD_DENSE_GFX950_HPP
#define NUMKONG_AMD_DENSE_GFX950_HPP

#include "mx_gfx950.hpp"
#include "numkong_amd/dense.h"

namespace nk_gfx950 {

/** Bytes of a value of a float type; 0: it is none. */
inline int float_bytes(int dtype) { return dtype == nk_f32_k ? 4 : dtype == nk_bf16_k || dtype == nk_f16_k ? 2 : 0; }
inline bool aligned_to(void const *p, uint64_t stride, uint64_t bytes) { return !((uintptr_t)p % bytes) && !(stride % bytes); }

/** A value of a float type that the host names: 0 f32, 1 bf16, 2 f16 (a branch that all lanes take alike). */
enum Kind : uint32_t { kF32 = 0, kBF16 = 1, kF16 = 2 };
inline Kind kind_of(int dtype) { return dtype == nk_bf16_k ? kBF16 : dtype == nk_f16_k ? kF16 : kF32; }
__host__ __device__ inline uint32_t bytes_of(uint32_t kind) { return kind == kF32 ? 4 : 2; }

/** Eight adjacent values of a row from column `col` on; zeros from column `k` on. */
template <class T>
__device__ __forceinline__ void load_adjacent(T const *row, uint32_t col, uint32_t k, float (&v)[8]) {
    if (col + 8 <= k) {
        if constexpr (sizeof(T) == 4) {
            v4u const low = *(v4u_anywhere const *)(row + col), high = *(v4u_anywhere const *)(row + col + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(low[i]), v[4 + i] = __uint_as_float(high[i]);
        } else widen<T>(*(v4u_anywhere const *)(row + col), v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < k ? (float)row[col + i] : 0.0f;
}
/** Four likewise. */
template <class T>
__device__ __forceinline__ void load_adjacent(T const *row, uint32_t col, uint32_t k, float (&v)[4]) {
    if (col + 4 <= k) {
        if constexpr (sizeof(T) == 4) {
            v4u const words = *(v4u_anywhere const *)(row + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(words[i]);
        } else {
            typedef v2u __attribute__((aligned(1))) v2u_anywhere;
            v2u const words = *(v2u_anywhere const *)(row + col);
            float both[8];
            widen<T>(v4u {words[0], words[1], 0, 0}, both);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = both[i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = col + i < k ? (float)row[col + i] : 0.0f;
}
template <int V>
__device__ __forceinline__ void load_adjacent(uint32_t kind, void const *row, uint32_t col, uint32_t k, float (&v)[V]) {
    if (kind == kF32) load_adjacent((float const *)row, col, k, v);
    else if (kind == kBF16) load_adjacent((__bf16 const *)row, col, k, v);
    else load_adjacent((_Float16 const *)row, col, k, v);
}
/** `count` (up to 8) adjacent results at column `col` of a row. */
__device__ __forceinline__ void store_8(uint32_t kind, void *row, uint32_t col, float const (&v)[8], uint32_t count) {
    if (kind == kF32) store_some((float *)row + col, v, count);
    else if (kind == kBF16) store_some((__bf16 *)row + col, v, count);
    else store_some((_Float16 *)row + col, v, count);
}
__device__ __forceinline__ float load_1(uint32_t kind, void const *row, uint64_t col) {
    return kind == kF32 ? ((float const *)row)[col] : kind == kBF16 ? (float)((__bf16 const *)row)[col] : (float)((_Float16 const *)row)[col];
}
__device__ __forceinline__ void store_1(uint32_t kind, void *row, uint64_t col, float v) {
    if (kind == kF32) ((float *)row)[col] = v;
    else if (kind == kBF16) ((__bf16 *)row)[col] = (__bf16)v;
    else ((_Float16 *)row)[col] = (_Float16)v;
}

/**
 *  A lane's eight values of a block of 32, which four adjacent lanes hold, to e4m3 codes (the first in the lowest byte) and the
 *  block's scale byte. The scale is the smallest power of two that keeps the largest magnitude within 448 = 1.75 x 2^8: its exponent
 *  field less 8, and one more where the mantissa is above 0.75; none is below 2^-127. Nothing saturates then, and the
 *  conversion, which divides by the scale, rounds to nearest even. A NaN or an infinity has the largest field and decides
 *  for its block.
 */
__device__ __forceinline__ v2u quantize_8(float const (&v)[8], uint32_t &scale) {
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t const magnitude = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        largest = largest > magnitude ? largest : magnitude;
    }
    largest = block_max<4>(largest);
    uint32_t const field = largest >> 23, above = (largest & 0x7FFFFFu) > 0x600000u;
    scale = field == 255 ? 255 : field + above > 8 ? field + above - 8 : 0;
    v2u codes = {0, 0};
#ifdef NK_MX_DEVICE_BUILTINS
    typedef short v2s __attribute__((ext_vector_type(2)));
    float const power = __uint_as_float(scale ? scale << 23 : 0x00400000u);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        v2s word = {0, 0};
        word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(word, v[4 * i], v[4 * i + 1], power, false);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(word, v[4 * i + 2], v[4 * i + 3], power, true);
        codes[i] = field == 255 ? 0u : __builtin_bit_cast(uint32_t, word);
    }
#endif
    return codes;
}
/** `count` (up to 8) codes to any address. */
__device__ __forceinline__ void store_codes(uint8_t *to, v2u codes, uint32_t count) {
    if (count >= 8) {
        typedef v2u __attribute__((aligned(1))) v2u_anywhere;
        *(v2u_anywhere *)to = codes;
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if (i < count) to[i] = (uint8_t)(codes[i / 4] >> 8 * (i % 4));
}

/** Rows to codes and scales: bytes, or words of four blocks, [word of the row][pitch rows]. */
struct QuantizeArgs {
    uint8_t const *x;
    uint64_t x_stride, stretches; // stretches: rows times `each`
    uint8_t *codes, *scales;      // scales or words: NULL, if it is the other
    uint64_t codes_stride, scales_stride;
    uint32_t *words;
    uint64_t pitch;
    uint32_t kind, each, k, stored; // each: 512 values, of a row; codes are written up to `stored`, zeros from k on
};
/** Four of the stretches, a wavefront each: eight values a lane, four lanes to a block. Memory is what bounds it (16384 x 8192 bf16 71 us, 5.7 TB/s). */
__device__ __forceinline__ void quantize_stretches(QuantizeArgs const &p, uint64_t four) {
    uint64_t const at = four * 4 + (threadIdx.x >> 6);
    if (at >= p.stretches) return;
    uint64_t const row = at / p.each;
    uint32_t const col = (uint32_t)(at - row * p.each) * 512 + (threadIdx.x & 63) * 8;
    float v[8];
    uint32_t scale;
    load_adjacent(p.kind, p.x + row * p.x_stride, col, p.k, v);
    v2u const code = quantize_8(v, scale);
    if (p.words) {
        uint32_t word = scale << (threadIdx.x & 12) * 2;
        word |= __shfl_xor(word, 4);
        word |= __shfl_xor(word, 8);
        if (!(threadIdx.x & 15) && col < p.k) p.words[col / 128 * p.pitch + row] = word;
    }
    if (col < p.stored) store_codes(p.codes + row * p.codes_stride + col, code, p.stored - col);
    if (p.scales && !(threadIdx.x & 3) && col < p.k) p.scales[row * p.scales_stride + col / 32] = (uint8_t)scale;
}

/** The four values of a word of e4m3 codes. */
__device__ __forceinline__ void widen_e4m3(uint32_t word, float (&v)[4]) {
#ifdef NK_MX_DEVICE_BUILTINS
    typedef float v2f __attribute__((ext_vector_type(2)));
    v2f const low = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false), high = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
    v[0] = low[0], v[1] = low[1], v[2] = high[0], v[3] = high[1];
#endif
}
/** The power of two of a scale byte. */
__device__ __forceinline__ float scale_of(uint32_t byte) {
    return byte == 255 ? __builtin_nanf("") : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

/**
 *  Activations and their slopes in 32 bits. An activation is off by at most 16 + 4 z units of 2^-24 of itself, z the magnitude of the exponent (x, for gelu_tanh
 *  1.6 (x + 0.045 x^3)), a slope by as many of the largest slope, and both by what the limits below leave out. The sigmoid is 1 / (1 + e^-x) by the part's own 2^x and reciprocal
 *  (one unit each; with the library's forms, chosen by a switch for each value, bias and relu of f16 8192 x 8191 x 1000 took 60 us more). The tanh of gelu_tanh is written as 1 - 2 / (1 + e^2z), so that 0.5 x (1 + tanh z) = x / (1 + e^-2z).
 *  Gelu: with h = erfc(|x| / sqrt 2) / 2 it is x - x h, or x h below zero, and h = e^(-x^2/2) t P(t), t = 1 / (1 + 0.35 |x|): P is fitted
 *  to that quotient over all |x| <= 16 by least squares weighted towards the largest relative error (8 degrees, 5 units of 2^-24 with its
 *  evaluation).
 *  Limits: the reciprocal of what is above 2^126 is zero, so that silu ends at -87.3 and gelu_tanh at -10.0 (both were below 1.1e-36 there). Gelu and its slope
 *  are at their limits beyond +-16, as e^(-x^2/2) is 0 in 32 bits already, silu's slope beyond +-80 (off by 1.5e-33), gelu_tanh's beyond +-9 (2.6e-27).
 */
__device__ __forceinline__ float power_of_2(float x) {
#ifdef NK_MX_DEVICE_BUILTINS
    return __builtin_amdgcn_exp2f(x);
#else
    return x;
#endif
}
__device__ __forceinline__ float reciprocal(float x) {
#ifdef NK_MX_DEVICE_BUILTINS
    return __builtin_amdgcn_rcpf(x);
#else
    return x;
#endif
}
constexpr float kLog2E = 1.4426950408889634f;
/** erfc(|x| / sqrt 2) / 2 and e^(-x^2/2), |x| <= 16. */
__device__ __forceinline__ float half_erfc(float x, float &bell) {
    float const square = x * x, rest = __builtin_fmaf(x, x, -square);
    float const power = square * (-0.5f * kLog2E); // (its rounding, and those of the square and the constant, would be 18 units at x = 5)
    float const lost = __builtin_fmaf(square, -0.5f * kLog2E, -power) + __builtin_fmaf(rest, -0.5f * kLog2E, square * -9.6298e-9f);
    bell = power_of_2(power);
    bell = __builtin_fmaf(bell, lost * 0.69314718f, bell);
    float const t = reciprocal(__builtin_fmaf(0.35f, fabsf(x), 1.0f));
    float h = -0.0291648954f;
    h = __builtin_fmaf(h, t, 0.144065633f), h = __builtin_fmaf(h, t, -0.255912066f), h = __builtin_fmaf(h, t, 0.159404889f), h = __builtin_fmaf(h, t, -0.0232723057f);
    h = __builtin_fmaf(h, t, 0.105578497f), h = __builtin_fmaf(h, t, 0.11981453f), h = __builtin_fmaf(h, t, 0.139864475f), h = __builtin_fmaf(h, t, 0.139621243f);
    return h * t * bell;
}
/** e^-z of gelu_tanh's sigmoid. */
__device__ __forceinline__ float gelu_tanh_power(float x) { return power_of_2(x * __builtin_fmaf(x * x, -0.044715f * 1.5957691216057308f * kLog2E, -1.5957691216057308f * kLog2E)); }
__device__ __forceinline__ float within(float x, float limit) { return x > limit ? limit : x < -limit ? -limit : x; } // (NaN stays)

__device__ __forceinline__ float relu(float x) { return x < 0 ? 0.0f : x; }
__device__ __forceinline__ float silu(float x) { return x < -128.0f ? -0.0f : x * reciprocal(1.0f + power_of_2(x * -kLog2E)); }
__device__ __forceinline__ float gelu(float x) {
    float bell;
    float const near = within(x, 16.0f);
    return relu(x) - fabsf(near) * half_erfc(near, bell);
}
__device__ __forceinline__ float gelu_tanh(float x) { return x < -128.0f ? -0.0f : x * reciprocal(1.0f + gelu_tanh_power(x)); }

__device__ __forceinline__ float relu_slope(float x) { return x > 0 ? 1.0f : 0.0f; }
__device__ __forceinline__ float silu_slope(float x) {
    float const e = power_of_2(within(x, 80.0f) * -kLog2E), s = reciprocal(1.0f + e);
    return fabsf(x) > 80.0f ? relu_slope(x) : __builtin_fmaf(x * e * s, s, s);
}
__device__ __forceinline__ float gelu_slope(float x) {
    float bell;
    float const near = within(x, 16.0f), h = half_erfc(near, bell);
    return __builtin_fmaf(near * 0.39894228040143268f, bell, x < 0 ? h : 1.0f - h);
}
__device__ __forceinline__ float gelu_tanh_slope(float x) {
    float const near = within(x, 9.0f), e = gelu_tanh_power(near), s = reciprocal(1.0f + e);
    float const bend = near * __builtin_fmaf(near * near, 0.134145f * 1.5957691216057308f, 1.5957691216057308f);
    return fabsf(x) > 9.0f ? relu_slope(x) : __builtin_fmaf(bend * e * s, s, s);
}
/** Many values at once: one branch, which all lanes take alike. (A branch for each eight costs a wavefront that is alone more than their products.) */
template <int N, int V>
__device__ __forceinline__ void activate(uint32_t kind, float (&x)[N][V]) {
#define NK_EACH(f)                                                                                                                                             \
    _Pragma("unroll") for (int i = 0; i < N * V; ++i) x[i / V][i % V] = f(x[i / V][i % V]);                                                                      \
    break
    switch (kind) {
    case nk_amd_relu: NK_EACH(relu);
    case nk_amd_silu: NK_EACH(silu);
    case nk_amd_gelu: NK_EACH(gelu);
    case nk_amd_gelu_tanh: NK_EACH(gelu_tanh);
    }
}
template <int N, int V>
__device__ __forceinline__ void slope(uint32_t kind, float (&x)[N][V]) {
    switch (kind) {
    case nk_amd_no_activation: NK_EACH([](float) { return 1.0f; });
    case nk_amd_relu: NK_EACH(relu_slope);
    case nk_amd_silu: NK_EACH(silu_slope);
    case nk_amd_gelu: NK_EACH(gelu_slope);
    case nk_amd_gelu_tanh: NK_EACH(gelu_tanh_slope);
    }
#undef NK_EACH
}

} // namespace nk_gfx950

#endif // NUMKONG_AMD_DENSE_GFX950_HPP
