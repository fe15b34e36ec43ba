/**
 *  @brief What the microscaled 4-bit kernels and the experts' kernels share: formats, the packed image, the plan.
 *  @file numkong_amd/csrc/mx_gfx950.hpp
 *
 *  The arithmetic. A block is 32 values of a row, x_t = q_t * 2^(s - 127) with 4-bit floats q_t and an 8-bit s, so
 *
 *      sum_t a_t b_t = sum over blocks of 2^(sa - 127) 2^(sb - 127) * sum over the block of qa_t qb_t
 *
 *  and v_mfma_scale_f32_16x16x128_f8f6f4 does just that: lane l brings 32 codes (16 bytes) of row l % 16, block l / 16 of
 *  the four that 128 values hold, and the scale byte of that very block. Measured on this part: its sums of 4-bit products
 *  lose nothing beyond what 32-bit sums lose (depth 8192, random codes and scales: 2.0e-7 of the result's norm against
 *  6.4e-7 for products added one by one in 32 bits; exact on quantised normal data), so one accumulator runs through the
 *  whole depth. A scale of 255 gives NaN also where every code of the block is zero.
 *
 *  Depth is walked in steps of 128 values, 64 bytes of codes a row; four steps (a super) share a 32-bit word of scales per
 *  lane, byte u for step u, which the instruction picks by an immediate.
 *
 *  Packed image (B, n columns of depth k, `count` matrices), little-endian:
 *
 *      [ 128-byte header ][ codes of every matrix ][ scales of every matrix ]
 *      codes:  [tile][step][lane] 16 bytes      1024 bytes that one wavefront loads at once and feeds to the instruction
 *      scales: [tile][super][lane] 4 bytes
 *
 *  A tile is 16 columns, four tiles a group of 64. Row q of tile j of a group is column 16 (q / 4) + 4 j + q % 4: a lane's
 *  results of the four tiles are then 16 adjacent columns of one row of C, and are stored as such.
 *
 *  Staged A (in the workspace): rows of codes `a_pitch` bytes apart, padded with zeros to whole steps; rows of scales
 *  [super][l / 16] 4 bytes, again byte u for step u.
 */
#ifndef NUMKONG_AMD_MX_GFX950_HPP
#define NUMKONG_AMD_MX_GFX950_HPP

#include <hip/hip_runtime.h>

#include <stddef.h>
#include <stdint.h>

#include "numkong_amd/hip_abi.h"
#include "numkong_amd/mx.h"

namespace nk_gfx950 {

/** The text that nk_hip_last_error() gives on this thread; both return a status for the caller to hand on. */
int mx_fail(hipError_t status, char const *what);
int mx_fail(char const *what);

constexpr uint32_t kMxMagic = 0x34584D4Eu; // "NMX4"
constexpr uint32_t kMxHeaderBytes = 128;
struct MxHeader {
    uint32_t magic, version, count, n, k, reserved[3];
};

struct MxGeometry {
    uint32_t steps, supers, tiles; // of one matrix
    uint64_t code_bytes, scale_bytes, total_bytes; // of one matrix, of one matrix, of the image
};
inline bool mx_geometry(size_t count, size_t n, size_t k, MxGeometry &g) {
    if (n >= (1ull << 31) || k >= (1ull << 31) || count >= (1ull << 20)) return false;
    g.steps = (uint32_t)((k + 127) / 128), g.supers = (g.steps + 3) / 4, g.tiles = (uint32_t)((n + 63) / 64) * 4;
    g.code_bytes = (uint64_t)g.tiles * g.steps * 1024, g.scale_bytes = (uint64_t)g.tiles * g.supers * 256;
    if (count && g.code_bytes + g.scale_bytes > (1ull << 46) / count) return false;
    g.total_bytes = kMxHeaderBytes + count * (g.code_bytes + g.scale_bytes);
    return true;
}

/**
 *  The plan of the experts' products, 32-bit words: header, first row of each expert, rows (slots sorted by expert), the
 *  row of each slot (-1: no expert), tiles of rows. Bucket `experts` holds the slots of no expert, in the last rows.
 */
struct PlanHeader {
    uint32_t magic, slots, experts, tile_rows, tile_count, valid_rows, reserved[2];
};
constexpr uint32_t kPlanMagic = 0x504C414Eu;
struct PlanTile {
    int32_t expert, first, last, reserved; // rows [first, last) of one expert; expert == experts: rows of none
};
struct PlanGeometry {
    uint32_t tile_rows, max_tiles;
    size_t offsets, order, place, tiles, total_words; // in words
};
/** Rows of a tile: what an expert has on average decides which kernel will run, and with it how its rows are cut. */
inline uint32_t plan_tile_rows(size_t slots, size_t experts) {
    size_t const mean = experts ? slots / experts : 0;
    return mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 96 ? 64 : mean <= 256 ? 128 : 256;
}
constexpr size_t kMaxExperts = 1024, kMaxTopK = 64, kMaxGroups = 64;
inline bool plan_geometry(size_t slots, size_t experts, PlanGeometry &g) {
    if (!experts || experts > kMaxExperts || slots >= (1ull << 30)) return false;
    g.tile_rows = plan_tile_rows(slots, experts);
    g.max_tiles = (uint32_t)(slots / g.tile_rows + (slots < experts + 1 ? slots : experts + 1));
    g.offsets = sizeof(PlanHeader) / 4;
    g.order = g.offsets + ((experts + 2 + 3) & ~(size_t)3);
    g.place = g.order + slots;
    g.tiles = (g.place + slots + 3) & ~(size_t)3;
    g.total_words = g.tiles + (size_t)g.max_tiles * 4;
    return true;
}

#ifdef __HIP_DEVICE_COMPILE__
#define NK_MX_DEVICE_BUILTINS 1
#endif

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

/** Eight adjacent values of a row from column `col` on, as 32-bit floats; zeros from column `k` on. `wide`: rows start on
 *  16-byte addresses. (Widening is exact, so whatever follows sees the values themselves.) */
template <class T>
__device__ __forceinline__ void load_eight(T const *row, uint32_t col, uint32_t k, bool wide, float (&v)[8]) {
    if (wide && col + 8 <= k) {
        if constexpr (sizeof(T) == 4) {
            v4f const low = *(v4f const *)(row + col), high = *(v4f const *)(row + col + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = low[i], v[4 + i] = high[i];
        }
        else {
            v4u const words = *(v4u const *)(row + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (__is_same(T, __bf16))
                    v[2 * i] = __uint_as_float(words[i] << 16), v[2 * i + 1] = __uint_as_float(words[i] & 0xFFFF0000u);
                else {
                    f16x2 const pair = __builtin_bit_cast(f16x2, (uint32_t)words[i]);
                    v[2 * i] = (float)pair[0], v[2 * i + 1] = (float)pair[1];
                }
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < k ? (float)row[col + i] : 0.0f;
}

/** The largest of four adjacent lanes, in all four. */
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
    uint32_t const y = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true); // lanes 1 0 3 2
    x = x > y ? x : y;
    uint32_t const z = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true); // lanes 2 3 0 1
    return x > z ? x : z;
}

/**
 *  Eight values of a block of 32 that four adjacent lanes hold, to eight codes and the block's scale byte. The exponent
 *  field of the largest magnitude, less 2, is the scale: e2m1's largest exponent is 2. (Magnitudes are compared as integers;
 *  a NaN or an infinity has the largest exponent field and so decides for its block; subnormal blocks end at 2^-127.) The
 *  conversion divides by the scale, rounds to nearest even and saturates: measured equal to that definition on every bf16
 *  value and on f32 and f16 values of every size, at scales from 2^-127 to 2^127.
 */
__device__ __forceinline__ uint32_t quantize_eight(float const (&v)[8], uint32_t &scale) {
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t const magnitude = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        largest = largest > magnitude ? largest : magnitude;
    }
    largest = quad_max(largest);
    uint32_t const field = largest >> 23;
    scale = field == 255 ? 255 : field > 2 ? field - 2 : 0;
    float const power = __uint_as_float(scale ? scale << 23 : 0x00400000u);
    uint32_t codes = 0;
#ifdef NK_MX_DEVICE_BUILTINS
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], power, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], power, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], power, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], power, 3);
#endif
    return field == 255 ? 0u : codes;
}

/** acc += W-fragment x A-fragment: rows of the result are the image's columns. `U`: which byte of the scale words. */
template <int U>
__device__ __forceinline__ v4f mx_multiply(v4u w, v4u a, v4f acc, uint32_t w_scale, uint32_t a_scale) {
#ifdef NK_MX_DEVICE_BUILTINS
    v8i const x = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    v8i const y = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, acc, 4, 4, U, (int)w_scale, U, (int)a_scale);
#else
    return acc;
#endif
}

typedef __attribute__((address_space(3))) void mx_lds_t;
typedef __attribute__((address_space(1))) void const mx_global_t;
/** 16 or 4 bytes per lane from each lane's own address into LDS at `dst` + 16 or 4 x lane (`dst` the same in all lanes). */
__device__ __forceinline__ void fetch_16(void const *src, void *dst) {
#ifdef NK_MX_DEVICE_BUILTINS
    __builtin_amdgcn_global_load_lds((mx_global_t *)src, (mx_lds_t *)dst, 16, 0, 0);
#endif
}
__device__ __forceinline__ void fetch_4(void const *src, void *dst) {
#ifdef NK_MX_DEVICE_BUILTINS
    __builtin_amdgcn_global_load_lds((mx_global_t *)src, (mx_lds_t *)dst, 4, 0, 0);
#endif
}

/** A number that a lambda's argument carries at compile time. */
template <int N>
struct Number {
    static constexpr int value = N;
};

/** `count` (up to N) adjacent results at `to`; all N as one vector where `wide` says that the address allows it. */
template <class Out, int N>
__device__ __forceinline__ void store_some(Out *to, float const (&v)[N], uint32_t count, bool wide) {
    if (wide && count >= N) {
        struct alignas(sizeof(Out) * N < 16 ? sizeof(Out) * N : 16) Pack {
            Out x[N];
        } pack;
#pragma unroll
        for (int i = 0; i < N; ++i) pack.x[i] = (Out)v[i];
        *(Pack *)to = pack;
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if ((uint32_t)i < count) to[i] = (Out)v[i];
}

} // namespace nk_gfx950

#endif // NUMKONG_AMD_MX_GFX950_HPP
