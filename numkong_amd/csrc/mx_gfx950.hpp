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
 *  lane, byte u for step u, which the instruction picks by an immediate. What is stored is padded to whole supers with zeros.
 *
 *  Fragments: 16 rows of a step are 1024 bytes, lane l's 16 bytes at 16 l (row l % 16, block l / 16 of the step's four), so a
 *  wavefront moves one with a single instruction and in one piece. Their scales of a super are 256 bytes, the word of row r
 *  and block g at word 4 r + 2 (g % 2) + g / 2: instructions of 32 rows take two blocks at a time, and their lanes find the
 *  words of both halves of a step side by side. Both operands of a product are held like this:
 *
 *  Packed image (B, n columns of depth k, `count` matrices), little-endian:
 *
 *      [ 128-byte header ][ codes of every matrix: [tile][step] ][ scales of every matrix: [tile][super] ]
 *
 *  A tile is 16 columns, four tiles a group of 64. Row q of tile j of a group is column 16 (q / 4) + 4 j + q % 4: a lane's
 *  results of the four tiles are then 16 adjacent columns of one row of C, and are stored as such.
 *
 *  Staged A (in the workspace): [16 rows][step] and [16 rows][super] likewise, rows in order (with experts: in the plan's).
 */
#ifndef NUMKONG_AMD_MX_GFX950_HPP
#define NUMKONG_AMD_MX_GFX950_HPP

#include <hip/hip_runtime.h>

#include <stddef.h>
#include <stdint.h>

#include "numkong_amd/hip_abi.h"
#include "numkong_amd/mx.h"

namespace nk_gfx950 {

/** Threads of one launch: HIP takes fewer than 2^32. What needs more is queued in several. */
constexpr uint64_t kMostThreads = 1ull << 31;

/** The text that nk_hip_last_error() gives on this thread; both return a status for the caller to hand on. */
int mx_fail(hipError_t status, char const *what);
int mx_fail(char const *what);
int compute_unit_count(); // of the current device (dots_gfx950.hip)

constexpr uint32_t kMxMagic = 0x34584D4Eu; // "NMX4"
constexpr uint32_t kMxHeaderBytes = 128;
struct MxHeader {
    uint32_t magic, version, count, n, k, reserved[3];
};

/** Depths of products: below 2^25, so that eight tiles of the image, and 128 rows of A, lie within 32-bit offsets; 256 rows but at the last
 *  128 depths, where their last bytes are the 2^32nd, which a buffer does not reach (buffer_of). */
constexpr uint64_t kMxMaxDepth = 1ull << 25;

struct MxGeometry {
    uint32_t steps, supers, tiles; // of one matrix (steps: those that hold values)
    uint64_t code_bytes, scale_bytes, total_bytes; // of one matrix, of one matrix, of the image
};
inline bool mx_geometry(size_t count, size_t n, size_t k, MxGeometry &g) {
    if (n >= (1ull << 31) || k >= kMxMaxDepth || count >= (1ull << 20)) return false;
    g.steps = (uint32_t)((k + 127) / 128), g.supers = (g.steps + 3) / 4, g.tiles = (uint32_t)((n + 63) / 64) * 4;
    g.code_bytes = (uint64_t)g.tiles * g.supers * 4096, g.scale_bytes = (uint64_t)g.tiles * g.supers * 256;
    if (count && g.code_bytes + g.scale_bytes > (1ull << 46) / count) return false;
    g.total_bytes = kMxHeaderBytes + count * (g.code_bytes + g.scale_bytes);
    return true;
}

/** Where, of a fragment's 64 words of scales, that of row r and block g is. */
__host__ __device__ inline uint32_t scale_word(uint32_t r, uint32_t g) { return r * 4 + (g & 1) * 2 + (g >> 1); }

/**
 *  The plan of the experts' products, 32-bit words: header, first row of each expert, the slot of each row, the row of each
 *  slot (-1: no expert), tiles of rows. Rows are the slots sorted by expert; an expert's rows start at a multiple of 16, so
 *  that its fragments are its own, and rows in between have slot -1. Bucket `experts` holds the slots of no expert, last.
 */
struct PlanHeader {
    uint32_t magic, slots, experts, tile_rows;
    uint32_t tile_count, zero_tiles; // tiles of the experts' rows; tiles of the rows of none, behind them
    uint32_t first_zero, end_zero;   // rows of the experts end, and rows of none begin, at the first; these end at the second
};
constexpr uint32_t kPlanMagic = 0x504C414Eu;
struct PlanTile {
    int32_t expert, first, last, reserved; // rows [first, last) of one expert; expert == experts: rows of none
};
struct PlanGeometry {
    uint32_t tile_rows, max_tiles, max_rows;
    size_t offsets, order, place, tiles, table, total_words; // in words
};
/** Rows of a tile: what an expert has on average decides which kernel will run, and with it how its rows are cut. (Tiles of 256
 *  rows: 117 us for 64 experts of 512 rows on average, against 104 us; more of the last tile of each expert is empty.) */
inline uint32_t plan_tile_rows(size_t slots, size_t experts) {
    size_t const mean = experts ? slots / experts : 0;
    return mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : 128;
}
constexpr size_t kPlanBlockSlots = 1024; // slots of a workgroup that makes the plan; its counts stand behind the tiles, then their sums
constexpr size_t kMaxExperts = 1024, kMaxTopK = 64, kMaxGroups = 64;
inline bool plan_geometry(size_t slots, size_t experts, PlanGeometry &g) {
    if (!experts || experts > kMaxExperts || slots >= (1ull << 30)) return false;
    size_t const buckets = slots < experts + 1 ? slots : experts + 1; // that can have any
    g.tile_rows = plan_tile_rows(slots, experts);
    g.max_tiles = (uint32_t)(slots / g.tile_rows + buckets);
    g.max_rows = (uint32_t)((slots + buckets * 15 + 15) / 16 * 16);
    g.offsets = sizeof(PlanHeader) / 4;
    g.order = g.offsets + ((experts + 2 + 3) & ~(size_t)3);
    g.place = g.order + g.max_rows;
    g.tiles = (g.place + slots + 3) & ~(size_t)3;
    g.table = g.tiles + (size_t)g.max_tiles * 4;
    g.total_words = g.table + ((slots + kPlanBlockSlots - 1) / kPlanBlockSlots + 1) * (experts + 1);
    return true;
}

#ifdef __HIP_DEVICE_COMPILE__
#define NK_MX_DEVICE_BUILTINS 1
#endif

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef v4u __attribute__((aligned(1))) v4u_anywhere; // loads and stores of global memory need no alignment
typedef uint32_t __attribute__((aligned(1))) u32_anywhere;
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

/** What a lane loads at once: 16 adjacent bytes of a row, four values of f32 and eight of bf16 and f16. */
template <class T>
constexpr int kEach = 16 / (int)sizeof(T);
/** They as 32-bit floats. (Widening is exact, so whatever follows sees the values themselves; a kernel loads several times
 *  before it widens the first.) */
template <class T>
__device__ __forceinline__ void widen(v4u words, float (&v)[kEach<T>]) {
#pragma unroll
    for (int i = 0; i < kEach<T>; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(words[i]);
        else if constexpr (__is_same(T, __bf16)) v[i] = __uint_as_float(i % 2 ? words[i / 2] & 0xFFFF0000u : words[i / 2] << 16);
        else v[i] = (float)__builtin_bit_cast(f16x2, (uint32_t)words[i / 2])[i % 2];
    }
}
/** Values of a row from column `col` on, wherever they lie; zeros from column `k` on. */
template <class T>
__device__ __forceinline__ void load_some(T const *row, uint32_t col, uint32_t k, float (&v)[kEach<T>]) {
#pragma unroll
    for (int i = 0; i < kEach<T>; ++i) v[i] = col + i < k ? (float)row[col + i] : 0.0f;
}

/** The largest of the adjacent lanes that share a block, in all of them: four lanes, or eight of f32. */
template <int LANES>
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
    uint32_t const y = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true); // lanes 1 0 3 2
    x = x > y ? x : y;
    uint32_t const z = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true); // lanes 2 3 0 1
    x = x > z ? x : z;
    if (LANES == 8) {
        uint32_t const w = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, true); // eights mirrored
        x = x > w ? x : w;
    }
    return x;
}

/**
 *  A lane's values of a block of 32 that adjacent lanes hold, to codes (four bits each, the first lowest) and the block's scale
 *  byte. The exponent field of the largest magnitude, less 2, is the scale: e2m1's largest exponent is 2. (Magnitudes are
 *  compared as integers; a NaN or an infinity has the largest exponent field and so decides for its block; subnormal blocks end
 *  at 2^-127.) The conversion divides by the scale, rounds to nearest even and saturates: measured equal to that definition on
 *  every bf16 value and on f32 and f16 values of every size, at scales from 2^-127 to 2^127.
 */
template <int N>
__device__ __forceinline__ uint32_t quantize_some(float const (&v)[N], uint32_t &scale) {
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        uint32_t const magnitude = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        largest = largest > magnitude ? largest : magnitude;
    }
    largest = block_max<32 / N>(largest);
    uint32_t const field = largest >> 23;
    scale = field == 255 ? 255 : field > 2 ? field - 2 : 0;
    float const power = __uint_as_float(scale ? scale << 23 : 0x00400000u);
    uint32_t codes = 0;
#ifdef NK_MX_DEVICE_BUILTINS
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], power, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], power, 1);
    if constexpr (N == 8) {
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], power, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], power, 3);
    }
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

/** The same with v_mfma_scale_f32_32x32x64_f8f6f4: lane l brings row l % 32, block l / 32 of two. */
template <int U>
__device__ __forceinline__ v16f mx_multiply(v4u w, v4u a, v16f acc, uint32_t w_scale, uint32_t a_scale) {
#ifdef NK_MX_DEVICE_BUILTINS
    v8i const x = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    v8i const y = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, acc, 4, 4, U, (int)w_scale, U, (int)a_scale);
#else
    return acc;
#endif
}

typedef __attribute__((address_space(3))) void mx_lds_t;
/** 16 bytes per lane at `lane_offset` + `offset` (the same in all lanes) of a buffer into LDS at `dst` + 16 x lane. */
__device__ __forceinline__ void fetch_16(__amdgpu_buffer_rsrc_t buffer, void *dst, uint32_t lane_offset, uint32_t offset) {
#ifdef NK_MX_DEVICE_BUILTINS
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (mx_lds_t *)dst, 16, (int)lane_offset, (int)offset, 0, 0);
#endif
}

/** 16, 4 or 8 bytes per lane at `lane_offset` + `offset` (the same in all lanes) of a buffer. */
__device__ __forceinline__ v4u load_16(__amdgpu_buffer_rsrc_t buffer, uint32_t lane_offset, uint32_t offset) {
#ifdef NK_MX_DEVICE_BUILTINS
    return __builtin_amdgcn_raw_buffer_load_b128(buffer, (int)lane_offset, (int)offset, 0);
#else
    return v4u {0, 0, 0, 0};
#endif
}
__device__ __forceinline__ uint32_t load_4(__amdgpu_buffer_rsrc_t buffer, uint32_t lane_offset, uint32_t offset) {
#ifdef NK_MX_DEVICE_BUILTINS
    return __builtin_amdgcn_raw_buffer_load_b32(buffer, (int)lane_offset, (int)offset, 0);
#else
    return 0;
#endif
}
__device__ __forceinline__ v2u load_8(__amdgpu_buffer_rsrc_t buffer, uint32_t lane_offset, uint32_t offset) {
#ifdef NK_MX_DEVICE_BUILTINS
    return __builtin_amdgcn_raw_buffer_load_b64(buffer, (int)lane_offset, (int)offset, 0);
#else
    return v2u {0, 0};
#endif
}
/** What is at `base`, the same in all lanes, as a buffer (callers stay inside what they address by it). */
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(void const *base) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, 0xFFFFFFFFu, 0x00020000);
}

/** 16 bytes to any address. */
__device__ __forceinline__ void store_16(void *to, v4u values) {
    *(v4u_anywhere *)to = values;
}

/** What lanes of a wavefront have written to LDS is there for its other lanes. */
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/** A number that a lambda's argument carries at compile time. */
template <int N>
struct Number {
    static constexpr int value = N;
};

/** `count` (up to N) adjacent results at `to`: all N as vectors, which global memory takes at any element's address. */
template <class Out, int N>
__device__ __forceinline__ void store_some(Out *to, float const (&v)[N], uint32_t count) {
    if (count >= N) {
        struct __attribute__((packed, aligned(sizeof(Out)))) Pack {
            Out x[N];
        } pack;
#pragma unroll
        for (int i = 0; i < N; ++i) pack.x[i] = (Out)v[i];
        __builtin_memcpy(to, &pack, sizeof(pack));
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if ((uint32_t)i < count) to[i] = (Out)v[i];
}

} // namespace nk_gfx950

#endif // NUMKONG_AMD_MX_GFX950_HPP
