/**
 *  @brief Microscaled 4-bit floats on gfx950: quantising, packing, products, the experts' products.
 *  @file numkong_amd/csrc/mx_gfx950.hip
 *
 *  Implements the mx half of <numkong_amd/mx.h>; formats and the shared pieces are in mx_gfx950.hpp.
 */
#include "mx_gfx950.hpp"

namespace nk_gfx950 {
namespace {

// ---- quantising and back ------------------------------------------------------------------------------------------

/**
 *  One thread for eight adjacent values, four for a block, so that a wavefront reads 1 KiB (2 KiB of f32) in one piece.
 *  STAGED: rows padded with zeros to whole steps and scales in the order of the products' operands (mx_gfx950.hpp);
 *  otherwise rows as the caller has them. `pieces`: eights of a row, whole blocks (STAGED: whole steps).
 */
template <class T, bool STAGED>
__global__ __launch_bounds__(256) void quantize_kernel(T const *x, uint64_t x_stride, uint32_t rows, uint32_t k, uint32_t pieces,
                                                       bool wide, uint8_t *codes, uint64_t codes_stride, bool whole_words,
                                                       uint8_t *scales, uint64_t scales_stride) {
    uint32_t const index = blockIdx.x * 256 + threadIdx.x;
    uint32_t const row = index / pieces, piece = index - row * pieces;
    if (row >= rows) return; // (pieces is a multiple of four: a block's lanes leave together)
    uint32_t const col = piece * 8;
    float v[8];
    load_eight((T const *)((uint8_t const *)x + row * x_stride), col, k, wide, v);
    uint32_t scale;
    uint32_t const word = quantize_eight(v, scale);
    uint32_t const block = piece >> 2;
    uint8_t *to = codes + row * codes_stride + piece * 4;
    if (STAGED) {
        *(uint32_t *)to = word;
        if (!(piece & 3)) scales[row * scales_stride + (block & ~15u) + (block & 3) * 4 + (block >> 2 & 3)] = (uint8_t)scale;
        return;
    }
    uint32_t const bytes = col >= k ? 0 : (k - col + 1) / 2;
    if (whole_words && bytes >= 4) *(uint32_t *)to = word;
    else
        for (uint32_t i = 0; i < (bytes < 4 ? bytes : 4); ++i) to[i] = (uint8_t)(word >> 8 * i);
    if (!(piece & 3)) scales[row * scales_stride + block] = (uint8_t)scale;
}

/** Rows of codes and scales as callers have them, to the staged form. One thread for a block. */
__global__ __launch_bounds__(256) void stage_codes_kernel(uint8_t const *codes, uint64_t codes_stride, uint8_t const *scales,
                                                          uint64_t scales_stride, uint32_t rows, uint32_t k, uint32_t blocks,
                                                          bool wide, uint8_t *to, uint64_t to_stride, uint8_t *to_scales,
                                                          uint64_t to_scales_stride) {
    uint32_t const index = blockIdx.x * 256 + threadIdx.x;
    uint32_t const row = index / blocks, block = index - row * blocks;
    if (row >= rows) return;
    uint8_t const *from = codes + row * codes_stride + block * 16;
    bool const inside = block * 32 < k;
    v4u word = {0, 0, 0, 0};
    if (wide && block * 32 + 32 <= k) word = *(v4u const *)from;
    else if (inside)
        for (uint32_t i = 0; i < 16; ++i) {
            uint32_t const col = block * 32 + 2 * i;
            uint32_t const byte = col + 1 < k ? from[i] : col < k ? from[i] & 15u : 0u;
            word[i / 4] |= byte << 8 * (i % 4);
        }
    *(v4u *)(to + row * to_stride + block * 16) = word;
    uint8_t const scale = inside ? scales[row * scales_stride + block] : (uint8_t)0;
    to_scales[row * to_scales_stride + (block & ~15u) + (block & 3) * 4 + (block >> 2 & 3)] = scale;
}

/** value = q * 2^(s - 127), built from the bits: 2 |q| is a whole number up to 12, and 12 * 2^(s - 128) fits 32 bits. */
template <class T>
__global__ __launch_bounds__(256) void dequantize_kernel(uint8_t const *codes, uint64_t codes_stride, bool whole_words,
                                                         uint8_t const *scales, uint64_t scales_stride, uint32_t rows,
                                                         uint32_t k, uint32_t pieces, T *x, uint64_t x_stride, bool wide) {
    uint32_t const index = blockIdx.x * 256 + threadIdx.x;
    uint32_t const row = index / pieces, col = (index - row * pieces) * 8;
    if (row >= rows) return;
    uint8_t const *from = codes + row * codes_stride + col / 2;
    uint32_t word = 0;
    if (whole_words && col + 8 <= k) word = *(uint32_t const *)from;
    else
        for (uint32_t i = 0; i < 4; ++i)
            if (col + 2 * i < k) word |= (uint32_t)from[i] << 8 * i;
    uint32_t const scale = scales[row * scales_stride + col / 32];
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t const code = word >> 4 * i & 15u;
        uint32_t const twice = (0xC8643210u >> 4 * (code & 7u)) & 15u; // 0 1 2 3 4 6 8 12
        float const magnitude = scale == 255 ? __uint_as_float(0x7FC00000u) : ldexpf((float)twice, (int)scale - 128);
        v[i] = code & 8u ? -magnitude : magnitude;
    }
    store_some<T, 8>((T *)((uint8_t *)x + row * x_stride) + col, v, k - col, wide);
}

// ---- packing ------------------------------------------------------------------------------------------------------

/** One thread for 16 bytes of a tile's codes or for a word of its scales; the header by the first workgroup. */
__global__ __launch_bounds__(256) void mx_pack_kernel(uint8_t const *codes, uint64_t codes_stride, uint64_t codes_matrix,
                                                      uint8_t const *scales, uint64_t scales_stride, uint64_t scales_matrix,
                                                      MxHeader header, uint32_t steps, uint32_t supers, uint32_t tiles,
                                                      uint64_t first, uint64_t code_lanes, uint64_t scale_lanes, bool wide,
                                                      uint8_t *image) {
    uint64_t const index = first + (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (index == 0) *(MxHeader *)image = header;
    uint32_t const lane = index & 63, g = lane >> 4;
    bool const of_codes = index < code_lanes * header.count;
    uint64_t const at = (of_codes ? index : index - code_lanes * header.count) >> 6;
    if (!of_codes && at >= scale_lanes / 64 * header.count) return;
    uint32_t const across = of_codes ? steps : supers;
    uint32_t const which = (uint32_t)(at % across); // step or super
    uint64_t const tile_of_all = at / across;
    uint32_t const tile = (uint32_t)(tile_of_all % tiles);
    uint64_t const matrix = tile_of_all / tiles;
    uint32_t const q = lane & 15, column = (tile >> 2) * 64 + (q >> 2) * 16 + (tile & 3) * 4 + (q & 3);
    uint32_t const k = header.k;
    if (of_codes) {
        uint32_t const block = which * 4 + g;
        uint8_t const *from = codes + matrix * codes_matrix + column * codes_stride + block * 16;
        v4u word = {0, 0, 0, 0};
        if (column < header.n) {
            if (wide && block * 32 + 32 <= k) word = *(v4u const *)from;
            else
                for (uint32_t i = 0; i < 16; ++i) {
                    uint32_t const col = block * 32 + 2 * i;
                    uint32_t const byte = col + 1 < k ? from[i] : col < k ? from[i] & 15u : 0u;
                    word[i / 4] |= byte << 8 * (i % 4);
                }
        }
        *(v4u *)(image + kMxHeaderBytes + index * 16) = word;
        return;
    }
    uint32_t word = 0;
    for (uint32_t u = 0; u < 4; ++u) {
        uint32_t const block = which * 16 + u * 4 + g;
        if (column < header.n && block * 32 < k)
            word |= (uint32_t)scales[matrix * scales_matrix + column * scales_stride + block] << 8 * u;
    }
    *(uint32_t *)(image + kMxHeaderBytes + code_lanes * header.count * 16 + (index - code_lanes * header.count) * 4) = word;
}

// ---- products -----------------------------------------------------------------------------------------------------

struct MxArgs {
    uint8_t const *a; // staged codes, or the caller's floats (products of few rows that quantise them themselves)
    uint8_t const *a_scales;
    uint8_t const *image;
    uint8_t *c;
    uint32_t const *plan; // NULL: one matrix, rows in order
    uint64_t a_pitch, scales_pitch, c_stride;
    uint32_t m, n, k, steps, supers, tiles, count;
    uint32_t tiles_m, tiles_n; // the grid: tiles of rows, tiles of columns
    uint32_t order, tile_list; // words into the plan
    uint32_t a_share;          // slots that share a row of A
    uint32_t sorted;           // 1: results in the plan's order of rows (and nothing for rows of no expert), 0: at their slots
    uint32_t a_wide, c_wide;
};

/** The rows of one tile. */
struct RowTile {
    uint32_t matrix, first, last; // rows [first, last): of C, or of the plan
    bool zero;                    // rows of no expert
};
__device__ __forceinline__ bool row_tile_of(MxArgs const &p, uint32_t tile, uint32_t rows, RowTile &t) {
    if (!p.plan) {
        t.matrix = 0, t.first = tile * rows, t.last = t.first + rows < p.m ? t.first + rows : p.m, t.zero = false;
        return true;
    }
    if (tile >= ((PlanHeader const *)p.plan)->tile_count) return false;
    PlanTile const entry = *(PlanTile const *)(p.plan + p.tile_list + tile * 4);
    t.matrix = (uint32_t)entry.expert, t.first = (uint32_t)entry.first, t.last = (uint32_t)entry.last;
    t.zero = t.matrix >= p.count;
    return !(t.zero && p.sorted);
}
__device__ __forceinline__ bool image_matches(MxArgs const &p) {
    MxHeader const h = *(MxHeader const *)p.image;
    return h.magic == kMxMagic && h.version == 1 && h.count == p.count && h.n == p.n && h.k == p.k;
}
/** Workgroup to tile: each of the eight dies gets one stretch of the walk, `bands` of eight tiles of rows at a time. */
__device__ __forceinline__ bool grid_tile(MxArgs const &p, uint32_t &tile_m, uint32_t &tile_n) {
    uint32_t const total = p.tiles_m * p.tiles_n, per = (total + 7) / 8;
    uint32_t const index = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || index >= total) return false;
    if (p.plan) { // the tiles of one expert stand side by side: their rows stay while the columns go by
        tile_m = index / p.tiles_n, tile_n = index - tile_m * p.tiles_n;
        return true;
    }
    uint32_t const band = index / (8 * p.tiles_n), first = band * 8, inside = index - band * 8 * p.tiles_n;
    uint32_t const high = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
    tile_n = inside / high, tile_m = first + inside - tile_n * high;
    return true;
}

/**
 *  The product for many rows: 16 WM FM rows x 64 WN columns by WM x WN wavefronts, each FM x 4 fragments of 16 x 16.
 *  Both operands go straight into LDS (four stages of one step, fetched three ahead), in the order in which fragments are
 *  read, so that no read meets another's bank; scales the same way, one super ahead. A stage's fetches are counted, not
 *  drained: every wavefront waits for its own, then all meet.
 */
template <int FM, int WM, int WN, class Out, bool GROUPED>
__global__ __launch_bounds__(64 * WM * WN) void mx_gemm_kernel(MxArgs p) {
    constexpr int kWaves = WM * WN, kA = WM * FM, kFragments = kA + WN * 4, kLoads = kFragments / kWaves;
    static_assert(kFragments % kWaves == 0, "every wavefront fetches the same number of fragments");
    constexpr int kRows = kA * 16, kColumns = WN * 64;
    __shared__ __attribute__((aligned(1024))) uint8_t ring0[kFragments * 1024];
    __shared__ __attribute__((aligned(1024))) uint8_t ring1[kFragments * 1024];
    __shared__ __attribute__((aligned(1024))) uint8_t ring2[kFragments * 1024];
    __shared__ __attribute__((aligned(1024))) uint8_t ring3[kFragments * 1024];
    __shared__ __attribute__((aligned(1024))) uint8_t scale0[kFragments * 256];
    __shared__ __attribute__((aligned(1024))) uint8_t scale1[kFragments * 256];

    uint32_t tile_m, tile_n;
    if (!grid_tile(p, tile_m, tile_n)) return;
    RowTile rows;
    if (!row_tile_of(p, tile_m, kRows, rows)) return;
    uint32_t const lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    bool const good = image_matches(p);

    v4f acc[FM][4];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = v4f {0, 0, 0, 0};

    if (good && !(GROUPED && rows.zero) && p.steps) {
        // what this wavefront fetches: fragments wave * kLoads ... of the stage, A's first
        uint8_t const *from[kLoads], *scale_from[kLoads];
        uint32_t advance[kLoads], scale_advance[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            uint32_t const f = wave * kLoads + i;
            if (f < (uint32_t)kA) {
                uint32_t at = rows.first + f * 16 + r;
                at = at < rows.last ? at : rows.last - 1; // (results of rows past the end are not stored)
                uint32_t const row = GROUPED ? p.plan[p.order + at] / p.a_share : at;
                from[i] = p.a + row * p.a_pitch + g * 16, advance[i] = 64;
                scale_from[i] = p.a_scales + row * p.scales_pitch + g * 4, scale_advance[i] = 16;
            }
            else {
                uint32_t tile = tile_n * (WN * 4) + f - kA;
                tile = tile < p.tiles ? tile : p.tiles - 1;
                uint64_t const of_all = (uint64_t)rows.matrix * p.tiles + tile;
                from[i] = p.image + kMxHeaderBytes + of_all * p.steps * 1024 + lane * 16, advance[i] = 1024;
                scale_from[i] = p.image + kMxHeaderBytes + (uint64_t)p.count * p.tiles * p.steps * 1024 + of_all * p.supers * 256 + lane * 4;
                scale_advance[i] = 256;
            }
        }
        uint32_t const last_step = p.steps - 1, last_super = p.supers - 1;
        auto fetch = [&](uint32_t step, uint8_t *ring) __attribute__((always_inline)) {
            step = step < last_step ? step : last_step; // (past the end: the last once more, so that the counts stay)
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                fetch_16(from[i] + (uint64_t)step * advance[i], ring + (wave * kLoads + i) * 1024);
        };
        auto fetch_scales = [&](uint32_t super, uint8_t *ring) __attribute__((always_inline)) {
            super = super < last_super ? super : last_super;
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                fetch_4(scale_from[i] + (uint64_t)super * scale_advance[i], ring + (wave * kLoads + i) * 256);
        };
        uint32_t a_scale[FM], w_scale[4];
        auto read_scales = [&](uint8_t const *ring) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < FM; ++i) a_scale[i] = *(uint32_t const *)(ring + (wm * FM + i) * 256 + lane * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) w_scale[j] = *(uint32_t const *)(ring + (kA + wn * 4 + j) * 256 + lane * 4);
        };
        auto step_of = [&](auto byte, uint8_t const *ring) __attribute__((always_inline)) {
            constexpr int U = decltype(byte)::value;
            v4u w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = *(v4u const *)(ring + (kA + wn * 4 + j) * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                v4u const a = *(v4u const *)(ring + (wm * FM + i) * 1024 + lane * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = mx_multiply<U>(w[j], a, acc[i][j], w_scale[j], a_scale[i]);
            }
        };
        // Every fetch into what is read next has arrived (`younger` were issued behind it and may be in flight), this
        // wavefront's reads are done, and everybody says so.
        auto meet = [&](auto younger_) __attribute__((always_inline)) {
            constexpr int younger = decltype(younger_)::value;
            static_assert(younger < 64, "what a wait can count to");
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0x0070 | (younger & 15) | (younger >> 4) << 14);
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        Number<0> const zero;
        Number<1> const one;
        Number<2> const two;
        Number<3> const three;
        Number<2 * kLoads> const few;  // two stages behind
        Number<3 * kLoads> const more; // two stages and a super's scales
        fetch_scales(0, scale0);
        fetch(0, ring0), fetch(1, ring1), fetch(2, ring2);
        uint32_t const whole = p.steps / 4, rest = p.steps % 4;
        // Stage s: wait for its fetches (three stages old), then fetch stage s + 3 into what stage s - 1 has left.
        auto super_of = [&](uint32_t q, uint8_t *scales_now, uint8_t *scales_next) __attribute__((always_inline)) {
            meet(few);
            fetch_scales(q + 1, scales_next), fetch(4 * q + 3, ring3);
            read_scales(scales_now);
            step_of(zero, ring0);
            meet(more);
            fetch(4 * q + 4, ring0);
            step_of(one, ring1);
            meet(more);
            fetch(4 * q + 5, ring1);
            step_of(two, ring2);
            meet(few);
            fetch(4 * q + 6, ring2);
            step_of(three, ring3);
        };
        uint32_t q = 0;
        for (; q + 2 <= whole; q += 2) super_of(q, scale0, scale1), super_of(q + 1, scale1, scale0);
        if (q < whole) super_of(q, scale0, scale1), ++q;
        meet(Number<0>()); // (nothing is fetched from here on)
        if (rest) {
            read_scales(q & 1 ? scale1 : scale0);
            step_of(zero, ring0);
            if (rest > 1) step_of(one, ring1);
            if (rest > 2) step_of(two, ring2);
        }
    }

    float const poison = __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        uint32_t const at = rows.first + (wm * FM + i) * 16 + r;
        if (at >= rows.last) continue;
        uint32_t const row = GROUPED && !p.sorted ? p.plan[p.order + at] : at;
        uint32_t const column = tile_n * kColumns + wn * 64 + g * 16;
        if (column >= p.n) continue;
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = good ? acc[i][j / 4][j % 4] : poison;
        store_some<Out, 16>((Out *)(p.c + row * p.c_stride) + column, v, p.n - column, p.c_wide);
    }
}

/**
 *  The product for few rows: the stream of B is the work, so a workgroup takes 16 NT columns and its eight wavefronts a
 *  stretch of the depth each, B straight into registers, and their sums meet in LDS. In: the type of A's values, which
 *  the workgroup quantises into LDS itself (one launch, and A is read by all lanes), or `uint8_t`: A is staged already.
 */
constexpr int kFewWaves = 8;
template <int FM, int NT, class In, class Out, bool GROUPED>
__global__ __launch_bounds__(64 * kFewWaves) void mx_few_kernel(MxArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
    constexpr bool FUSED = sizeof(In) != 1;
    uint32_t const tile_m = blockIdx.x / p.tiles_n, tile_n = blockIdx.x - tile_m * p.tiles_n;
    RowTile rows;
    if (!row_tile_of(p, tile_m, FM * 16, rows)) return;
    uint32_t const lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    bool const good = image_matches(p);
    uint32_t const here = rows.last - rows.first;
    v4f acc[FM][NT];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4f {0, 0, 0, 0};

    uint32_t const lds_pitch = p.steps * 64 + 16; // (16 bytes on: rows start in different banks)
    uint8_t *lds_scales = few_lds + here * lds_pitch;
    bool const computes = good && !(GROUPED && rows.zero) && p.steps;
    if (FUSED && computes) {
        uint32_t const pieces = p.steps * 16;
        for (uint32_t index = threadIdx.x; index < here * pieces; index += 64 * kFewWaves) {
            uint32_t const row = index / pieces, piece = index - row * pieces;
            uint32_t const at = rows.first + row, source = GROUPED ? p.plan[p.order + at] / p.a_share : at;
            float v[8];
            if constexpr (FUSED) load_eight((In const *)(p.a + source * p.a_pitch), piece * 8, p.k, p.a_wide, v);
            uint32_t scale;
            uint32_t const word = quantize_eight(v, scale);
            *(uint32_t *)(few_lds + row * lds_pitch + piece * 4) = word;
            if (!(piece & 3)) lds_scales[row * (p.steps * 4) + (piece >> 2)] = (uint8_t)scale;
        }
    }
    if (FUSED) __syncthreads();
    if (computes) {
        uint32_t const begin = (uint32_t)((uint64_t)wave * p.steps / kFewWaves), end = (uint32_t)((uint64_t)(wave + 1) * p.steps / kFewWaves);
        uint64_t const of_all = (uint64_t)rows.matrix * p.tiles + tile_n * NT;
        uint8_t const *w_from = p.image + kMxHeaderBytes + of_all * p.steps * 1024 + lane * 16;
        uint8_t const *w_scale_from = p.image + kMxHeaderBytes + (uint64_t)p.count * p.tiles * p.steps * 1024 + of_all * p.supers * 256 + lane * 4;
        uint8_t const *a_from[FM], *a_scale_from[FM];
        bool there[FM];
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            there[i] = i * 16 + r < here;
            uint32_t const row = there[i] ? i * 16 + r : 0;
            if constexpr (FUSED) a_from[i] = few_lds + row * lds_pitch + g * 16, a_scale_from[i] = lds_scales + row * (p.steps * 4) + g;
            else {
                uint32_t const at = rows.first + row, source = GROUPED ? p.plan[p.order + at] / p.a_share : at;
                a_from[i] = p.a + source * p.a_pitch + g * 16, a_scale_from[i] = p.a_scales + source * p.scales_pitch + g * 4;
            }
        }
        constexpr int kBatch = 4;
        for (uint32_t base = begin; base < end; base += kBatch) {
            v4u w[kBatch][NT], a[kBatch][FM];
            uint32_t w_scale[kBatch][NT], a_scale[kBatch][FM];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                uint32_t const s = base + u < end ? base + u : end - 1;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    w[u][j] = *(v4u const *)(w_from + ((uint64_t)j * p.steps + s) * 1024);
                    w_scale[u][j] = *(uint32_t const *)(w_scale_from + ((uint64_t)j * p.supers + (s >> 2)) * 256) >> 8 * (s & 3);
                }
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    a[u][i] = *(v4u const *)(a_from[i] + (uint64_t)s * 64);
                    if constexpr (FUSED) a_scale[u][i] = a_scale_from[i][s * 4];
                    else a_scale[u][i] = *(uint32_t const *)(a_scale_from[i] + (s >> 2) * 16) >> 8 * (s & 3);
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (base + u >= end) break;
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    v4u const rows_of_a = there[i] ? a[u][i] : v4u {0, 0, 0, 0};
                    uint32_t const scale_of_a = there[i] ? a_scale[u][i] : 0;
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = mx_multiply<0>(w[u][j], rows_of_a, acc[i][j], w_scale[u][j], scale_of_a);
                }
            }
        }
    }
    if (FUSED) __syncthreads(); // (the sums go where A was)
    v4f *sums = (v4f *)few_lds;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) sums[(wave * FM * NT + i * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    float const poison = __uint_as_float(0x7FC00000u);
    for (uint32_t index = threadIdx.x; index < FM * NT * 64; index += 64 * kFewWaves) {
        uint32_t const of_lane = index & 63, fragment = index >> 6, i = fragment / NT, j = fragment % NT;
        uint32_t const local = i * 16 + (of_lane & 15);
        if (local >= here) continue;
        v4f sum = sums[index];
#pragma unroll
        for (int w = 1; w < kFewWaves; ++w) sum += sums[w * FM * NT * 64 + index];
        uint32_t const at = rows.first + local, row = GROUPED && !p.sorted ? p.plan[p.order + at] : at;
        uint32_t const tile = tile_n * NT + j, column = (tile >> 2) * 64 + (of_lane >> 4) * 16 + (tile & 3) * 4;
        if (column >= p.n) continue;
        float v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = good ? sum[t] : poison;
        store_some<Out, 4>((Out *)(p.c + row * p.c_stride) + column, v, p.n - column, p.c_wide);
    }
}

/** out[token] = sum over its slots of weight * row of the plan, slots without an expert left out; a thread for four columns. */
template <class In, class Out>
__global__ __launch_bounds__(256) void combine_kernel(In const *rows, uint64_t row_values, uint32_t const *plan, uint32_t place,
                                                      float const *weights, uint32_t top_k, uint32_t tokens, uint32_t n,
                                                      uint32_t pieces, Out *c, uint64_t c_stride, bool wide) {
    uint32_t const index = blockIdx.x * 256 + threadIdx.x;
    uint32_t const token = index / pieces, column = (index - token * pieces) * 4;
    if (token >= tokens) return;
    float sum[4] = {0, 0, 0, 0};
    for (uint32_t i = 0; i < top_k; ++i) {
        uint32_t const slot = token * top_k + i;
        int32_t const row = (int32_t)plan[place + slot];
        if (row < 0) continue;
        float const weight = weights[slot];
        struct alignas(4 * sizeof(In)) Four {
            In x[4];
        } const four = *(Four const *)(rows + (uint64_t)row * row_values + column); // (rows are padded to whole fours)
#pragma unroll
        for (int t = 0; t < 4; ++t) sum[t] = __builtin_fmaf(weight, (float)four.x[t], sum[t]);
    }
    store_some<Out, 4>((Out *)((uint8_t *)c + token * c_stride) + column, sum, n - column, wide);
}

// ---- host side ----------------------------------------------------------------------------------------------------

int element_bytes(int dtype) { return dtype == nk_f32_k ? 4 : dtype == nk_bf16_k || dtype == nk_f16_k ? 2 : 0; }
bool aligned(void const *ptr, uint64_t stride, uint64_t to) { return !(((uintptr_t)ptr | stride) & (to - 1)); }
constexpr uint64_t kMostThreads = 1ull << 31;

/** Calls `f` with a value of the element type's C++ type. */
template <class F>
int with_type(int dtype, F &&f) {
    if (dtype == nk_f32_k) return f(float());
    if (dtype == nk_bf16_k) return f(__bf16());
    return f(_Float16());
}

template <bool STAGED>
int launch_quantize(int dtype, void const *x, uint64_t rows, uint32_t k, uint64_t x_stride, uint8_t *codes, uint64_t codes_stride,
                    uint8_t *scales, uint64_t scales_stride, hipStream_t stream) {
    uint64_t const pieces = STAGED ? (uint64_t)(k + 127) / 128 * 16 : (uint64_t)(k + 31) / 32 * 4;
    if (!rows || !pieces) return 0;
    bool const wide = aligned(x, x_stride, 16), whole_words = aligned(codes, codes_stride, 4);
    uint64_t const slab = kMostThreads / pieces; // rows of one launch
    for (uint64_t first = 0; first < rows; first += slab) {
        uint64_t const here = rows - first < slab ? rows - first : slab;
        uint8_t const *from = (uint8_t const *)x + first * x_stride;
        int const status = with_type(dtype, [&](auto value) {
            typedef decltype(value) T;
            hipLaunchKernelGGL((quantize_kernel<T, STAGED>), dim3((uint32_t)((here * pieces + 255) / 256)), dim3(256), 0, stream,
                               (T const *)from, x_stride, (uint32_t)here, k, (uint32_t)pieces, wide, codes + first * codes_stride,
                               codes_stride, whole_words, scales + first * scales_stride, scales_stride);
            hipError_t const e = hipGetLastError();
            return e == hipSuccess ? 0 : mx_fail(e, "quantize_kernel");
        });
        if (status) return status;
    }
    return 0;
}

/** How A is laid out in the workspace. */
struct Staging {
    uint64_t pitch, scales_pitch, scales_at, bytes;
};
Staging staging_of(uint64_t rows, MxGeometry const &g) {
    Staging s;
    // rows an odd number of 256 bytes apart: a stage reads 64 bytes of each row of a tile, and with a power of two between
    // rows these would all come from the same few channels of the L2
    s.pitch = (uint64_t)g.steps * 64;
    s.pitch = (s.pitch + 255) / 256 * 256;
    if (!(s.pitch & 256)) s.pitch += 256;
    s.scales_pitch = (uint64_t)g.supers * 16;
    s.scales_at = rows * s.pitch;
    s.bytes = (s.scales_at + rows * s.scales_pitch + 255) / 256 * 256;
    return s;
}
int stage(int a_dtype, void const *a, uint64_t a_stride, void const *a_scales, uint64_t a_scales_stride, uint64_t rows, uint32_t k,
          MxGeometry const &g, Staging const &s, uint8_t *to, hipStream_t stream) {
    if (!a_scales) return launch_quantize<true>(a_dtype, a, rows, k, a_stride, to, s.pitch, to + s.scales_at, s.scales_pitch, stream);
    uint32_t const blocks = g.steps * 4;
    if (!rows || !blocks) return 0;
    uint64_t const slab = kMostThreads / blocks;
    for (uint64_t first = 0; first < rows; first += slab) {
        uint64_t const here = rows - first < slab ? rows - first : slab;
        hipLaunchKernelGGL(stage_codes_kernel, dim3((uint32_t)((here * blocks + 255) / 256)), dim3(256), 0, stream,
                           (uint8_t const *)a + first * a_stride, a_stride, (uint8_t const *)a_scales + first * a_scales_stride,
                           a_scales_stride, (uint32_t)here, k, blocks, aligned(a, a_stride, 16), to + first * s.pitch, s.pitch,
                           to + s.scales_at + first * s.scales_pitch, s.scales_pitch);
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, "stage_codes_kernel");
    }
    return 0;
}

/** Can products of few rows quantise A themselves? What a workgroup holds of it has to fit, and to stay small. */
constexpr uint32_t kFusedBytes = 64 * 1024;
uint32_t fused_bytes(uint32_t rows, MxGeometry const &g) { return rows * (g.steps * 64 + 16) + rows * g.steps * 4; }
bool fuses(uint64_t rows, MxGeometry const &g) { return rows <= 16 && (uint64_t)rows * (g.steps * 68 + 16) <= kFusedBytes; }

template <int FM, int NT, class In, class Out, bool GROUPED>
int launch_few(MxArgs &p, uint32_t max_rows, MxGeometry const &g, hipStream_t stream) {
    p.tiles_n = (p.tiles + NT - 1) / NT;
    uint64_t const grid = (uint64_t)p.tiles_m * p.tiles_n;
    if (grid > 0x7FFFFFFFull) return mx_fail("mx product: too many tiles");
    uint32_t lds = kFewWaves * FM * NT * 1024;
    if (sizeof(In) != 1 && fused_bytes(max_rows, g) > lds) lds = fused_bytes(max_rows, g);
    hipLaunchKernelGGL((mx_few_kernel<FM, NT, In, Out, GROUPED>), dim3((uint32_t)grid), dim3(64 * kFewWaves), lds, stream, p);
    hipError_t const e = hipGetLastError();
    return e == hipSuccess ? 0 : mx_fail(e, "mx_few_kernel");
}
template <int FM, int WM, int WN, class Out, bool GROUPED>
int launch_gemm(MxArgs &p, hipStream_t stream) {
    p.tiles_n = (p.tiles + WN * 4 - 1) / (WN * 4);
    if (!GROUPED) p.tiles_m = (p.m + 16 * WM * FM - 1) / (16 * WM * FM);
    uint64_t const grid = ((uint64_t)p.tiles_m * p.tiles_n + 7) / 8 * 8;
    if (grid > 0x7FFFFFFFull) return mx_fail("mx product: too many tiles");
    hipLaunchKernelGGL((mx_gemm_kernel<FM, WM, WN, Out, GROUPED>), dim3((uint32_t)grid), dim3(64 * WM * WN), 0, stream, p);
    hipError_t const e = hipGetLastError();
    return e == hipSuccess ? 0 : mx_fail(e, "mx_gemm_kernel");
}

/** Which kernel: by the rows of a tile (the plan's where there is one). */
template <class Out, bool GROUPED>
int launch_product(MxArgs &p, uint32_t rows, int a_dtype, bool fused, uint32_t fused_rows, MxGeometry const &g, hipStream_t stream) {
    if (rows <= 16) {
        if (!GROUPED) p.tiles_m = 1;
        if (!fused) return launch_few<1, 2, uint8_t, Out, GROUPED>(p, rows, g, stream);
        return with_type(a_dtype, [&](auto value) { return launch_few<1, 2, decltype(value), Out, GROUPED>(p, fused_rows, g, stream); });
    }
    if (rows <= 64) {
        if (!GROUPED) p.tiles_m = 1;
        if (rows <= 32) return launch_few<2, 2, uint8_t, Out, GROUPED>(p, rows, g, stream);
        return launch_few<4, 2, uint8_t, Out, GROUPED>(p, rows, g, stream);
    }
    if (GROUPED ? rows <= 128 : (uint64_t)((p.m + 255) / 256) * ((p.n + 255) / 256) < 256) return launch_gemm<4, 2, 2, Out, GROUPED>(p, stream);
    return launch_gemm<8, 2, 4, Out, GROUPED>(p, stream);
}

int check_a(int a_dtype, void const *a, void const *a_scales, uint64_t a_stride) {
    if (a_scales) return a ? 0 : mx_fail("mx product: codes are NULL");
    int const bytes = element_bytes(a_dtype);
    if (!bytes) return mx_fail("mx product: A has to be f32, bf16 or f16");
    if (!a || !aligned(a, a_stride, bytes)) return mx_fail("mx product: A is NULL or not aligned to its elements");
    return 0;
}
int check_c(int c_dtype, void const *c, uint64_t c_stride) {
    int const bytes = element_bytes(c_dtype);
    if (!bytes) return mx_fail("mx product: C has to be f32, bf16 or f16");
    if (!c || !aligned(c, c_stride, bytes)) return mx_fail("mx product: C is NULL or not aligned to its elements");
    return 0;
}

/** Where the parts of the experts' workspace are. */
struct ExpertsLayout {
    Staging staged;
    uint64_t sums_at, sums_values, bytes; // rows of the plan before they are summed: values a row
    int sums_dtype;
    bool fused;
};
ExpertsLayout experts_layout(uint64_t slots, uint64_t a_share, uint64_t experts, uint64_t n, MxGeometry const &g, bool a_is_codes,
                             int c_dtype, bool weighted) {
    ExpertsLayout l = {};
    l.fused = !a_is_codes && plan_tile_rows(slots, experts) == 16 && fuses(16, g);
    if (!l.fused) l.staged = staging_of((slots + a_share - 1) / a_share, g);
    l.sums_at = l.staged.bytes;
    // rows that are still to be summed by weight: as wide as the result where that is bf16 (each is rounded once more, by at
    // most 2^-9 of itself, half of what the result's own rounding may do to it; at 32 bits they are most of the traffic),
    // 32 bits otherwise (f16 might overflow where the sum does not)
    l.sums_dtype = c_dtype == nk_bf16_k ? nk_bf16_k : nk_f32_k;
    l.sums_values = (n + 15) / 16 * 16;
    l.bytes = l.sums_at + (weighted ? (slots * l.sums_values * element_bytes(l.sums_dtype) + 255) / 256 * 256 : 0);
    return l;
}

} // namespace
} // namespace nk_gfx950

using namespace nk_gfx950;

extern "C" {

int nk_amd_mx_quantize_async(nk_dtype_t dtype, void const *x, nk_size_t rows, nk_size_t depth, nk_size_t x_stride, void *codes,
                             nk_size_t codes_stride, void *scales, nk_size_t scales_stride, void *stream) {
    int const bytes = element_bytes(dtype);
    if (!bytes) return mx_fail("mx_quantize: x has to be f32, bf16 or f16");
    if (rows >= (1ull << 31) || depth >= (1ull << 31)) return mx_fail("mx_quantize: too many rows or columns");
    if (!rows || !depth) return 0;
    if (!x || !codes || !scales) return mx_fail("mx_quantize: NULL operand");
    if (!aligned(x, x_stride, bytes)) return mx_fail("mx_quantize: x is not aligned to its elements");
    return launch_quantize<false>(dtype, x, rows, (uint32_t)depth, x_stride, (uint8_t *)codes, codes_stride, (uint8_t *)scales,
                                  scales_stride, (hipStream_t)stream);
}

int nk_amd_mx_dequantize_async(nk_dtype_t dtype, void const *codes, nk_size_t codes_stride, void const *scales,
                               nk_size_t scales_stride, nk_size_t rows, nk_size_t depth, void *x, nk_size_t x_stride, void *stream) {
    int const bytes = element_bytes(dtype);
    if (!bytes) return mx_fail("mx_dequantize: x has to be f32, bf16 or f16");
    if (rows >= (1ull << 31) || depth >= (1ull << 31)) return mx_fail("mx_dequantize: too many rows or columns");
    if (!rows || !depth) return 0;
    if (!x || !codes || !scales) return mx_fail("mx_dequantize: NULL operand");
    if (!aligned(x, x_stride, bytes)) return mx_fail("mx_dequantize: x is not aligned to its elements");
    uint64_t const pieces = (depth + 7) / 8, slab = kMostThreads / pieces;
    for (uint64_t first = 0; first < rows; first += slab) {
        uint64_t const here = rows - first < slab ? rows - first : slab;
        int const status = with_type(dtype, [&](auto value) {
            typedef decltype(value) T;
            hipLaunchKernelGGL((dequantize_kernel<T>), dim3((uint32_t)((here * pieces + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                               (uint8_t const *)codes + first * codes_stride, codes_stride, aligned(codes, codes_stride, 4),
                               (uint8_t const *)scales + first * scales_stride, scales_stride, (uint32_t)here, (uint32_t)depth,
                               (uint32_t)pieces, (T *)((uint8_t *)x + first * x_stride), x_stride, aligned(x, x_stride, 16));
            hipError_t const e = hipGetLastError();
            return e == hipSuccess ? 0 : mx_fail(e, "dequantize_kernel");
        });
        if (status) return status;
    }
    return 0;
}

nk_size_t nk_amd_mx_packed_size(nk_size_t count, nk_size_t width, nk_size_t depth) {
    MxGeometry g;
    return mx_geometry(count, width, depth, g) ? g.total_bytes : 0;
}

int nk_amd_mx_pack_async(void const *codes, nk_size_t codes_stride, nk_size_t codes_matrix, void const *scales,
                         nk_size_t scales_stride, nk_size_t scales_matrix, nk_size_t count, nk_size_t width, nk_size_t depth,
                         void *packed, void *stream) {
    MxGeometry g;
    if (!mx_geometry(count, width, depth, g)) return mx_fail("mx_pack: unsupported dimensions");
    if (!packed || ((uintptr_t)packed & 15)) return mx_fail("mx_pack: the image has to be 16-byte aligned");
    if (count && width && depth && (!codes || !scales)) return mx_fail("mx_pack: NULL operand");
    MxHeader const header = {kMxMagic, 1, (uint32_t)count, (uint32_t)width, (uint32_t)depth, {0, 0, 0}};
    uint64_t const code_lanes = g.code_bytes / 16, scale_lanes = g.scale_bytes / 4;
    uint64_t const total = count * (code_lanes + scale_lanes);
    bool const wide = aligned(codes, codes_stride | codes_matrix, 16);
    uint64_t const steps = g.steps ? g.steps : 1, supers = g.supers ? g.supers : 1, tiles = g.tiles ? g.tiles : 1;
    for (uint64_t first = 0; first == 0 || first < total; first += kMostThreads) {
        uint64_t const here = total - first < kMostThreads ? total - first : kMostThreads;
        hipLaunchKernelGGL(mx_pack_kernel, dim3((uint32_t)(here ? (here + 255) / 256 : 1)), dim3(256), 0, (hipStream_t)stream,
                           (uint8_t const *)codes, codes_stride, codes_matrix, (uint8_t const *)scales, scales_stride,
                           scales_matrix, header, (uint32_t)steps, (uint32_t)supers, (uint32_t)tiles, first, code_lanes, scale_lanes,
                           wide, (uint8_t *)packed);
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, "mx_pack_kernel");
    }
    return 0;
}

nk_size_t nk_amd_mx_dots_workspace_size(nk_size_t height, nk_size_t width, nk_size_t depth, int a_is_codes) {
    MxGeometry g;
    if (!height || !width || height >= (1ull << 31) || !mx_geometry(1, width, depth, g)) return 0;
    return !a_is_codes && fuses(height, g) ? 0 : staging_of(height, g).bytes;
}

int nk_amd_mx_dots_packed_async(nk_dtype_t a_dtype, void const *a, nk_size_t a_stride, void const *a_scales,
                                nk_size_t a_scales_stride, void const *packed, nk_dtype_t c_dtype, void *c, nk_size_t c_stride,
                                nk_size_t height, nk_size_t width, nk_size_t depth, void *workspace, nk_size_t workspace_bytes,
                                void *stream_) {
    MxGeometry g;
    hipStream_t const stream = (hipStream_t)stream_;
    if (height >= (1ull << 31) || !mx_geometry(1, width, depth, g)) return mx_fail("mx_dots_packed: unsupported dimensions");
    if (!height || !width) return 0;
    if (int const status = depth ? check_a(a_dtype, a, a_scales, a_stride) : 0) return status;
    if (int const status = check_c(c_dtype, c, c_stride)) return status;
    if (!packed || ((uintptr_t)packed & 15)) return mx_fail("mx_dots_packed: the image has to be 16-byte aligned");
    bool const fused = !a_scales && fuses(height, g);
    MxArgs p = {};
    p.image = (uint8_t const *)packed, p.c = (uint8_t *)c, p.c_stride = c_stride;
    p.m = (uint32_t)height, p.n = (uint32_t)width, p.k = (uint32_t)depth, p.count = 1, p.a_share = 1;
    p.steps = g.steps, p.supers = g.supers, p.tiles = g.tiles, p.c_wide = aligned(c, c_stride, 16);
    if (fused) p.a = (uint8_t const *)a, p.a_pitch = a_stride, p.a_wide = aligned(a, a_stride, 16);
    else {
        Staging const s = staging_of(height, g);
        if (s.bytes && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < s.bytes))
            return mx_fail("mx_dots_packed: the workspace is too small or not 256-byte aligned");
        if (int const status = stage(a_dtype, a, a_stride, a_scales, a_scales_stride, height, p.k, g, s, (uint8_t *)workspace, stream))
            return status;
        p.a = (uint8_t const *)workspace, p.a_scales = p.a + s.scales_at, p.a_pitch = s.pitch, p.scales_pitch = s.scales_pitch;
    }
    return with_type(c_dtype, [&](auto value) {
        uint32_t const rows = height > 256 ? 256 : (uint32_t)height;
        return launch_product<decltype(value), false>(p, rows, a_dtype, fused, rows, g, stream);
    });
}

nk_size_t nk_amd_mx_experts_workspace_size(nk_size_t slots, nk_size_t a_share, nk_size_t experts, nk_size_t width,
                                           nk_size_t depth, int a_is_codes, nk_dtype_t c_dtype, int weighted) {
    MxGeometry g;
    if (!slots || !a_share || slots >= (1ull << 30) || !mx_geometry(experts, width, depth, g)) return 0;
    return experts_layout(slots, a_share, experts, width, g, a_is_codes != 0, c_dtype, weighted != 0).bytes;
}

int nk_amd_mx_dots_experts_async(nk_dtype_t a_dtype, void const *a, nk_size_t a_stride, void const *a_scales,
                                 nk_size_t a_scales_stride, nk_size_t a_share, void const *packed, void const *plan, nk_size_t slots,
                                 nk_size_t experts, nk_size_t top_k, float const *weights, nk_dtype_t c_dtype, void *c,
                                 nk_size_t c_stride, nk_size_t width, nk_size_t depth, void *workspace, nk_size_t workspace_bytes,
                                 void *stream_) {
    MxGeometry g;
    PlanGeometry shape;
    hipStream_t const stream = (hipStream_t)stream_;
    if (!mx_geometry(experts, width, depth, g) || !plan_geometry(slots, experts, shape)) return mx_fail("mx_dots_experts: unsupported dimensions");
    if (!a_share || !top_k || slots % top_k || slots % a_share) return mx_fail("mx_dots_experts: slots have to be whole rows of top_k and of a_share");
    if (!slots || !width) return 0;
    if (int const status = depth ? check_a(a_dtype, a, a_scales, a_stride) : 0) return status;
    if (int const status = check_c(c_dtype, c, c_stride)) return status;
    if (!packed || ((uintptr_t)packed & 15) || !plan || ((uintptr_t)plan & 15)) return mx_fail("mx_dots_experts: image and plan have to be 16-byte aligned");
    ExpertsLayout const l = experts_layout(slots, a_share, experts, width, g, a_scales != nullptr, c_dtype, weights != nullptr);
    if (l.bytes && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < l.bytes))
        return mx_fail("mx_dots_experts: the workspace is too small or not 256-byte aligned");
    MxArgs p = {};
    p.image = (uint8_t const *)packed, p.plan = (uint32_t const *)plan;
    p.m = (uint32_t)slots, p.n = (uint32_t)width, p.k = (uint32_t)depth, p.count = (uint32_t)experts, p.a_share = (uint32_t)a_share;
    p.steps = g.steps, p.supers = g.supers, p.tiles = g.tiles;
    p.tiles_m = shape.max_tiles, p.order = (uint32_t)shape.order, p.tile_list = (uint32_t)shape.tiles;
    if (l.fused) p.a = (uint8_t const *)a, p.a_pitch = a_stride, p.a_wide = aligned(a, a_stride, 16);
    else {
        if (int const status = stage(a_dtype, a, a_stride, a_scales, a_scales_stride, slots / a_share, p.k, g, l.staged, (uint8_t *)workspace, stream))
            return status;
        p.a = (uint8_t const *)workspace, p.a_scales = p.a + l.staged.scales_at, p.a_pitch = l.staged.pitch, p.scales_pitch = l.staged.scales_pitch;
    }
    uint8_t *sums = (uint8_t *)workspace + l.sums_at;
    int const product_dtype = weights ? l.sums_dtype : (int)c_dtype;
    if (weights) p.sorted = 1, p.c = sums, p.c_stride = l.sums_values * element_bytes(l.sums_dtype), p.c_wide = 1;
    else p.c = (uint8_t *)c, p.c_stride = c_stride, p.c_wide = aligned(c, c_stride, 16);
    int const status = with_type(product_dtype, [&](auto value) {
        return launch_product<decltype(value), true>(p, shape.tile_rows, a_dtype, l.fused, 16, g, stream);
    });
    if (status || !weights) return status;
    uint64_t const tokens = slots / top_k, pieces = (width + 3) / 4;
    uint64_t const slab = kMostThreads / pieces; // tokens of one launch
    for (uint64_t first = 0; first < tokens; first += slab) {
        uint64_t const here = tokens - first < slab ? tokens - first : slab;
        uint32_t const place = (uint32_t)(shape.place + first * top_k);
        auto const combine = [&](auto in, auto out) {
            typedef decltype(in) In;
            typedef decltype(out) Out;
            hipLaunchKernelGGL((combine_kernel<In, Out>), dim3((uint32_t)((here * pieces + 255) / 256)), dim3(256), 0, stream,
                               (In const *)sums, l.sums_values, p.plan, place, weights + first * top_k, (uint32_t)top_k, (uint32_t)here,
                               p.n, (uint32_t)pieces, (Out *)((uint8_t *)c + first * c_stride), (uint64_t)c_stride, aligned(c, c_stride, 16));
            hipError_t const e = hipGetLastError();
            return e == hipSuccess ? 0 : mx_fail(e, "combine_kernel");
        };
        int const done = c_dtype == nk_bf16_k ? combine(__bf16(), __bf16()) : c_dtype == nk_f32_k ? combine(float(), float()) : combine(float(), _Float16());
        if (done) return done;
    }
    return 0;
}

} // extern "C"
