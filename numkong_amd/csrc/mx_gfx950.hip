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

/** A wavefront of the two kernels below takes so many stretches of 512 adjacent values of a row: 2 KiB on their way. */
template <class T>
constexpr uint32_t kStretches = sizeof(T) == 4 ? 1 : 2;

/**
 *  16 bytes of x a load, side by side over the wavefront, past the caches (x is read once); codes leave a word a lane. A lane's
 *  load of f32 is half a word of codes, so the two halves of a stretch are exchanged between neighbours. What bounds it is
 *  memory: 8192 x 8192 of f32, 268 MB in and 36 MB out, take 49 us. (Eight values a lane, loads of 32 bytes apart: 52 us in a
 *  kernel that does no more; such halves, through the caches: 52 us; past them: 47 us.)
 */
template <class T>
__global__ __launch_bounds__(256) void quantize_kernel(T const *x, uint64_t x_stride, uint32_t rows, uint32_t k, uint32_t stretches,
                                                       uint8_t *codes, uint64_t codes_stride,
                                                       uint8_t *scales, uint64_t scales_stride) {
    constexpr int N = kEach<T>, kHalves = 8 / N;
    uint32_t const lane = threadIdx.x & 63, first = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kStretches<T>;
    uint32_t row[kStretches<T>], from[kStretches<T>];
    v4u raw[kStretches<T>][kHalves];
#pragma unroll
    for (uint32_t t = 0; t < kStretches<T>; ++t) {
        row[t] = (first + t) / stretches, from[t] = (first + t - row[t] * stretches) * 512;
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
            uint32_t const col = from[t] + half * 256 + lane * N;
            raw[t][half] = v4u {0, 0, 0, 0};
            if (row[t] < rows && col + N <= k)
                raw[t][half] = __builtin_nontemporal_load((v4u_anywhere const *)((T const *)((uint8_t const *)x + row[t] * x_stride) + col));
        }
    }
#pragma unroll
    for (uint32_t t = 0; t < kStretches<T>; ++t) {
        if (row[t] >= rows) return;
        uint32_t word[kHalves], scale[kHalves];
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
            uint32_t const col = from[t] + half * 256 + lane * N;
            float v[N];
            if (col + N <= k) widen<T>(raw[t][half], v);
            else load_some((T const *)((uint8_t const *)x + row[t] * x_stride), col, k, v);
            word[half] = quantize_some(v, scale[half]);
        }
        uint32_t its_word = word[0], its_scale = scale[0], at = lane, block = lane >> 2;
        bool has_scale = !(lane & 3);
        if constexpr (kHalves == 2) { // an even lane takes its neighbour's of the first half, an odd one of the second
            uint32_t const low = (uint32_t)__builtin_amdgcn_mov_dpp((int)word[0], 0xB1, 0xF, 0xF, true);
            uint32_t const high = (uint32_t)__builtin_amdgcn_mov_dpp((int)word[1], 0xB1, 0xF, 0xF, true);
            bool const odd = lane & 1;
            its_word = odd ? high | word[1] << 16 : word[0] | low << 16, its_scale = odd ? scale[1] : scale[0];
            at = (lane >> 1) + odd * 32, block = (lane >> 3) + odd * 8, has_scale = (lane & 7) < 2;
        }
        uint32_t const col = from[t] + at * 8, bytes = col >= k ? 0 : (k - col + 1) / 2;
        uint8_t *to = codes + row[t] * codes_stride + col / 2;
        if (bytes >= 4) *(u32_anywhere *)to = its_word;
        else
            for (uint32_t i = 0; i < (bytes < 4 ? bytes : 4); ++i) to[i] = (uint8_t)(its_word >> 8 * i);
        if (has_scale && from[t] + block * 32 < k) scales[row[t] * scales_stride + from[t] / 32 + block] = (uint8_t)its_scale;
    }
}

/** A block's 16 bytes of a row's codes; zeros from column k on. */
__device__ __forceinline__ v4u load_codes(uint8_t const *row, uint32_t block, uint32_t k) {
    v4u word = {0, 0, 0, 0};
    if (block * 32 + 32 <= k) return *(v4u_anywhere const *)(row + block * 16);
    for (uint32_t i = 0; i < 16; ++i) {
        uint32_t const col = block * 32 + 2 * i;
        uint32_t const byte = col + 1 < k ? row[col / 2] : col < k ? row[col / 2] & 15u : 0u;
        word[i / 4] |= byte << 8 * (i % 4);
    }
    return word;
}

struct StageArgs {
    void const *a;
    uint64_t a_stride;
    uint8_t const *scales; // A as codes: its scales
    uint64_t scales_stride;
    uint8_t *to, *to_scales;
    uint32_t const *plan; // rows in the plan's order, or NULL
    uint32_t rows, k, supers, order, a_share;
    uint32_t slots, experts; // that the plan is for
    uint32_t first;          // workgroups of the launches before
};
/** Is what is at `plan` a plan for so many slots and experts? (One of others has its parts elsewhere, and may end sooner.) */
__device__ __forceinline__ bool plan_matches(void const *plan, uint32_t slots, uint32_t experts) {
    PlanHeader const &h = *(PlanHeader const *)plan;
    return h.magic == kPlanMagic && h.slots == slots && h.experts == experts;
}
/** The row of A that row `row` of the fragments is; false where there is none. */
__device__ __forceinline__ bool source_of(StageArgs const &p, uint32_t row, uint64_t &source) {
    source = row;
    if (!p.plan) return row < p.rows;
    uint32_t const slot = p.plan[p.order + row];
    source = slot / p.a_share;
    return (int32_t)slot >= 0;
}

/**
 *  A into fragments: a workgroup for 16 rows of a super, a wavefront for a step of it. Four lanes share a block, 16 lanes read
 *  the 128 values of a row side by side, four rows at a time, and the codes change places in LDS, so that the fragment is
 *  written in one piece as well. (A lane with a block to itself reads 64-byte pieces 16 bytes at a time: 8192 x 8192 bf16 took
 *  46 us so, and takes 32 to 37 us: 170 MB.)
 */
template <class In>
__global__ __launch_bounds__(256) void stage_kernel(StageArgs p) {
    __shared__ __attribute__((aligned(16))) uint32_t words[4][256];
    __shared__ __attribute__((aligned(4))) uint8_t bytes[256];
    constexpr int kLoads = sizeof(In) / 2; // 16-byte loads of a lane's eight values
    uint32_t const index = p.first + blockIdx.x, tile = index / p.supers, super = index - tile * p.supers;
    uint32_t const lane = threadIdx.x & 63, u = threadIdx.x >> 6, piece = lane & 15, g = piece >> 2;
    uint32_t const block = (super * 4 + u) * 4 + g, col = block * 32 + (piece & 3) * 8;
    if (p.plan && (!plan_matches(p.plan, p.slots, p.experts) || tile * 16 >= ((PlanHeader const *)p.plan)->first_zero)) return;
    bool const whole = col + 8 <= p.k;
    In const *from[4];
    bool there[4];
    v4u raw[4][kLoads];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        uint64_t source;
        there[t] = source_of(p, tile * 16 + t * 4 + (lane >> 4), source) && col < p.k;
        from[t] = (In const *)((uint8_t const *)p.a + source * p.a_stride);
    }
    if (whole)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) raw[t][i] = ((v4u_anywhere const *)((there[t] ? from[t] : (In const *)p.a) + col))[i];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (there[t])
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                float part[kEach<In>];
                if (whole) widen<In>(raw[t][i], part);
                else load_some(from[t], col + i * kEach<In>, p.k, part);
#pragma unroll
                for (int j = 0; j < kEach<In>; ++j) v[i * kEach<In> + j] = part[j];
            }
        uint32_t scale;
        uint32_t const r = t * 4 + (lane >> 4), codes = quantize_some(v, scale);
        words[u][(g * 16 + r) * 4 + (piece & 3)] = codes;
        if (!(piece & 3)) bytes[scale_word(r, g) * 4 + u] = (uint8_t)scale;
    }
    __syncthreads();
    *(v4u *)(p.to + (((uint64_t)tile * p.supers + super) * 4 + u) * 1024 + lane * 16) = *(v4u const *)(words[u] + lane * 4);
    if (threadIdx.x < 64) *(uint32_t *)(p.to_scales + ((uint64_t)tile * p.supers + super) * 256 + lane * 4) = *(uint32_t const *)(bytes + lane * 4);
}

/** The same from codes: a lane's 16 bytes of a row are its 16 bytes of the fragment. */
__global__ __launch_bounds__(256) void stage_codes_kernel(StageArgs p) {
    __shared__ __attribute__((aligned(4))) uint8_t bytes[256];
    uint32_t const index = p.first + blockIdx.x, tile = index / p.supers, super = index - tile * p.supers;
    uint32_t const lane = threadIdx.x & 63, u = threadIdx.x >> 6, r = lane & 15, g = lane >> 4, block = (super * 4 + u) * 4 + g;
    if (p.plan && (!plan_matches(p.plan, p.slots, p.experts) || tile * 16 >= ((PlanHeader const *)p.plan)->first_zero)) return;
    uint64_t source;
    v4u codes = {0, 0, 0, 0};
    uint32_t scale = 0;
    if (source_of(p, tile * 16 + r, source) && block * 32 < p.k)
        codes = load_codes((uint8_t const *)p.a + source * p.a_stride, block, p.k), scale = p.scales[source * p.scales_stride + block];
    *(v4u *)(p.to + (((uint64_t)tile * p.supers + super) * 4 + u) * 1024 + lane * 16) = codes;
    bytes[scale_word(r, g) * 4 + u] = (uint8_t)scale;
    __syncthreads();
    if (threadIdx.x < 64) *(uint32_t *)(p.to_scales + ((uint64_t)tile * p.supers + super) * 256 + lane * 4) = *(uint32_t const *)(bytes + lane * 4);
}

/**
 *  value = q * 2^(s - 127). A word of codes a lane; of f32 its eight values are two stores' worth, and lanes fetch each other's
 *  words so that every store is side by side over the wavefront. `past`: x is larger than what the caches would keep of it, and is
 *  written past them (8192 x 8192 of f32: 43 us; 56 us through the caches in a kernel that does no more, 43 us past them).
 */
template <class T>
__global__ __launch_bounds__(256) void dequantize_kernel(uint8_t const *codes, uint64_t codes_stride,
                                                         uint8_t const *scales, uint64_t scales_stride, uint32_t rows, uint32_t k,
                                                         uint32_t stretches, T *x, uint64_t x_stride, bool past) {
    constexpr int N = kEach<T>, kHalves = 8 / N;
    uint32_t const lane = threadIdx.x & 63, first = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kStretches<T>;
    uint32_t row[kStretches<T>], from[kStretches<T>], word[kStretches<T>], scale[kStretches<T>];
#pragma unroll
    for (uint32_t t = 0; t < kStretches<T>; ++t) {
        row[t] = (first + t) / stretches, from[t] = (first + t - row[t] * stretches) * 512, word[t] = 0, scale[t] = 0;
        uint32_t const col = from[t] + lane * 8;
        if (row[t] >= rows || col >= k) continue;
        uint8_t const *its = codes + row[t] * codes_stride + col / 2;
        if (col + 8 <= k) word[t] = *(u32_anywhere const *)its;
        else
            for (uint32_t i = 0; i < 4; ++i)
                if (col + 2 * i < k) word[t] |= (uint32_t)its[i] << 8 * i;
        scale[t] = scales[row[t] * scales_stride + col / 32];
    }
#pragma unroll
    for (uint32_t t = 0; t < kStretches<T>; ++t) {
        if (row[t] >= rows) return;
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
            uint32_t its_word = word[t], its_scale = scale[t];
            if constexpr (kHalves == 2) {
                int const source = half * 32 + (int)(lane >> 1);
                its_word = (uint32_t)__shfl((int)word[t], source) >> 16 * (lane & 1), its_scale = (uint32_t)__shfl((int)scale[t], source);
            }
            float const power = __uint_as_float(its_scale ? its_scale << 23 : 0x00400000u);
            float v[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                uint32_t const code = its_word >> 4 * i & 15u, twice = (0xC8643210u >> 4 * (code & 7u)) & 15u; // 0 1 2 3 4 6 8 12
                float const magnitude = its_scale == 255 ? __uint_as_float(0x7FC00000u) : 0.5f * (float)twice * power;
                v[i] = code & 8u ? -magnitude : magnitude;
            }
            uint32_t const col = from[t] + half * 256 + lane * N;
            if (col >= k) continue;
            T *to = (T *)((uint8_t *)x + row[t] * x_stride) + col;
            if (past && col + N <= k) {
                struct alignas(16) Piece {
                    T x[N];
                } piece;
#pragma unroll
                for (int i = 0; i < N; ++i) piece.x[i] = (T)v[i];
                __builtin_nontemporal_store(__builtin_bit_cast(v4u, piece), (v4u *)to);
            }
            else store_some<T, N>(to, v, k - col);
        }
    }
}

// ---- packing ------------------------------------------------------------------------------------------------------

/** One thread for 16 bytes of a tile's codes or for a word of its scales; the header by the first workgroup. Memory bounds it
 *  (8192 x 8192: 14.8 us, 4.8 TB/s read and written; 32 matrices of 2050 x 1000, whose rows end inside a block that is fetched by
 *  bytes: 17.4 us, 4.1 TB/s), and it runs once for a matrix. */
__global__ __launch_bounds__(256) void mx_pack_kernel(uint8_t const *codes, uint64_t codes_stride, uint64_t codes_matrix,
                                                      uint8_t const *scales, uint64_t scales_stride, uint64_t scales_matrix,
                                                      MxHeader header, uint32_t supers, uint32_t tiles, uint64_t first,
                                                      uint64_t code_lanes, uint64_t scale_lanes, uint8_t *image) {
    uint64_t const index = first + (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (index == 0) *(MxHeader *)image = header;
    uint32_t const lane = index & 63;
    bool const of_codes = index < code_lanes;
    uint64_t const at = (of_codes ? index : index - code_lanes) >> 6;
    if (!of_codes && at >= scale_lanes / 64) return;
    uint32_t const across = of_codes ? supers * 4 : supers, which = (uint32_t)(at % across); // step or super
    uint64_t const tile_of_all = at / across;
    uint32_t const tile = (uint32_t)(tile_of_all % tiles);
    uint64_t const matrix = tile_of_all / tiles;
    uint32_t const q = of_codes ? lane & 15 : lane >> 2, g = of_codes ? lane >> 4 : (lane & 1) * 2 + (lane >> 1 & 1); // (scale_word)
    uint32_t const column = (tile >> 2) * 64 + (q >> 2) * 16 + (tile & 3) * 4 + (q & 3);
    uint32_t const k = header.k;
    if (of_codes) {
        uint32_t const block = which * 4 + g;
        v4u word = {0, 0, 0, 0};
        if (column < header.n && block * 32 < k) word = load_codes(codes + matrix * codes_matrix + column * codes_stride, block, k);
        *(v4u *)(image + kMxHeaderBytes + index * 16) = word;
        return;
    }
    uint32_t word = 0;
    for (uint32_t u = 0; u < 4; ++u) {
        uint32_t const block = which * 16 + u * 4 + g;
        if (column < header.n && block * 32 < k)
            word |= (uint32_t)scales[matrix * scales_matrix + column * scales_stride + block] << 8 * u;
    }
    *(uint32_t *)(image + kMxHeaderBytes + code_lanes * 16 + (index - code_lanes) * 4) = word;
}

// ---- products -----------------------------------------------------------------------------------------------------

struct MxArgs {
    uint8_t const *a; // staged codes, or the caller's floats (products of few rows that quantise them themselves)
    uint8_t const *a_scales;
    uint8_t const *image;
    uint8_t *c;
    uint32_t const *plan; // NULL: one matrix, rows in order
    uint64_t a_pitch, c_stride;
    uint32_t m, n, k, steps, supers, tiles, count;
    uint32_t tiles_m, tiles_n; // the grid: tiles of rows, tiles of columns
    uint32_t band;             // tiles of rows that are walked side by side
    uint32_t order, tile_list; // words into the plan
    uint32_t a_share;          // slots that share a row of A
    uint32_t sorted;           // 1: results in the plan's order of rows (and nothing for rows of no expert), 0: at their slots
};

/** The rows of one tile. */
struct RowTile {
    uint32_t matrix, first, last; // rows [first, last): of C, or of the plan
};
__device__ __forceinline__ RowTile row_tile_of(MxArgs const &p, uint32_t tile, uint32_t rows) {
    if (!p.plan) {
        uint32_t const first = tile * rows;
        return {0, first, first + rows < p.m ? first + rows : p.m};
    }
    PlanTile const entry = *(PlanTile const *)(p.plan + p.tile_list + tile * 4);
    return {(uint32_t)entry.expert, (uint32_t)entry.first, (uint32_t)entry.last};
}
__device__ __forceinline__ bool image_matches(MxArgs const &p) {
    MxHeader const h = *(MxHeader const *)p.image;
    return h.magic == kMxMagic && h.version == 1 && h.count == p.count && h.n == p.n && h.k == p.k;
}

/**
 *  The product for many rows: four wavefronts side by side, each 32 FM rows x 64 columns in blocks of 32 x 32 by
 *  v_mfma_scale_f32_32x32x64_f8f6f4 (in blocks of 16 x 16 the accumulators are four times as many values of the compiler's,
 *  and at 256 registers of them it moved these about, 632 moves for 256 products). A block's operand of half a step is
 *  lane l = row l % 32, block l / 32: sixteen rows' worth from each of two fragments, 256 bytes at a time.
 *
 *  A goes straight into LDS (a ring of four steps, fetched three ahead) in the order in which it is read, so that no read
 *  meets another's bank; each wavefront reads all of it, kAhead operands ahead of the products. B comes from the image straight
 *  into registers, each column of it into one wavefront's, the halves of a step refilled kSets steps ahead as they fall free.
 *  Fetches are counted, not drained: shortly before a step reads the first of the next step's A, the fetches of two steps ago
 *  have arrived, and everybody says so. Scales come a super ahead.
 *
 *  Workgroups stay: one walks its tiles, and the fetches of the next tile's first steps go out under the last steps of the one
 *  before, so that a tile starts at once. Each of the eight dies gets one stretch of the walk, in bands of some tiles of rows: low
 *  bands write whole rows at a time, which memory takes faster (stores alone, 268 MB of f32: bands of 256 rows 45 us, 512 52, 1,024
 *  60, 2,048 64), high ones read less of B (us, bands of 1, 2, 4 and 8: tiles of 128 rows, bf16 8192 x 8192 x 1024 68, 57, 63, 60, x 4096
 *  190, 150, 145, 147, f32 8192 x 6656 x 2048 103, 88, 91, 92; tiles of 256, 8192^3 bf16 270, 262, 262, 274, f32 284, 275, 295, 300).
 *
 *  8192^3 with bf16 results takes 260 to 265 us (4.2 PFLOP/s; on other days from 246; the matrix instructions alone, on such codes, 6.5):
 *  power holds the clock at 1.6 GHz, a step takes 1226 cycles of which 1024 are matrix instructions, a tile's end a tenth of its
 *  time. (Among the others are moves of scalar registers, of which the bases of two tiles and the choices between them take more than
 *  there are: the compiler keeps 55 to 98 of them in lanes of vector registers.) Shallow products of f32 results are bound by their stores
 *  (8192 x 8191 x 1000: 74 to 79 us for 268 MB), experts by both (64 of 512 rows on average, 2048 x 2048: 99 to 107 us for 313 MB).
 */
template <int FM, class Out, bool GROUPED>
__global__ __launch_bounds__(256, FM >= 8 ? 1 : 2) void mx_gemm_kernel(MxArgs p) {
    constexpr int FN = 2, kA = 2 * FM, kFetches = kA / 4, kScales = FM + FN, kAhead = 4, kSets = FM >= 8 ? 4 : 2, kMeet = 2 * FM - kAhead;
    static_assert(kA % 4 == 0 && kA % kAhead == 0, "whole fetches; operands of A keep their registers from step to step");
    static_assert(kMeet > kFetches && kMeet >= FM, "before a step's meeting: its fetches of A, its scales, B's first half");
    constexpr int kRows = FM * 32, kColumns = 256;
    constexpr int kPieces = 64 * (int)sizeof(Out) / 16, kEach = 16 / (int)sizeof(Out); // 16-byte pieces of a wavefront's row of C
    __shared__ __attribute__((aligned(1024))) uint8_t ring0[kA * 1024];
    __shared__ __attribute__((aligned(1024))) uint8_t ring1[kA * 1024];
    __shared__ __attribute__((aligned(1024))) uint8_t ring2[kA * 1024];
    __shared__ __attribute__((aligned(1024))) uint8_t ring3[kA * 1024];
    __shared__ __attribute__((aligned(1024))) uint8_t results[4][32 * kPieces * 16];

    uint32_t const lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
    uint32_t const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (GROUPED && !plan_matches(p.plan, p.m, p.count)) { // NaNs (sums by weight become that where they are made)
        for (uint32_t slot = blockIdx.x; !p.sorted && slot < p.m; slot += gridDim.x)
            for (uint32_t column = threadIdx.x; column < p.n; column += 256) ((Out *)(p.c + slot * p.c_stride))[column] = (Out)__uint_as_float(0x7FC00000u);
        return;
    }
    if (GROUPED && !p.sorted) { // rows of no expert are zeros
        PlanHeader const &h = *(PlanHeader const *)p.plan;
        for (uint32_t at = h.first_zero + blockIdx.x; at < h.end_zero; at += gridDim.x) {
            Out *row = (Out *)(p.c + p.plan[p.order + at] * p.c_stride);
            for (uint32_t column = threadIdx.x; column < p.n; column += 256) row[column] = (Out)0.0f;
        }
    }
    uint32_t const tiles_m = GROUPED ? ((PlanHeader const *)p.plan)->tile_count : p.tiles_m;
    uint32_t const total = tiles_m * p.tiles_n, stretch = (total + 7) / 8, turns = gridDim.x / 8;
    bool const good = image_matches(p);

    struct Tile {
        RowTile rows;
        uint32_t tile_n;
        uint8_t const *a, *a_scales, *b, *b_scales;
    };
    uint64_t const row_bytes = (uint64_t)p.supers * 4096, scale_row_bytes = (uint64_t)p.supers * 256; // of 16 rows or columns
    auto tile_at = [&](uint32_t turn, Tile &t) __attribute__((always_inline)) -> bool {
        uint32_t const inside = turn * turns + (blockIdx.x >> 3), index = (blockIdx.x & 7) * stretch + inside;
        if (inside >= stretch || index >= total) return false;
        uint32_t tile_m;
        if (GROUPED) tile_m = index / p.tiles_n, t.tile_n = index - tile_m * p.tiles_n; // (an expert's tiles side by side)
        else {
            uint32_t const band = index / (p.band * p.tiles_n), first = band * p.band, at = index - band * p.band * p.tiles_n;
            uint32_t const high = tiles_m - first < p.band ? tiles_m - first : p.band;
            t.tile_n = at / high, tile_m = first + at - t.tile_n * high;
        }
        t.rows = row_tile_of(p, tile_m, kRows);
        // (staged A has room for the rows of a whole tile behind its last; results of such rows are not stored)
        t.a = p.a + t.rows.first / 16 * row_bytes, t.a_scales = p.a_scales + t.rows.first / 16 * scale_row_bytes;
        // this wavefront's group of columns, four tiles side by side in the image; a group past its end is its last
        uint32_t const group = t.tile_n * 4 + wave, first_tile = (group * 4 < p.tiles ? group : p.tiles / 4 - 1) * 4;
        uint64_t const of_all = (uint64_t)t.rows.matrix * p.tiles + first_tile;
        t.b = p.image + kMxHeaderBytes + of_all * row_bytes;
        t.b_scales = p.image + kMxHeaderBytes + (uint64_t)p.count * p.tiles * row_bytes + of_all * scale_row_bytes;
        return true;
    };
    Tile now, then;
    if (!good || !p.supers) { // no depth: zeros; an image of something else: NaNs
        Out const value = (Out)(good ? 0.0f : __uint_as_float(0x7FC00000u));
        for (uint32_t turn = 0; tile_at(turn, now); ++turn)
            for (uint32_t at = now.rows.first; at < now.rows.last; ++at) {
                uint32_t const row = GROUPED && !p.sorted ? p.plan[p.order + at] : at, column = now.tile_n * kColumns + threadIdx.x;
                if (column < p.n) ((Out *)(p.c + row * p.c_stride))[column] = value;
            }
        return;
    }
    if (!tile_at(0, now)) return;

    uint32_t const steps = p.supers * 4, lane16 = lane * 16;
    // where a lane's 16 bytes of the first half of a step are: in LDS, in the image; and its two words of scales
    uint32_t const a_lane = (r >> 4) * 1024 + (g * 16 + (r & 15)) * 16;
    uint32_t const b_lane = (r >> 4) * (uint32_t)row_bytes + (g * 16 + (r & 15)) * 16;
    uint32_t const scale_lane = (r >> 4) * (uint32_t)scale_row_bytes + ((r & 15) * 4 + g * 2) * 4;

    v16f acc[FM][FN];
    v4u a[kAhead], b[kSets][2][FN]; // [step % kSets][half][block]
    v2u a_scale[FM], b_scale[FN], a_scale_next[FM], b_scale_next[FN]; // [half]
    auto fetch_a = [&](Tile const &t, uint32_t step, uint8_t *ring, int i) __attribute__((always_inline)) {
        uint32_t const f = wave * kFetches + i;
        fetch_16(buffer_of(t.a), ring + f * 1024, lane16, f * (uint32_t)row_bytes + step * 1024);
    };
    auto read_a = [&](uint8_t const *ring, int half, int i) __attribute__((always_inline)) -> v4u {
        return *(v4u const *)(ring + i * 2048 + half * 512 + a_lane);
    };
    auto load_b = [&](Tile const &t, uint32_t step, int half, int j) __attribute__((always_inline)) -> v4u {
        return load_16(buffer_of(t.b), b_lane, 2 * j * (uint32_t)row_bytes + step * 1024 + half * 512);
    };
    auto load_scale = [&](Tile const &t, uint32_t super, int i) __attribute__((always_inline)) { // FM of A's, then FN of B's
        if (i < FM) a_scale_next[i < FM ? i : 0] = load_8(buffer_of(t.a_scales), scale_lane, 2 * i * (uint32_t)scale_row_bytes + super * 256);
        else b_scale_next[i < FM ? 0 : i - FM] = load_8(buffer_of(t.b_scales), scale_lane, 2 * (i - FM) * (uint32_t)scale_row_bytes + super * 256);
    };
    // All but the last `younger` of this wavefront's fetches have arrived (< 0: they have anyway), what it has read from LDS as
    // well, and everybody says so.
    auto meet = [&](auto younger_) __attribute__((always_inline)) {
        constexpr int given = decltype(younger_)::value, younger = given < 0 ? 63 : given; // (63: no wait)
        static_assert(younger < 64, "what a wait can count to");
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | (younger & 15) | (younger >> 4) << 14);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // Step s, byte U of its super's scales. FRESH: of a tile's first super.
    auto step_of = [&](auto byte, auto fresh, uint32_t s, uint8_t const *here, uint8_t const *next, uint8_t *free) __attribute__((always_inline)) {
        constexpr int U = decltype(byte)::value, P = U % kSets;
        constexpr bool FRESH = decltype(fresh)::value != 0;
        bool const wrap_a = s + 3 >= steps, wrap_b = s + kSets >= steps, wrap_scales = s + 4 >= steps;
        uint32_t const step_a = wrap_a ? s + 3 - steps : s + 3, step_b = wrap_b ? s + kSets - steps : s + kSets;
        uint32_t const super = wrap_scales ? 0 : (s >> 2) + 1;
        if (U == 0) {
#pragma unroll
            for (int i = 0; i < FM; ++i) a_scale[i] = a_scale_next[i];
#pragma unroll
            for (int j = 0; j < FN; ++j) b_scale[j] = b_scale_next[j];
        }
#pragma unroll
        for (int at = 0; at < 2 * FM; ++at) {
            int const half = at / FM, i = at % FM, ahead = at + kAhead;
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = mx_multiply<U>(b[P][half][j], a[at % kAhead], FRESH && U == 0 && half == 0 ? v16f {} : acc[i][j], b_scale[j][half], a_scale[i][half]);
            // What went out behind the fetches of two steps ago: B's and scales of that step, all of the last, this one's so far.
            // (Fetches from before a tile's first step were waited for before the last tile's results were stored.)
            if (at == kMeet) meet(Number<FRESH && U < 2 ? -1 : 5 * FN + 2 * kFetches + (U < 3 ? kScales : 0)>());
            a[at % kAhead] = ahead < 2 * FM ? read_a(here, ahead / FM % 2, ahead % FM) : read_a(next, ahead % (2 * FM) / FM, ahead % FM);
            if (at < kFetches) fetch_a(wrap_a ? then : now, step_a, free, at < kFetches ? at : 0);
            if (U == 0 && at >= kFetches && at < kMeet)
#pragma unroll
                for (int k = (at - kFetches) * kScales / (kMeet - kFetches); k < (at - kFetches + 1) * kScales / (kMeet - kFetches); ++k)
                    load_scale(wrap_scales ? then : now, super, k);
            if (i == FM - 1)
#pragma unroll
                for (int j = 0; j < FN; ++j) b[P][half][j] = load_b(wrap_b ? then : now, step_b, half, j);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

#pragma unroll
    for (int i = 0; i < kScales; ++i) load_scale(now, 0, i);
#pragma unroll
    for (int t = 0; t < 3; ++t)
#pragma unroll
        for (int i = 0; i < kFetches; ++i) fetch_a(now, t, t == 0 ? ring0 : t == 1 ? ring1 : ring2, i);
#pragma unroll
    for (int t = 0; t < kSets; ++t)
#pragma unroll
        for (int j = 0; j < 2 * FN; ++j) b[t][j / FN][j % FN] = load_b(now, t, j / FN, j % FN);
    meet(Number<0>());
#pragma unroll
    for (int i = 0; i < kAhead; ++i) a[i] = read_a(ring0, i / FM, i % FM);
    for (uint32_t turn = 1;; ++turn) {
        bool const more = tile_at(turn, then);
        if (!more) then = now; // (its first steps are fetched once more and not used)
        uint32_t slots[(kRows + 63) / 64]; // where the rows of this tile go
        if (GROUPED && !p.sorted)
#pragma unroll
            for (int x = 0; x < (kRows + 63) / 64; ++x) {
                uint32_t const at = now.rows.first + x * 64 + lane;
                slots[x] = p.plan[p.order + (at < now.rows.last ? at : now.rows.last - 1)];
            }
        step_of(Number<0>(), Number<1>(), 0, ring0, ring1, ring3);
        step_of(Number<1>(), Number<1>(), 1, ring1, ring2, ring0);
        step_of(Number<2>(), Number<1>(), 2, ring2, ring3, ring1);
        step_of(Number<3>(), Number<1>(), 3, ring3, ring0, ring2);
        for (uint32_t s = 4; s < steps; s += 4) {
            step_of(Number<0>(), Number<0>(), s, ring0, ring1, ring3);
            step_of(Number<1>(), Number<0>(), s + 1, ring1, ring2, ring0);
            step_of(Number<2>(), Number<0>(), s + 2, ring2, ring3, ring1);
            step_of(Number<3>(), Number<0>(), s + 3, ring3, ring0, ring2);
        }

        // Rows of the image's columns in a block: 8 (t / 4) + 4 g + t % 4 of value t, which the image's order of columns makes
        // two runs of 16 adjacent columns (2 x + g of the four in a group, x = 0, 1), four values from each of the group's four
        // tiles. 32 rows at a time they go through the wavefront's own part of LDS (16-byte pieces, piece c of row r at
        // c ^ (r & 7)), so that a row is stored in one piece: 128 or 256 adjacent bytes, whatever address it starts at.
        // (Stores past the caches: 273 against 277 us for 8192^3, 116 against 85 where rows do not start on 128-byte lines; a choice
        // between the two in the kernel costs what it brings.)
        uint8_t *const mine = results[wave];
        uint32_t const wave_column = now.tile_n * kColumns + wave * 64;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            wave_fence();
#pragma unroll
            for (int part = 0; part < 2 * 16 / kEach; ++part) {
                int const x = part * kEach / 16;
                struct alignas(16) Piece {
                    Out v[kEach];
                } values;
#pragma unroll
                for (int t = 0; t < kEach; ++t) {
                    int const j = part * kEach % 16 + t;
                    values.v[t] = (Out)acc[i][j / 8][(j / 4) % 2 * 8 + x * 4 + j % 4];
                }
                uint32_t const piece = ((2 * x + g) * 16 + part * kEach % 16) / kEach;
                *(Piece *)(mine + (r * kPieces + (piece ^ (r & 7))) * 16) = values;
            }
            wave_fence();
            if (i == 0) { // (what the next tile's first steps need: from here on stores are behind it)
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_waitcnt(0x0F70);
                asm volatile("" ::: "memory");
            }
            auto const store_row = [&](int round, bool whole) __attribute__((always_inline)) {
                uint32_t const local = round * (64 / kPieces) + lane / kPieces, piece = lane % kPieces;
                v4u const values = *(v4u const *)(mine + (local * kPieces + (piece ^ (local & 7))) * 16);
                uint32_t const at = now.rows.first + i * 32 + local, column = wave_column + piece * kEach;
                uint32_t row = at;
                if (GROUPED && !p.sorted) row = (uint32_t)__shfl((int)slots[i / 2], i % 2 * 32 + local);
                if (at >= now.rows.last || (!whole && column >= p.n)) return;
                Out *to = (Out *)(p.c + row * p.c_stride) + column;
                if (whole || column + kEach <= p.n) store_16(to, values);
                else
                    for (uint32_t t = 0; t < p.n - column; ++t) { // (every element with its own word: no array of them)
                        uint32_t const word = t * sizeof(Out) / 4 == 0 ? values[0] : t * sizeof(Out) / 4 == 1 ? values[1] : t * sizeof(Out) / 4 == 2 ? values[2] : values[3];
                        if constexpr (sizeof(Out) == 4) ((uint32_t *)to)[t] = word;
                        else ((uint16_t *)to)[t] = (uint16_t)(word >> 16 * (t & 1));
                    }
            };
            if (wave_column + 64 <= p.n) {
#pragma unroll
                for (int round = 0; round < kPieces / 2; ++round) store_row(round, true);
            }
            else
#pragma unroll 1
                for (int round = 0; round < kPieces / 2; ++round) store_row(round, false);
        }
        if (!more) break;
        now = then;
    }
    __builtin_amdgcn_s_waitcnt(0x0F70); // (nothing is on its way into LDS when the workgroup ends)
}

/**
 *  The product for few rows: the stream of B is the work, so a workgroup takes 16 NT columns and its wavefronts the supers of
 *  the depth in turn, B straight into registers, and their sums meet in LDS. In: the type of A's values, which the workgroup
 *  quantises into LDS itself (one launch, and A is read by all lanes), or `uint8_t`: A is staged already, and goes into registers.
 *  B's first loads are on their way while A is quantised. 1 x 8192 against 8192 columns: 8.8 us, 4.1 TB/s of the image; 64 rows 12.1 us,
 *  as each of 256 workgroups reads all of A (278 KB, 71 MB out of the L2s beside 36 MB of image: 107 MB of requests were counted); 32 slots of 29
 *  experts, 2048 x 2048: 14.3 us, 4.5 TB/s.
 */
template <int WAVES, int FM, int NT, class In, class Out, bool GROUPED>
__global__ __launch_bounds__(64 * WAVES, FM >= 4 ? 2 : 4) void mx_few_kernel(MxArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
    constexpr bool FUSED = sizeof(In) != 1;
    uint32_t tile_m, tile_n;
    if (!GROUPED) { // the tiles of rows of the same columns on one die, one after the other: it reads them once
        uint32_t const index = blockIdx.x >> 3, column = index / p.tiles_m;
        tile_m = index - column * p.tiles_m, tile_n = column * 8 + (blockIdx.x & 7);
        if (tile_n >= p.tiles_n) return;
    }
    else {
        tile_m = blockIdx.x / p.tiles_n, tile_n = blockIdx.x - tile_m * p.tiles_n;
        if (!plan_matches(p.plan, p.m, p.count)) { // NaNs, as in mx_gemm_kernel
            uint32_t const column = tile_n * NT * 16 + threadIdx.x;
            if (!p.sorted && threadIdx.x < NT * 16 && column < p.n)
                for (uint32_t slot = tile_m; slot < p.m; slot += p.tiles_m) ((Out *)(p.c + slot * p.c_stride))[column] = (Out)__uint_as_float(0x7FC00000u);
            return;
        }
        PlanHeader const &h = *(PlanHeader const *)p.plan;
        if (tile_m >= h.tile_count + (p.sorted ? 0 : h.zero_tiles)) return;
    }
    RowTile const rows = row_tile_of(p, tile_m, FM * 16);
    uint32_t const lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    bool const good = image_matches(p), computes = good && !(GROUPED && rows.matrix >= p.count) && p.steps;
    uint32_t const here = rows.last - rows.first;
    uint32_t const row_bytes = p.supers * 4096, scale_row_bytes = p.supers * 256, lane16 = lane * 16, scale_lane = scale_word(r, g) * 4;
    v4f acc[FM][NT];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4f {0, 0, 0, 0};

    uint64_t const of_all = (uint64_t)rows.matrix * p.tiles + tile_n * NT;
    uint8_t const *const codes = p.image + kMxHeaderBytes;
    __amdgpu_buffer_rsrc_t const w_from = buffer_of(codes + of_all * row_bytes);
    __amdgpu_buffer_rsrc_t const w_scale_from = buffer_of(codes + (uint64_t)p.count * p.tiles * row_bytes + of_all * scale_row_bytes);
    v4u w[4][NT];
    uint32_t w_scale[NT];
    auto load_w = [&](uint32_t super) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            uint32_t const s = super * 4 + u < p.steps ? super * 4 + u : p.steps - 1; // (what pads the last super is not fetched)
#pragma unroll
            for (int j = 0; j < NT; ++j) w[u][j] = load_16(w_from, lane16, j * row_bytes + s * 1024);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) w_scale[j] = load_4(w_scale_from, scale_lane, j * scale_row_bytes + super * 256);
    };
    if (computes && wave < p.supers) load_w(wave);

    uint32_t const lds_pitch = p.steps * 64 + 16; // (16 bytes on: rows start in different banks)
    uint8_t *lds_scales = few_lds + here * lds_pitch;
    if constexpr (FUSED) {
        constexpr int N = kEach<In>, kLanes = 32 / N;
        uint32_t const pieces = p.steps * (128 / N);
        for (uint32_t index = threadIdx.x; computes && index < here * pieces; index += 64 * WAVES) {
            uint32_t const row = index / pieces, piece = index - row * pieces;
            uint32_t const at = rows.first + row, source = GROUPED ? p.plan[p.order + at] / p.a_share : at;
            In const *from = (In const *)(p.a + source * p.a_pitch);
            float v[N];
            if (piece * N + N <= p.k) widen<In>(*(v4u_anywhere const *)(from + piece * N), v);
            else load_some(from, piece * N, p.k, v);
            uint32_t scale;
            uint32_t const word = quantize_some(v, scale);
            if constexpr (N == 8) *(uint32_t *)(few_lds + row * lds_pitch + piece * 4) = word;
            else *(uint16_t *)(few_lds + row * lds_pitch + piece * 2) = (uint16_t)word;
            if (piece % kLanes == 0) lds_scales[row * (p.steps * 4) + piece / kLanes] = (uint8_t)scale;
        }
    }
    if (FUSED) __syncthreads();
    if (computes) {
        uint32_t const fragment = rows.first / 16;
        __amdgpu_buffer_rsrc_t const a_from = buffer_of(p.a + (uint64_t)fragment * row_bytes), a_scale_from = buffer_of(p.a_scales + (uint64_t)fragment * scale_row_bytes);
        for (uint32_t super = wave; super < p.supers; super += WAVES) {
            if (super != wave) load_w(super);
            v4u a[4][FM];
            uint32_t a_scale[FM];
            if constexpr (!FUSED) {
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < FM; ++i) a[u][i] = load_16(a_from, lane16, i * row_bytes + (super * 4 + u) * 1024);
#pragma unroll
                for (int i = 0; i < FM; ++i) a_scale[i] = load_4(a_scale_from, scale_lane, i * scale_row_bytes + super * 256);
            }
            auto step_of = [&](auto byte) __attribute__((always_inline)) {
                constexpr int U = decltype(byte)::value;
                uint32_t const s = super * 4 + U;
                if (s >= p.steps) return;
                if constexpr (FUSED) {
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        bool const there = i * 16 + r < here;
                        uint32_t const row = there ? i * 16 + r : 0;
                        v4u const codes_of_a = *(v4u const *)(few_lds + row * lds_pitch + s * 64 + g * 16);
                        uint32_t const scale_of_a = lds_scales[row * (p.steps * 4) + s * 4 + g];
                        a[U][i] = there ? codes_of_a : v4u {0, 0, 0, 0};
                        a_scale[i] = there ? scale_of_a << 8 * U : 0u;
                    }
                }
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = mx_multiply<U>(w[U][j], a[U][i], acc[i][j], w_scale[j], a_scale[i]);
            };
            step_of(Number<0>()), step_of(Number<1>()), step_of(Number<2>()), step_of(Number<3>());
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
    for (uint32_t index = threadIdx.x; index < FM * NT * 64; index += 64 * WAVES) {
        uint32_t const of_lane = index & 63, fragment = index >> 6, i = fragment / NT, j = fragment % NT;
        uint32_t const local = i * 16 + (of_lane & 15);
        if (local >= here) continue;
        v4f sum = sums[index];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sum += sums[w * FM * NT * 64 + index];
        uint32_t const at = rows.first + local, row = GROUPED && !p.sorted ? p.plan[p.order + at] : at;
        uint32_t const tile = tile_n * NT + j, column = (tile >> 2) * 64 + (of_lane >> 4) * 16 + (tile & 3) * 4;
        if (column >= p.n) continue;
        float v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = good ? sum[t] : poison;
        store_some<Out, 4>((Out *)(p.c + row * p.c_stride) + column, v, p.n - column);
    }
}

/** out[token] = sum over its slots of weight * row of the plan, slots without an expert left out; a thread for four columns, four
 *  rows under way at a time. Memory bounds it (1001 tokens, 4 of 2050 columns: 8.0 us, 5.1 TB/s). */
template <class Out>
__global__ __launch_bounds__(256) void combine_kernel(float const *rows, uint64_t row_values, uint32_t const *plan, uint32_t slots,
                                                      uint32_t experts, uint32_t place, float const *weights, uint32_t top_k,
                                                      uint32_t tokens, uint32_t n, uint32_t pieces, Out *c, uint64_t c_stride) {
    uint32_t const index = blockIdx.x * 256 + threadIdx.x;
    uint32_t const token = index / pieces, column = (index - token * pieces) * 4;
    if (token >= tokens) return;
    bool const good = plan_matches(plan, slots, experts);
    float const start = good ? 0.0f : __uint_as_float(0x7FC00000u);
    float sum[4] = {start, start, start, start};
    for (uint32_t first = 0; good && first < top_k; first += 4) {
        int32_t row[4];
        float weight[4];
        v4f values[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t const slot = token * top_k + (first + i < top_k ? first + i : 0);
            row[i] = first + i < top_k ? (int32_t)plan[place + slot] : -1, weight[i] = weights[slot];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) // (rows are padded to whole fours; row 0 is there, whatever it holds)
            values[i] = *(v4f const *)(rows + (uint64_t)(row[i] < 0 ? 0 : row[i]) * row_values + column);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) sum[t] = row[i] < 0 ? sum[t] : __builtin_fmaf(weight[i], values[i][t], sum[t]);
    }
    store_some<Out, 4>((Out *)((uint8_t *)c + token * c_stride) + column, sum, n - column);
}

// ---- host side ----------------------------------------------------------------------------------------------------

int element_bytes(int dtype) { return dtype == nk_f32_k ? 4 : dtype == nk_bf16_k || dtype == nk_f16_k ? 2 : 0; }
bool aligned(void const *ptr, uint64_t stride, uint64_t to) { return !(((uintptr_t)ptr | stride) & (to - 1)); }

/** Calls `f` with a value of the element type's C++ type. */
template <class F>
int with_type(int dtype, F &&f) {
    if (dtype == nk_f32_k) return f(float());
    if (dtype == nk_bf16_k) return f(__bf16());
    return f(_Float16());
}

/** Rows that follow one another without a gap, in whole blocks, are one row: nothing has to ask which row it is in. */
bool one_row(uint64_t rows, uint64_t k, uint64_t x_stride, int bytes, uint64_t codes_stride, uint64_t scales_stride) {
    return k % 32 == 0 && x_stride == k * bytes && codes_stride == k / 2 && scales_stride == k / 32 && rows * k < 1ull << 31;
}
/** Launches `f(rows before, rows, stretches of a row, workgroups)` for all rows, many at a time. */
template <class T, class F>
int by_stretches(uint64_t rows, uint64_t k, F &&f) {
    uint64_t const stretches = (k + 511) / 512, slab = kMostThreads / 64 / stretches; // rows of one launch (k < 2^31: 8 at the least)
    for (uint64_t first = 0; first < rows; first += slab) {
        uint64_t const here = rows - first < slab ? rows - first : slab;
        f(first, (uint32_t)here, (uint32_t)stretches, dim3((uint32_t)((here * stretches + 4 * kStretches<T> - 1) / (4 * kStretches<T>))));
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, "quantize_kernel or dequantize_kernel");
    }
    return 0;
}

int launch_quantize(int dtype, void const *x, uint64_t rows, uint64_t k, uint64_t x_stride, uint8_t *codes, uint64_t codes_stride,
                    uint8_t *scales, uint64_t scales_stride, hipStream_t stream) {
    if (one_row(rows, k, x_stride, element_bytes(dtype), codes_stride, scales_stride)) k *= rows, rows = 1;
    return with_type(dtype, [&](auto value) {
        typedef decltype(value) T;
        return by_stretches<T>(rows, k, [&](uint64_t first, uint32_t here, uint32_t stretches, dim3 grid) {
            hipLaunchKernelGGL((quantize_kernel<T>), grid, dim3(256), 0, stream, (T const *)((uint8_t const *)x + first * x_stride), x_stride,
                               here, (uint32_t)k, stretches, codes + first * codes_stride, codes_stride,
                               scales + first * scales_stride, scales_stride);
        });
    });
}

/** How A is laid out in the workspace: room for `rows` and, behind them, for what the last tile reads past its last row. */
struct Staging {
    uint64_t scales_at, bytes;
};
constexpr uint64_t kMostTileRows = 256;
Staging staging_of(uint64_t rows, MxGeometry const &g) {
    uint64_t const fragments = (rows + 15) / 16 + kMostTileRows / 16;
    Staging s;
    s.scales_at = fragments * g.supers * 4096;
    s.bytes = (s.scales_at + fragments * g.supers * 256 + 255) / 256 * 256;
    return s;
}
/** A into the workspace: rows in order, or the rows of a plan. */
int stage(int a_dtype, void const *a, uint64_t a_stride, void const *a_scales, uint64_t a_scales_stride, uint32_t rows, uint32_t k,
          MxGeometry const &g, Staging const &s, uint8_t *to, void const *plan, size_t order, uint32_t a_share, uint32_t slots, uint32_t experts, hipStream_t stream) {
    uint64_t const total = (uint64_t)((rows + 15) / 16) * g.supers;
    StageArgs p = {a, a_stride, (uint8_t const *)a_scales, a_scales_stride, to, to + s.scales_at, (uint32_t const *)plan, rows, k,
                   g.supers, (uint32_t)order, a_share, slots, experts, 0};
    for (uint64_t first = 0; first < total; first += kMostThreads / 256) {
        dim3 const grid((uint32_t)(total - first < kMostThreads / 256 ? total - first : kMostThreads / 256));
        p.first = (uint32_t)first;
        if (a_scales) hipLaunchKernelGGL(stage_codes_kernel, grid, dim3(256), 0, stream, p);
        else
            with_type(a_dtype, [&](auto value) {
                hipLaunchKernelGGL(stage_kernel<decltype(value)>, grid, dim3(256), 0, stream, p);
                return 0;
            });
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, "stage_kernel");
    }
    return 0;
}
/** Fragments of A and tiles of C are counted in 32 bits: looked at before anything is queued. `row_tiles`: of 128 rows, or of a plan. */
int check_size(uint64_t rows, uint64_t row_tiles, uint64_t n, MxGeometry const &g) {
    if ((rows + 15) / 16 * g.supers > 0x7FFFFFFFull) return mx_fail("mx product: A is too large");
    if (row_tiles * ((n + 255) / 256) > 0x7FFFFFFFull) return mx_fail("mx product: too many tiles");
    return 0;
}

/**
 *  Do products of few rows quantise A themselves? Every workgroup then does it for all columns that it has, and no launch goes
 *  before: 1 x 8192 against 8192 columns takes 9.1 us so, 8 x 8192 16.1 us, and 10.9 us where a launch stages A first; 4 x 4096 against 4096 columns 4.7 us so.
 *  `values`: of A, as many as a workgroup is expected to have; `rows`: the most that it may have, which have to fit.
 */
constexpr uint32_t kFusedBytes = 64 * 1024, kFusedValues = 16 * 1024;
/** Does a launch take all tiles of a product of few rows, at 512 threads for 16 columns of a tile of rows? Where it does not (2^27 columns, 2^15 of
 *  a thousand experts) the kernel for many rows has the work, whose workgroups stay, and A is staged for it. (The kernel for few rows in
 *  several launches, each told where its columns begin: 1 x 8192 x 8192 8.9 us instead of 8.6.) */
bool launches_few(uint64_t row_tiles, uint64_t n) { return row_tiles * ((n + 15) / 16 + 7) * 512 < 1ull << 32; }
uint32_t fused_bytes(uint32_t rows, MxGeometry const &g) { return rows * (g.steps * 64 + 16) + rows * g.steps * 4; }
bool fuses(uint64_t rows, uint64_t values, MxGeometry const &g) {
    return rows <= 16 && values <= kFusedValues && (uint64_t)rows * (g.steps * 68 + 16) <= kFusedBytes;
}

template <int WAVES, int FM, int NT, class In, class Out, bool GROUPED>
int launch_few_of(MxArgs &p, uint32_t max_rows, MxGeometry const &g, hipStream_t stream) {
    p.tiles_n = (p.tiles + NT - 1) / NT;
    if (!GROUPED) p.tiles_m = (p.m + 16 * FM - 1) / (16 * FM);
    uint32_t const grid = p.tiles_m * (GROUPED ? p.tiles_n : (p.tiles_n + 7) / 8 * 8); // (launches_few)
    uint32_t lds = WAVES * FM * NT * 1024;
    if (sizeof(In) != 1 && fused_bytes(max_rows, g) > lds) lds = fused_bytes(max_rows, g);
    hipLaunchKernelGGL((mx_few_kernel<WAVES, FM, NT, In, Out, GROUPED>), dim3(grid), dim3(64 * WAVES), lds, stream, p);
    hipError_t const e = hipGetLastError();
    return e == hipSuccess ? 0 : mx_fail(e, "mx_few_kernel");
}
template <int FM, int NT, class In, class Out, bool GROUPED>
int launch_few(MxArgs &p, uint32_t max_rows, MxGeometry const &g, hipStream_t stream) {
    return g.steps < 32 ? launch_few_of<4, FM, NT, In, Out, GROUPED>(p, max_rows, g, stream) : launch_few_of<8, FM, NT, In, Out, GROUPED>(p, max_rows, g, stream);
}
template <int FM, class Out, bool GROUPED>
int launch_gemm(MxArgs &p, hipStream_t stream) {
    p.tiles_n = (p.tiles + 15) / 16, p.band = FM >= 8 || p.steps <= 16 ? 2 : 4;
    if (!GROUPED) p.tiles_m = (p.m + 32 * FM - 1) / (32 * FM);
    uint64_t const tiles = (uint64_t)p.tiles_m * p.tiles_n, resident = (uint64_t)compute_unit_count() * (FM >= 8 ? 1 : 2);
    if (!resident) return mx_fail("mx product: no GPU");
    uint64_t const grid = ((tiles < resident ? tiles : resident) + 7) / 8 * 8;
    hipLaunchKernelGGL((mx_gemm_kernel<FM, Out, GROUPED>), dim3((uint32_t)grid), dim3(256), 0, stream, p);
    hipError_t const e = hipGetLastError();
    return e == hipSuccess ? 0 : mx_fail(e, "mx_gemm_kernel");
}

/**
 *  Which kernel. With experts, the rows of a tile decide (plan_tile_rows). Otherwise products of fewer than 64 tiles of 128 x 256
 *  are of few rows, in tiles of up to 64: those tiles would each take as long as it takes to walk the depth, with most of the
 *  compute units idle (us, few rows against many: 128 x 8192 x 8192 19.1 and 27.1, 512 x 2048 x 2048 10.6 and 12.5, 1024 x 1024 x
 *  8192 23.1 and 30.8; at 64 tiles 256 x 8192 x 8192 29.9 and 28.5, 1024 x 2048 x 2048 15.4 and 13.9). A workgroup of few rows
 *  takes one tile of columns while there are fewer than 512 (64 x 2048 x 2048 7.0 us with one, 7.5 with two; 64 x 8192 x 8192
 *  17.0 and 15.0). Among many rows tiles of 128, two workgroups to a compute unit, which hide
 *  each other's ends (a workgroup's results hold up its next tile: stores are waited for in order); of 256 only past a depth of
 *  6,144 and where they fill the compute units in whole rounds, as less of B is read then (us, 128 rows and 256: bf16 8192 x 8192,
 *  depth 512 41 and 54, 1,024 57 and 73, 4,096 146 and 151, 6,144 205 and 205, 8,192 265 and 263, 16384 x 8192 x 8192 543 and 522, f32
 *  8192^3 289 and 273; but 9000 x 9000 x 8192, 6 rounds of 256 rows for 5.06, 327 and 356, 6000 x 6000 x 8192, 3 for 2.25, 164 and 183).
 */
template <class Out, bool GROUPED>
int launch_product(MxArgs &p, bool few, uint32_t tile_rows, int a_dtype, bool fused, uint32_t fused_rows, MxGeometry const &g, hipStream_t stream) {
    auto const tiles_of = [&](uint64_t rows, uint64_t columns) { return (p.m + rows - 1) / rows * ((p.n + columns - 1) / columns); };
    auto const whole_rounds = [&] { // (within a twentieth)
        uint64_t const large = tiles_of(256, 256), units = (uint64_t)compute_unit_count();
        return units && large * 20 >= (large + units - 1) / units * units * 19;
    };
    bool const small = p.m <= 32 || tiles_of(128, 256) < 64;
    uint32_t const rows = GROUPED ? (few ? tile_rows : 128) : few && small ? (p.m < 64 ? p.m : 64) : g.steps > 48 && g.steps < kMxMaxDepth / 128 && whole_rounds() ? 256 : 128;
    if (rows <= 16) {
        constexpr int NT = GROUPED ? 2 : 1; // (experts of 4 tokens, 28 matrices of 2048 x 2048: 13.0 us with two, 14.0 with one)
        if (!fused) return launch_few<1, NT, uint8_t, Out, GROUPED>(p, rows, g, stream);
        return with_type(a_dtype, [&](auto value) { return launch_few<1, NT, decltype(value), Out, GROUPED>(p, fused_rows, g, stream); });
    }
    if (rows <= 64) {
        bool const narrow = p.tiles * (GROUPED ? (uint64_t)p.tiles_m : tiles_of(64, p.n)) < 512;
        if (rows <= 32) return narrow ? launch_few<2, 1, uint8_t, Out, GROUPED>(p, rows, g, stream) : launch_few<2, 2, uint8_t, Out, GROUPED>(p, rows, g, stream);
        return narrow ? launch_few<4, 1, uint8_t, Out, GROUPED>(p, rows, g, stream) : launch_few<4, 2, uint8_t, Out, GROUPED>(p, rows, g, stream);
    }
    if constexpr (!GROUPED)
        if (rows > 128) return launch_gemm<8, Out, GROUPED>(p, stream);
    return launch_gemm<4, Out, GROUPED>(p, stream);
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
    uint64_t codes_at, codes_stride, codes_scales_at, codes_scales_stride; // A's rows as codes, where they are quantised first
    uint64_t sums_at, sums_values, bytes; // rows of the plan before they are summed: values a row
    bool few, fused, quantised;
};
ExpertsLayout experts_layout(PlanGeometry const &shape, uint64_t slots, uint64_t a_share, uint64_t experts, uint64_t n, uint64_t k,
                             MxGeometry const &g, bool a_is_codes, bool weighted) {
    ExpertsLayout l = {};
    l.few = launches_few(shape.max_tiles, n);
    l.fused = l.few && !a_is_codes && shape.tile_rows == 16 && fuses(16, (slots / experts + 1) * k, g);
    if (!l.fused) l.staged = staging_of(shape.max_rows, g);
    uint64_t at = l.staged.bytes;
    // Rows that go to several experts are quantised once and gathered as codes, where that is worth a launch more (32,768 slots
    // of 4,096 rows of 2048: 26 us as floats, 19 us so).
    l.quantised = !l.fused && !a_is_codes && a_share > 1 && slots * k >= 1ull << 24;
    if (l.quantised) {
        l.codes_stride = (k / 2 + 15) / 16 * 16 + 16, l.codes_scales_stride = (k + 31) / 32;
        l.codes_at = at, l.codes_scales_at = at + (slots / a_share + 1) * l.codes_stride;
        at = (l.codes_scales_at + (slots / a_share + 1) * l.codes_scales_stride + 255) / 256 * 256;
    }
    l.sums_at = at;
    // (rows that are still to be summed by weight stand in 32 bits, whatever the result has: rounded to 16 they would err as much
    // again as the result's own rounding, and without bound against a sum that cancels)
    l.sums_values = (n + 15) / 16 * 16;
    l.bytes = l.sums_at + (weighted ? (shape.max_rows * l.sums_values * 4 + 255) / 256 * 256 : 0);
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
    return launch_quantize(dtype, x, rows, depth, x_stride, (uint8_t *)codes, codes_stride, (uint8_t *)scales,
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
    bool const past = rows * depth * bytes >= 64ull << 20 && aligned(x, x_stride, 16);
    if (one_row(rows, depth, x_stride, bytes, codes_stride, scales_stride)) depth *= rows, rows = 1;
    return with_type(dtype, [&](auto value) {
        typedef decltype(value) T;
        return by_stretches<T>(rows, depth, [&](uint64_t first, uint32_t here, uint32_t stretches, dim3 grid) {
            hipLaunchKernelGGL((dequantize_kernel<T>), grid, dim3(256), 0, (hipStream_t)stream, (uint8_t const *)codes + first * codes_stride,
                               codes_stride, (uint8_t const *)scales + first * scales_stride, scales_stride, here, (uint32_t)depth,
                               stretches, (T *)((uint8_t *)x + first * x_stride), x_stride, past);
        });
    });
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
    uint64_t const code_lanes = count * (g.code_bytes / 16), scale_lanes = count * (g.scale_bytes / 4);
    uint64_t const total = code_lanes + scale_lanes;
    uint64_t const supers = g.supers ? g.supers : 1, tiles = g.tiles ? g.tiles : 1;
    for (uint64_t first = 0; first == 0 || first < total; first += kMostThreads) {
        uint64_t const here = total - first < kMostThreads ? total - first : kMostThreads;
        hipLaunchKernelGGL(mx_pack_kernel, dim3((uint32_t)(here ? (here + 255) / 256 : 1)), dim3(256), 0, (hipStream_t)stream,
                           (uint8_t const *)codes, codes_stride, codes_matrix, (uint8_t const *)scales, scales_stride,
                           scales_matrix, header, (uint32_t)supers, (uint32_t)tiles, first, code_lanes, scale_lanes,
                           (uint8_t *)packed);
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, "mx_pack_kernel");
    }
    return 0;
}

nk_size_t nk_amd_mx_dots_workspace_size(nk_size_t height, nk_size_t width, nk_size_t depth, int a_is_codes) {
    MxGeometry g;
    if (!height || !width || height >= (1ull << 31) || !mx_geometry(1, width, depth, g)) return 0;
    return !a_is_codes && launches_few((height + 63) / 64, width) && fuses(height, height * depth, g) ? 0 : staging_of(height, g).bytes;
}

int nk_amd_mx_dots_packed_async(nk_dtype_t a_dtype, void const *a, nk_size_t a_stride, void const *a_scales,
                                nk_size_t a_scales_stride, void const *packed, nk_dtype_t c_dtype, void *c, nk_size_t c_stride,
                                nk_size_t height, nk_size_t width, nk_size_t depth, void *workspace, nk_size_t workspace_bytes,
                                void *stream_) {
    MxGeometry g;
    hipStream_t const stream = (hipStream_t)stream_;
    if (height >= (1ull << 31) || !mx_geometry(1, width, depth, g)) return mx_fail("mx_dots_packed: unsupported dimensions");
    if (!height || !width) return 0;
    if (int const status = check_size(height, (height + 127) / 128, width, g)) return status;
    if (int const status = depth ? check_a(a_dtype, a, a_scales, a_stride) : 0) return status;
    if (int const status = check_c(c_dtype, c, c_stride)) return status;
    if (!packed || ((uintptr_t)packed & 15)) return mx_fail("mx_dots_packed: the image has to be 16-byte aligned");
    bool const few = launches_few((height + 63) / 64, width), fused = few && !a_scales && fuses(height, height * depth, g);
    MxArgs p = {};
    p.image = (uint8_t const *)packed, p.c = (uint8_t *)c, p.c_stride = c_stride;
    p.m = (uint32_t)height, p.n = (uint32_t)width, p.k = (uint32_t)depth, p.count = 1, p.a_share = 1;
    p.steps = g.steps, p.supers = g.supers, p.tiles = g.tiles;
    if (fused) p.a = (uint8_t const *)a, p.a_pitch = a_stride;
    else {
        Staging const s = staging_of(height, g);
        if (s.bytes && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < s.bytes))
            return mx_fail("mx_dots_packed: the workspace is too small or not 256-byte aligned");
        if (int const status = stage(a_dtype, a, a_stride, a_scales, a_scales_stride, p.m, p.k, g, s, (uint8_t *)workspace, nullptr, 0, 1, 0, 0, stream))
            return status;
        p.a = (uint8_t const *)workspace, p.a_scales = p.a + s.scales_at;
    }
    return with_type(c_dtype, [&](auto value) {
        return launch_product<decltype(value), false>(p, few, 0, a_dtype, fused, p.m, g, stream);
    });
}

nk_size_t nk_amd_mx_experts_workspace_size(nk_size_t slots, nk_size_t a_share, nk_size_t experts, nk_size_t width,
                                           nk_size_t depth, int a_is_codes, int weighted) {
    MxGeometry g;
    PlanGeometry shape;
    if (!slots || !a_share || !mx_geometry(experts, width, depth, g) || !plan_geometry(slots, experts, shape)) return 0;
    return experts_layout(shape, slots, a_share, experts, width, depth, g, a_is_codes != 0, weighted != 0).bytes;
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
    if (int const status = check_size(shape.max_rows, shape.max_tiles, width, g)) return status;
    if (int const status = depth ? check_a(a_dtype, a, a_scales, a_stride) : 0) return status;
    if (int const status = check_c(c_dtype, c, c_stride)) return status;
    if (!packed || ((uintptr_t)packed & 15) || !plan || ((uintptr_t)plan & 15)) return mx_fail("mx_dots_experts: image and plan have to be 16-byte aligned");
    ExpertsLayout const l = experts_layout(shape, slots, a_share, experts, width, depth, g, a_scales != nullptr, weights != nullptr);
    if (l.bytes && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < l.bytes))
        return mx_fail("mx_dots_experts: the workspace is too small or not 256-byte aligned");
    MxArgs p = {};
    p.image = (uint8_t const *)packed, p.plan = (uint32_t const *)plan;
    p.m = (uint32_t)slots, p.n = (uint32_t)width, p.k = (uint32_t)depth, p.count = (uint32_t)experts, p.a_share = (uint32_t)a_share;
    p.steps = g.steps, p.supers = g.supers, p.tiles = g.tiles;
    p.tiles_m = shape.max_tiles, p.order = (uint32_t)shape.order, p.tile_list = (uint32_t)shape.tiles;
    if (l.fused) p.a = (uint8_t const *)a, p.a_pitch = a_stride;
    else {
        if (l.quantised) {
            uint8_t *const codes = (uint8_t *)workspace + l.codes_at, *const scales = (uint8_t *)workspace + l.codes_scales_at;
            if (int const status = launch_quantize(a_dtype, a, slots / a_share, depth, a_stride, codes, l.codes_stride, scales, l.codes_scales_stride, stream))
                return status;
            a = codes, a_stride = l.codes_stride, a_scales = scales, a_scales_stride = l.codes_scales_stride;
        }
        if (int const status = stage(a_dtype, a, a_stride, a_scales, a_scales_stride, shape.max_rows, p.k, g, l.staged, (uint8_t *)workspace, plan, shape.order, p.a_share, p.m, p.count, stream))
            return status;
        p.a = (uint8_t const *)workspace, p.a_scales = p.a + l.staged.scales_at;
    }
    uint8_t *sums = (uint8_t *)workspace + l.sums_at;
    int const product_dtype = weights ? (int)nk_f32_k : (int)c_dtype;
    if (weights) p.sorted = 1, p.c = sums, p.c_stride = l.sums_values * 4;
    else p.c = (uint8_t *)c, p.c_stride = c_stride;
    int const status = with_type(product_dtype, [&](auto value) {
        return launch_product<decltype(value), true>(p, l.few, shape.tile_rows, a_dtype, l.fused, 16, g, stream);
    });
    if (status || !weights) return status;
    uint64_t const tokens = slots / top_k, pieces = (width + 3) / 4;
    uint64_t const slab = kMostThreads / pieces; // tokens of one launch
    for (uint64_t first = 0; first < tokens; first += slab) {
        uint64_t const here = tokens - first < slab ? tokens - first : slab;
        uint32_t const place = (uint32_t)(shape.place + first * top_k);
        int const done = with_type(c_dtype, [&](auto value) {
            typedef decltype(value) Out;
            hipLaunchKernelGGL((combine_kernel<Out>), dim3((uint32_t)((here * pieces + 255) / 256)), dim3(256), 0, stream,
                               (float const *)sums, l.sums_values, p.plan, p.m, p.count, place, weights + first * top_k, (uint32_t)top_k, (uint32_t)here,
                               p.n, (uint32_t)pieces, (Out *)((uint8_t *)c + first * c_stride), (uint64_t)c_stride);
            hipError_t const e = hipGetLastError();
            return e == hipSuccess ? 0 : mx_fail(e, "combine_kernel");
        });
        if (done) return done;
    }
    return 0;
}

} // extern "C"
