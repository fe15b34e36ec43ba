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
#include "dense_tiles_gfx950.hpp"

namespace nk_gfx950 {

int launch_column_sum(float const *values, uint64_t rows, uint64_t k, uint32_t kind, void *out, hipStream_t stream);

namespace {

inline uint64_t up_to(uint64_t n, uint64_t step) { return (n + step - 1) / step * step; }

/** Up to 16 bytes of a row of `bytes` from `at` on, wherever they lie; zeros behind the end. (The row's last piece is its last 16 bytes, shifted: byte by
 *  byte, 1 x 8192 x 1000 in 8 bits took 12 us, and 5.6 with twice the bytes and no such piece.) */
__device__ __forceinline__ v4u load_piece(uint8_t const *row, uint32_t at, uint32_t bytes) {
    if (at + 16 <= bytes) return *(v4u_anywhere const *)(row + at);
    v4u piece = {0, 0, 0, 0};
    if (at >= bytes) return piece;
    if (bytes >= 16) {
        v4u const last = *(v4u_anywhere const *)(row + bytes - 16);
        uint32_t const gone = (at + 16 - bytes) * 8; // bits: 8 to 120
        uint64_t const low = last[0] | (uint64_t)last[1] << 32, high = last[2] | (uint64_t)last[3] << 32;
        uint64_t const first = gone < 64 ? low >> gone | high << (64 - gone) : high >> (gone - 64), second = gone < 64 ? high >> gone : 0;
        return v4u {(uint32_t)first, (uint32_t)(first >> 32), (uint32_t)second, (uint32_t)(second >> 32)};
    }
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
        if (at + i < bytes) piece[i / 4] |= (uint32_t)row[at + i] << 8 * (i % 4);
    return piece;
}

// ---- operands as the tiles take them -------------------------------------------------------------------------------

/** Rows of `bytes` to where they are 16-byte aligned, zeros up to the next multiple of 16: a thread for 16 bytes. */
struct MoveArgs {
    uint8_t const *from;
    uint64_t from_stride, pieces; // rows times `each`
    uint8_t *to;
    uint64_t to_stride;
    uint32_t each, bytes;
};
__device__ __forceinline__ void move_rows(MoveArgs const &p, uint64_t block) {
    uint64_t const at = block * 256 + threadIdx.x;
    if (at >= p.pieces) return;
    uint64_t const row = at / p.each;
    uint32_t const piece = (uint32_t)(at - row * p.each);
    *(v4u *)(p.to + row * p.to_stride + piece * 16) = load_piece(p.from + row * p.from_stride, piece * 16, p.bytes);
}

/** Scales as the tiles read them, words of four blocks by stage and row (zeros where there is no block): 32 rows times 32 stages a workgroup, through LDS, as
 *  rows are read and written along different axes. */
struct WordsArgs {
    uint8_t const *scales;
    uint64_t stride;
    uint32_t *words;
    uint32_t rows, blocks, stages, pitch;
};
__device__ __forceinline__ void scale_words(WordsArgs const &p, uint64_t block, uint32_t (&tile)[32][33]) {
    uint32_t const high = p.pitch / 32, row0 = (uint32_t)(block % high) * 32, stage0 = (uint32_t)(block / high) * 32, x = threadIdx.x % 32;
#pragma unroll
    for (uint32_t y = threadIdx.x / 32; y < 32; y += 8) {
        uint32_t const row = row0 + y, at = (stage0 + x) * 4;
        uint32_t word = 0;
        if (row < p.rows && at < p.blocks) {
            uint8_t const *const from = p.scales + row * p.stride + at;
            if (at + 4 <= p.blocks) word = *(u32_anywhere const *)from;
            else
                for (uint32_t i = 0; i < p.blocks - at; ++i) word |= (uint32_t)from[i] << 8 * i;
        }
        tile[y][x] = word;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t y = threadIdx.x / 32; y < 32; y += 8)
        if (stage0 + y < p.stages) p.words[(uint64_t)(stage0 + y) * p.pitch + row0 + x] = tile[x][y];
}

/** What is made of a product's operands before it: every job in one launch, as each by itself takes 3 us of a small product's 14. */
struct Preparation {
    QuantizeArgs quantize;
    MoveArgs move[3];
    WordsArgs words[3];
    uint64_t ends[7]; // the first workgroup behind each job's
    uint64_t first;   // of the launch
    int moves, scaled;
    void add(QuantizeArgs const &q) { quantize = q; }
    void add(uint8_t const *from, uint64_t from_stride, uint64_t rows, uint64_t bytes, uint8_t *to, uint64_t to_stride) {
        uint64_t const each = (bytes + 15) / 16;
        move[moves++] = {from, from_stride, rows * each, to, to_stride, (uint32_t)each, (uint32_t)bytes};
    }
    void add(WordsArgs const &w) { words[scaled++] = w; }
};
__global__ __launch_bounds__(256) void prepare_kernel(Preparation p) {
    __shared__ uint32_t tile[32][33];
    uint64_t const block = p.first + blockIdx.x;
    if (block < p.ends[0]) return quantize_stretches(p.quantize, block);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        if (block < p.ends[1 + i]) return move_rows(p.move[i], block - p.ends[i]);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        if (block < p.ends[4 + i]) return scale_words(p.words[i], block - p.ends[3 + i], tile);
    }
}
int launch_preparation(Preparation &p, hipStream_t stream) {
    uint64_t end = 0;
    p.ends[0] = end += (p.quantize.stretches + 3) / 4;
    for (int i = 0; i < 3; ++i) p.ends[1 + i] = end += (p.move[i].pieces + 255) / 256;
    for (int i = 0; i < 3; ++i) p.ends[4 + i] = end += (uint64_t)(p.words[i].pitch / 32) * ((p.words[i].stages + 31) / 32);
    for (p.first = 0; p.first < end; p.first += kMostThreads / 256) {
        uint64_t const here = end - p.first < kMostThreads / 256 ? end - p.first : kMostThreads / 256;
        hipLaunchKernelGGL(prepare_kernel, dim3((uint32_t)here), dim3(256), 0, stream, p);
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, "prepare_kernel");
    }
    return 0;
}

/** Sums of the splits, in their order, and what follows: eight adjacent results a thread. */
template <bool GATED>
__global__ __launch_bounds__(256) void join_kernel(float const *partial, uint32_t splits, uint32_t m, uint32_t n, Epilogue e) {
    uint32_t const each = (n + 7) / 8;
    uint64_t const at = (uint64_t)blockIdx.x * 256 + threadIdx.x, row = at / each, plane = (uint64_t)m * n;
    if (row >= m) return;
    uint32_t const col = (uint32_t)(at - row * each) * 8;
    float v[1][8] = {}, q[1][8] = {};
#pragma unroll 4
    for (uint32_t i = 0; i < splits; ++i) { // (several parts on their way at a time)
        float part[8];
        load_adjacent(partial + i * plane * (GATED ? 2 : 1) + row * n, col, n, part);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[0][j] += part[j];
        if constexpr (GATED) {
            load_adjacent(partial + (2 * i + 1) * plane + row * n, col, n, part);
#pragma unroll
            for (int j = 0; j < 8; ++j) q[0][j] += part[j];
        }
    }
    finish<GATED>(e, (uint32_t)row, m, col, n, v, q);
}

// ---- few rows ------------------------------------------------------------------------------------------------------

struct FewSide {
    uint8_t const *values;
    uint64_t stride;
    uint8_t const *scales;
    uint64_t scales_stride;
};
struct FewArgs {
    FewSide a, b[2];
    uint32_t m, n, bytes; // bytes of a row
    uint32_t first;       // of the launch's blocks of columns
    Epilogue e;
};
/** c += x y for 16 rows of each and 64 bytes of depth of 16-bit values. */
template <class T>
__device__ __forceinline__ v4f multiply_16(v4u x, v4u y, v4f c) {
#ifdef NK_MX_DEVICE_BUILTINS
    if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x), __builtin_bit_cast(v8bf, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0, 0);
#else
    return c;
#endif
}
/** 128 8-bit values; a lane's scales. */
__device__ __forceinline__ v4f multiply_16(v4u const (&x)[2], v4u const (&y)[2], v4f c, uint32_t x_scale, uint32_t y_scale) {
#ifdef NK_MX_DEVICE_BUILTINS
    v8i const p = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], (int)x[1][0], (int)x[1][1], (int)x[1][2], (int)x[1][3]};
    v8i const q = {(int)y[0][0], (int)y[0][1], (int)y[0][2], (int)y[0][3], (int)y[1][0], (int)y[1][1], (int)y[1][2], (int)y[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p, q, c, 0, 0, 0, (int)x_scale, 0, (int)y_scale);
#else
    return c;
#endif
}

/**
 *  Up to 16 MB rows: the stream of the matrix is what bounds it. A workgroup has 16 NB columns (of both matrices, where gated); its wavefronts take every
 *  WAVES-th 256 bytes of depth, and their sums are joined at the end in their order. Each wavefront reads whole 256-byte pieces of rows, at any
 *  alignment, two pieces ahead, and turns them to fragments through LDS of its own (16-byte piece p of row r at p ^ r), without a barrier.
 */
template <class T, int MB, int NB, bool GATED, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void few_kernel(FewArgs p) {
    constexpr bool kScaled = __is_same(T, Mx8);
    constexpr int kMatrices = GATED ? 2 : 1, kBlocks = NB * kMatrices, kSteps = kScaled ? 2 : 4;
    __shared__ __attribute__((aligned(1024))) uint8_t rooms[WAVES][(kBlocks + MB) * 4096];
    uint32_t const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, r4 = l / 16, piece = l % 16;
    uint32_t const col0 = (p.first + blockIdx.x) * 16 * NB, row0 = blockIdx.y * 16 * MB, rows = p.m - row0, chunks = (p.bytes + 255) / 256;
    uint8_t *const room = rooms[wave];

    uint8_t const *w_rows[kBlocks][4], *a_rows[MB][4]; // rows past the end are the last one again: their results are dropped
    uint8_t const *w_scales[kBlocks], *a_scales[MB];
    uint32_t const blocks = (p.bytes + 31) / 32;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        FewSide const &side = p.b[b / NB];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t const col = col0 + b % NB * 16 + i * 4 + r4;
            w_rows[b][i] = side.values + (col < p.n ? col : p.n - 1) * side.stride;
        }
        uint32_t const col = col0 + b % NB * 16 + l % 16;
        w_scales[b] = side.scales + (col < p.n ? col : p.n - 1) * side.scales_stride;
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t const row = b * 16 + i * 4 + r4;
            a_rows[b][i] = p.a.values + (row0 + (row < rows ? row : rows - 1)) * p.a.stride;
        }
        uint32_t const row = b * 16 + l % 16;
        a_scales[b] = p.a.scales + (row0 + (row < rows ? row : rows - 1)) * p.a.scales_stride;
    }

    v4f sum[kBlocks][MB] = {};
    v4u w[2][kBlocks][4], a[2][MB][4] = {};
    uint32_t w_scale[2][kBlocks][2], a_scale[2][MB][2];
    auto const load = [&](auto slot, uint32_t c) {
        constexpr int kSlot = decltype(slot)::value;
        uint32_t const at = c * 256 + piece * 16;
        if constexpr (kScaled) { // the lane's blocks: those of its quarter of the wavefront
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint32_t const block = c * 8 + s * 4 + r4;
                bool const there = block < blocks;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) w_scale[kSlot][b][s] = there ? w_scales[b][block] : 0;
#pragma unroll
                for (int b = 0; b < MB; ++b) a_scale[kSlot][b][s] = there ? a_scales[b][block] : 0;
            }
        }
        if ((c + 1) * 256 <= p.bytes) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[kSlot][b][i] = *(v4u_anywhere const *)(w_rows[b][i] + at);
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (b * 16 + i * 4 < rows) a[kSlot][b][i] = *(v4u_anywhere const *)(a_rows[b][i] + at);
        } else {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[kSlot][b][i] = load_piece(w_rows[b][i], at, p.bytes);
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (b * 16 + i * 4 < rows) a[kSlot][b][i] = load_piece(a_rows[b][i], at, p.bytes);
        }
    };
    auto const fragment = [&](int b, int at) { return *(v4u const *)(room + b * 4096 + l % 16 * 256 + (((uint32_t)at) ^ (l % 16)) * 16); };
    auto const step = [&](auto slot, uint32_t c) {
        constexpr int kSlot = decltype(slot)::value;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t const r = i * 4 + r4, to = r * 256 + (piece ^ r) * 16;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) *(v4u *)(room + b * 4096 + to) = w[kSlot][b][i];
#pragma unroll
            for (int b = 0; b < MB; ++b) *(v4u *)(room + (kBlocks + b) * 4096 + to) = a[kSlot][b][i];
        }
        uint32_t ws[kBlocks][2], as[MB][2];
        if constexpr (kScaled) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) ws[b][s] = w_scale[kSlot][b][s];
#pragma unroll
                for (int b = 0; b < MB; ++b) as[b][s] = a_scale[kSlot][b][s];
            }
        }
        if (c + 2 * WAVES < chunks) load(slot, c + 2 * WAVES);
        wave_fence();
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if constexpr (kScaled) { // of the 128 values at 128 s a lane has 16 of the first 64 and as many of the second
                int const first = 8 * s + r4;
                v4u x[kBlocks][2], y[MB][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) x[b][h] = fragment(b, first + 4 * h);
#pragma unroll
                    for (int b = 0; b < MB; ++b) y[b][h] = fragment(kBlocks + b, first + 4 * h);
                }
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                    for (int j = 0; j < MB; ++j) sum[i][j] = multiply_16(x[i], y[j], sum[i][j], ws[i][s], as[j][s]);
            } else {
                v4u x[kBlocks], y[MB];
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) x[b] = fragment(b, 4 * s + r4);
#pragma unroll
                for (int b = 0; b < MB; ++b) y[b] = fragment(kBlocks + b, 4 * s + r4);
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                    for (int j = 0; j < MB; ++j) sum[i][j] = multiply_16<T>(x[i], y[j], sum[i][j]);
            }
        }
        wave_fence();
    };
    if (wave < chunks) load(Number<0>(), wave);
    if (wave + WAVES < chunks) load(Number<1>(), wave + WAVES);
    for (uint32_t c = wave; c < chunks; c += 2 * WAVES) {
        step(Number<0>(), c);
        if (c + WAVES < chunks) step(Number<1>(), c + WAVES);
    }

    // sums of the wavefronts: [matrix][row][column], a lane has four columns of a row
    constexpr uint32_t kPitch = 16 * NB + 4, kRoom = kMatrices * MB * 16 * kPitch;
    static_assert(kRoom * 4 <= sizeof(rooms[0]), "sums have to fit the wavefront's room");
    wave_fence();
    float *const mine = (float *)room;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < MB; ++i) *(v4f *)(mine + ((b / NB * MB + i) * 16 + l % 16) * kPitch + b % NB * 16 + r4 * 4) = sum[b][i];
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < MB * 16 * NB * 2; t += 64 * WAVES) {
        uint32_t const r = t / (NB * 2), c = t % (NB * 2) * 8;
        if (r >= rows || col0 + c >= p.n) continue;
        float v[1][8] = {}, q[1][8] = {};
        for (int i = 0; i < WAVES; ++i) {
            float const *const its = (float const *)rooms[i] + r * kPitch + c;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[0][j] += its[j];
                if (GATED) q[0][j] += its[MB * 16 * kPitch + j];
            }
        }
        finish<GATED>(p.e, row0 + r, p.m, col0 + c, p.n, v, q);
    }
}
template <class T, int MB, int NB, bool GATED, int WAVES>
int launch_few(FewArgs p, hipStream_t stream) {
    uint32_t const high = (p.m + 16 * MB - 1) / (16 * MB), blocks = (p.n + 16 * NB - 1) / (16 * NB);
    uint64_t const most = kMostThreads / (64 * WAVES) / high; // blocks of a launch
    for (uint64_t first = 0; first < blocks; first += most) {
        p.first = (uint32_t)first;
        hipLaunchKernelGGL((few_kernel<T, MB, NB, GATED, WAVES>), dim3((uint32_t)(blocks - first < most ? blocks - first : most), high), dim3(64 * WAVES), 0, stream, p);
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, "few_kernel");
    }
    return 0;
}
template <class T>
int launch_few_of(FewArgs const &p, bool gated, hipStream_t stream) {
    if (p.m <= 16) return gated ? launch_few<T, 1, 1, true, 4>(p, stream) : launch_few<T, 1, 1, false, 8>(p, stream);
    return gated ? launch_few<T, 2, 1, true, 4>(p, stream) : launch_few<T, 2, 1, false, 8>(p, stream);
}
/**
 *  Which products go there: those of up to 16 rows, and of up to 64 where the matrix is small. Each workgroup reads all of A, and every 32 rows all of its
 *  columns, so that tiles win with size: 24 x 8192 x 8192 bf16 38.6 us here and 33 in tiles, 24 x 1024 x 8192 12.5 and 14, 64 x 2048 x 2048, the largest that goes here, 6.4 and 10.9.
 *  (Whole passes over three sets of operands, bf16; 8 bits go by the same limit, with 24 x 8192 x 8192 20 us in tiles.)
 */
bool of_few_rows(uint64_t m, uint64_t n, uint64_t k, bool gated) { return m <= 16 || (m <= 64 && (double)m * (double)n * (double)k * (gated ? 2 : 1) <= 0x1p28); }

// ---- tiles ---------------------------------------------------------------------------------------------------------

constexpr uint64_t kMostTiles = (1ull << 24) - 1; // of a launch, which has fewer than 2^32 threads

struct TilePlan {
    int shape;
    uint32_t splits, split_stages;
};
/**
 *  The shape of tiles and the splits of the depth that take the least time by a simple account, in microseconds of a compute unit, from what was
 *  measured with bf16: a stage of a workgroup that is alone (512 x 4096 x 4096 and 64 x 8192 x 8192), one among as many as the account takes to fit (8192 x 8192 by depths of 64 to
 *  4096), what a tile's beginning and end add, and a launch and the partial sums' way through memory where there are splits. It is within a
 *  sixth of the times of ten bf16 products between 64 x 8192 x 8192 and 4096 x 4096 x 1024. The transposing reads of depths along columns cost tiles of 128 rows more (the
 *  gradient of 4096 x 2048 over 16384: 316 us in such tiles).
 *
 *  All types and forms go by it, some of them worse. Of gated tiles of 64 rows three fit, where four are counted, and of those in 8 bits with depths that end at any byte two:
 *  1001 x 2050 x 1000 has 528 tiles for 512 places, so that it takes 19 to 20.5 us and not 9.6. The results' bytes are not counted: f16 8192 x 8191 x 1000 to f32 takes 190 to 222 us and
 *  not 149 (153 for tiles of 128 rows).
 */
TilePlan tile_plan(uint64_t m, uint64_t n, uint64_t stages, bool gated, bool b_columns = false) {
    static constexpr double kAlone[3] = {0.45, 0.57, 1.48}, kEach[3] = {0.173, 0.442, 1.48}, kEnds[3] = {0.8, 2.5, 13.5};
    static constexpr uint64_t kResident[3] = {4, 2, 1};
    uint64_t const found = (uint64_t)compute_unit_count(), units = found ? found : 256; // (a size may be asked for where there is no GPU)
    TilePlan best = {0, 1, (uint32_t)stages};
    double least = 1e300;
    for (int shape = 0; shape < 3; ++shape) {
        uint64_t const rows = 64u << shape, columns = gated ? (shape == 2 ? 128 : 64) : rows;
        uint64_t const tiles = ((m + rows - 1) / rows) * ((n + columns - 1) / columns);
        if (tiles > kMostTiles) continue; // (2^30 x 8 in tiles of 64 rows)
        double const each = gated && shape == 0 ? 0.3 : b_columns && shape == 1 ? 0.54 : kEach[shape];
        auto const together = [&](uint64_t workgroups) { return workgroups * each > kAlone[shape] ? workgroups * each : workgroups ? kAlone[shape] : 0.0; };
        for (uint64_t splits = 1; splits <= 16; splits *= 2) {
            if (splits > 1 && (stages < splits * 4 || tiles * splits > units * 4)) break;
            uint64_t const some = (stages + splits - 1) / splits, its = splits > 1 ? up_to(some, 2) : some, there = stages ? (stages + its - 1) / its : 1;
            uint64_t const on_unit = (tiles * there + units - 1) / units;
            double const joined = there > 1 ? 4 + (double)m * n * (gated ? 2 : 1) * (there + 1) * 4 / 3e6 : 0;
            double const time = its * (on_unit / kResident[shape] * together(kResident[shape]) + together(on_unit % kResident[shape])) + on_unit * kEnds[shape] + joined;
            if (time < least) least = time, best = {shape, (uint32_t)there, (uint32_t)its};
        }
    }
    return best;
}
/** Are there more results than the tiles of one launch make? (Then those of every shape are too many.) */
bool too_many(TilePlan const &t, uint64_t m, uint64_t n, bool gated) {
    uint64_t const rows = 64u << t.shape, columns = gated ? (t.shape == 2 ? 128 : 64) : rows;
    return ((m + rows - 1) / rows) * ((n + columns - 1) / columns) * t.splits > kMostTiles;
}
uint64_t partial_bytes(TilePlan const &t, uint64_t m, uint64_t n, bool gated) { return t.splits > 1 ? up_to(t.splits * m * n * (gated ? 8 : 4), 256) : 0; }

/** Queues the tiles of a product (extents, depths and operands are in `p`) and what joins their splits. */
int launch_tiles(int dtype, TileForm form, TilePlan const &t, TileArgs p, float *partial, hipStream_t stream) {
    form.shape = t.shape;
    p.splits = t.splits, p.split_stages = t.split_stages, p.partial = partial;
    uint32_t const rows = 64u << t.shape, columns = form.gated ? (t.shape == 2 ? 128 : 64) : rows;
    p.tiles_m = (p.m + rows - 1) / rows, p.tiles_n = (p.n + columns - 1) / columns;
    if (int const status = dtype == nk_bf16_k ? launch_tiles_bf16(form, p, stream) : dtype == nk_f16_k ? launch_tiles_f16(form, p, stream) : launch_tiles_mx8(form, p, stream)) return status;
    if (t.splits == 1) return 0;
    uint64_t const eights = (uint64_t)p.m * ((p.n + 7) / 8);
    dim3 const grid((uint32_t)((eights + 255) / 256));
    if (form.gated) hipLaunchKernelGGL(join_kernel<true>, grid, dim3(256), 0, stream, partial, p.splits, p.m, p.n, p.e);
    else hipLaunchKernelGGL(join_kernel<false>, grid, dim3(256), 0, stream, partial, p.splits, p.m, p.n, p.e);
    hipError_t const e = hipGetLastError();
    return e == hipSuccess ? 0 : mx_fail(e, "join_kernel");
}

/** Can the tiles read these rows in place? */
bool in_place(void const *values, uint64_t stride) { return !((uintptr_t)values & 3) && !(stride & 3) && stride <= kTileStride; }

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
            float g[8], x[1][8], up[8], d[8], e[1][8];
            load_adjacent(p.grad_kind, p.grad + row * p.grad_stride, col, p.n, g);
            if (p.pre) load_adjacent((float const *)((uint8_t const *)p.pre + row * p.pre_stride), col, p.n, x[0]);
            if (p.gated) {
                load_adjacent((float const *)((uint8_t const *)p.pre_up + row * p.pre_stride), col, p.n, up);
#pragma unroll
                for (int j = 0; j < 8; ++j) e[0][j] = x[0][j];
                activate(p.activation, e);
            }
            if (p.pre) slope(p.activation, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                d[j] = p.pre ? g[j] * x[0][j] : g[j];
                if (p.gated) d[j] *= up[j], e[0][j] *= g[j];
                sum[j] += d[j];
            }
            if (p.d) {
                T *const to = (T *)(p.d + row * p.d_stride) + col;
                store_some(to, d, p.padded - col);
                if (p.gated) store_some(to + p.up_at, e[0], p.padded - col);
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
    if (mx8 && (l->pre || l->pre_up)) return mx_fail("linear: sums are left by products of 16-bit matrices (those of mx8 have no gradient, and not the bits of f32)");
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

/** Where a product's workspace has what it makes of its operands. */
struct LinearLayout {
    bool few, quantises, moves_a, moves_w, moves_up; // A's codes are made; rows are moved to where the tiles can read them
    uint64_t codes_stride, moved_stride;
    uint64_t scales_stride, scales_at; // A's scales as bytes (few rows)
    uint64_t a_pitch, w_pitch, a_words_at, w_words_at, up_words_at;
    uint64_t a_at, w_at, up_at, partial_at, bytes;
    uint64_t stages;
    TilePlan tiles;
};
LinearLayout linear_layout(nk_amd_linear_t const *l) {
    LinearLayout y = {};
    if (!l->height || !l->width) return y;
    bool const mx8 = l->w_dtype == nk_e4m3_k;
    uint64_t const bytes = l->depth * (mx8 ? 1 : 2);
    uint64_t end = 0;
    auto const room = [&](uint64_t size) { uint64_t const at = end; return end += up_to(size, 256), at; };
    y.quantises = mx8 && l->a_dtype != nk_e4m3_k && l->depth;
    y.codes_stride = up_to(l->depth, 128), y.moved_stride = up_to(bytes, 128);
    y.few = of_few_rows(l->height, l->width, l->depth, l->gated);
    if (y.quantises) y.a_at = room(l->height * y.codes_stride);
    if (y.few) {
        y.scales_stride = y.codes_stride / 32;
        if (y.quantises) y.scales_at = room(l->height * y.scales_stride);
        return y.bytes = end, y;
    }
    y.stages = (bytes + 127) / 128;
    y.tiles = tile_plan(l->height, l->width, y.stages, l->gated);
    bool const ends = y.tiles.shape < 2 || bytes % 16 == 0; // (the depth may end where it does)
    y.moves_a = !y.quantises && bytes && !(ends && in_place(l->a, l->a_stride));
    y.moves_w = bytes && !(ends && in_place(l->w, l->w_stride));
    y.moves_up = l->gated && bytes && !(ends && in_place(l->w_up, l->w_up_stride));
    if (y.moves_a) y.a_at = room(l->height * y.moved_stride);
    if (y.moves_w) y.w_at = room(l->width * y.moved_stride);
    if (y.moves_up) y.up_at = room(l->width * y.moved_stride);
    if (mx8) {
        y.a_pitch = up_to(l->height, 256), y.w_pitch = up_to(l->width, 256);
        y.a_words_at = room(y.stages * y.a_pitch * 4), y.w_words_at = room(y.stages * y.w_pitch * 4);
        if (l->gated) y.up_words_at = room(y.stages * y.w_pitch * 4);
    }
    y.partial_at = room(partial_bytes(y.tiles, l->height, l->width, l->gated));
    return y.bytes = end, y;
}
/** Where a backward pass's workspace has d (and e behind it in each row), the sums of d, operands moved to where the tiles can read them, and splits. */
struct BackwardLayout {
    uint64_t padded, d_stride, column_sums_at, partials, rows_each, bytes;
    bool writes_d, sums, moves_a, moves_w, moves_up;
    uint64_t moved_stride, a_at, w_at, up_at, partial_at;
    uint64_t stages, first_stages; // of the depth of A's gradient
    TilePlan of_a, of_w;
};
BackwardLayout backward_layout(nk_amd_linear_backward_t const *l) {
    BackwardLayout y = {};
    uint64_t end = 0;
    auto const room = [&](uint64_t size) { uint64_t const at = end; return end += up_to(size, 256), at; };
    bool const gated = l->gated, some = l->height && l->width, of_a = l->grad_a && some && l->depth, of_w = (l->grad_w || l->grad_w_up) && some && l->depth;
    y.writes_d = (of_a || of_w) && (gated || l->activation || l->grad_dtype != l->dtype || l->width % 8 || !in_place(l->grad, l->grad_stride));
    y.sums = l->grad_bias != nullptr;
    y.padded = up_to(l->width, 64), y.d_stride = y.padded * 2 * (gated ? 2 : 1);
    // Rows of a workgroup that makes d: 64 (128, where a grid would be too high), fewer until there are 1024 workgroups (343 x 1150 gated: 51 us with 64).
    y.rows_each = l->height <= 1u << 21 ? 64 : 128;
    while (y.rows_each > 4 && (l->height + y.rows_each - 1) / y.rows_each * ((y.padded + 511) / 512) < 1024) y.rows_each /= 2;
    y.partials = (l->height + y.rows_each - 1) / y.rows_each;
    if (y.writes_d) room(l->height * y.d_stride); // (at 0)
    if (y.sums) y.column_sums_at = room(y.partials * l->width * 4);
    y.moved_stride = up_to(l->depth * 2, 128);
    y.moves_a = of_w && !in_place(l->a, l->a_stride);
    y.moves_w = of_a && !in_place(l->w, l->w_stride);
    y.moves_up = gated && of_a && !in_place(l->w_up, l->w_up_stride);
    if (y.moves_a) y.a_at = room(l->height * y.moved_stride);
    if (y.moves_w) y.w_at = room(l->width * y.moved_stride);
    if (y.moves_up) y.up_at = room(l->width * y.moved_stride);
    y.first_stages = y.padded / 64, y.stages = y.first_stages * (gated ? 2 : 1);
    y.of_a = tile_plan(l->height, l->depth, y.stages, false, true), y.of_w = tile_plan(l->width, l->depth, (l->height + 63) / 64, false, true);
    uint64_t const a_bytes = of_a ? partial_bytes(y.of_a, l->height, l->depth, false) : 0, w_bytes = of_w ? partial_bytes(y.of_w, l->width, l->depth, false) : 0;
    y.partial_at = room(a_bytes > w_bytes ? a_bytes : w_bytes);
    return y.bytes = end, y;
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

int nk_amd_linear_async(nk_amd_linear_t const *l, void *workspace, nk_size_t workspace_bytes, void *raw_stream) {
    if (int const status = check_linear(l)) return status;
    if (!l->height || !l->width) return 0;
    if (int const status = check_linear_operands(l)) return status;
    LinearLayout const y = linear_layout(l);
    if (check_workspace("linear: the workspace is too small or not 256-byte aligned", workspace, workspace_bytes, y.bytes)) return -1;
    if (!y.few && too_many(y.tiles, l->height, l->width, l->gated)) return mx_fail("linear: more results than one launch makes");
    bool const mx8 = l->w_dtype == nk_e4m3_k, gated = l->gated;
    hipStream_t const stream = (hipStream_t)raw_stream;
    uint8_t *const room = (uint8_t *)workspace;
    uint64_t const bytes = l->depth * (mx8 ? 1 : 2);
    Epilogue const e = {l->bias, (uint8_t const *)l->residual, (uint8_t *)l->c, l->pre, l->pre_up, l->residual_stride, l->c_stride, l->pre_stride, kind_of(l->bias_dtype),
                        kind_of(l->residual_dtype), kind_of(l->c_dtype), (uint32_t)l->activation};
    Preparation before = {};
    if (y.quantises) {
        uint64_t const each = (l->depth + 511) / 512;
        before.add(QuantizeArgs {(uint8_t const *)l->a, l->a_stride, l->height * each, room + y.a_at, y.few ? room + y.scales_at : nullptr, y.codes_stride, y.scales_stride,
                    y.few ? nullptr : (uint32_t *)(room + y.a_words_at), y.a_pitch, kind_of(l->a_dtype), (uint32_t)each, (uint32_t)l->depth, (uint32_t)up_to(l->depth, 16)});
    }
    if (y.few) {
        FewArgs p = {};
        p.m = (uint32_t)l->height, p.n = (uint32_t)l->width, p.bytes = (uint32_t)bytes, p.e = e;
        p.a = {(uint8_t const *)l->a, l->a_stride, (uint8_t const *)l->a_scales, l->a_scales_stride};
        if (y.quantises) p.a = {room + y.a_at, y.codes_stride, room + y.scales_at, y.scales_stride};
        p.b[0] = {(uint8_t const *)l->w, l->w_stride, (uint8_t const *)l->w_scales, l->w_scales_stride};
        p.b[1] = {(uint8_t const *)l->w_up, l->w_up_stride, (uint8_t const *)l->w_up_scales, l->w_up_scales_stride};
        if (int const status = launch_preparation(before, stream)) return status;
        return mx8 ? launch_few_of<Mx8>(p, gated, stream) : l->w_dtype == nk_f16_k ? launch_few_of<_Float16>(p, gated, stream) : launch_few_of<__bf16>(p, gated, stream);
    }
    TileArgs p = {};
    p.m = (uint32_t)l->height, p.n = (uint32_t)l->width, p.stages = p.first_stages = (uint32_t)y.stages, p.e = e;
    p.a.extent = p.m, p.b.extent = p.n, p.a.k = p.b.k = (uint32_t)l->depth;
    uint32_t const whole = (uint32_t)(up_to(bytes, 16) / (mx8 ? 1 : 2)); // (what is moved or quantised ends with zeros)
    if (y.quantises || y.moves_a) p.a.k = whole;
    if (y.moves_w && (!gated || y.moves_up)) p.b.k = whole;
    p.a.pitch = (uint32_t)y.a_pitch, p.b.pitch = (uint32_t)y.w_pitch;
    p.a.values[0] = (uint8_t const *)l->a, p.a.stride[0] = l->a_stride;
    p.b.values[0] = (uint8_t const *)l->w, p.b.stride[0] = l->w_stride;
    p.b.values[1] = (uint8_t const *)l->w_up, p.b.stride[1] = l->w_up_stride;
    if (y.quantises) p.a.values[0] = room + y.a_at, p.a.stride[0] = y.codes_stride;
    auto const move = [&](TileSide &side, int which, uint64_t rows, uint64_t at) {
        before.add(side.values[which], side.stride[which], rows, bytes, room + at, y.moved_stride);
        side.values[which] = room + at, side.stride[which] = y.moved_stride;
    };
    if (y.moves_a) move(p.a, 0, l->height, y.a_at);
    if (y.moves_w) move(p.b, 0, l->width, y.w_at);
    if (y.moves_up) move(p.b, 1, l->width, y.up_at);
    if (mx8 && y.stages) {
        p.a.scales[0] = (uint32_t *)(room + y.a_words_at), p.b.scales[0] = (uint32_t *)(room + y.w_words_at), p.b.scales[1] = (uint32_t *)(room + y.up_words_at);
        uint32_t const blocks = (uint32_t)((l->depth + 31) / 32);
        before.add(WordsArgs {(uint8_t const *)l->w_scales, l->w_scales_stride, (uint32_t *)p.b.scales[0], p.n, blocks, p.stages, p.b.pitch});
        if (gated) before.add(WordsArgs {(uint8_t const *)l->w_up_scales, l->w_up_scales_stride, (uint32_t *)p.b.scales[1], p.n, blocks, p.stages, p.b.pitch});
        if (!y.quantises) before.add(WordsArgs {(uint8_t const *)l->a_scales, l->a_scales_stride, (uint32_t *)p.a.scales[0], p.m, blocks, p.stages, p.a.pitch});
    }
    if (int const status = launch_preparation(before, stream)) return status;
    return launch_tiles(l->w_dtype, {0, false, false, gated}, y.tiles, p, (float *)(room + y.partial_at), stream);
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
    if ((l->grad_a && too_many(y.of_a, l->height, l->depth, false)) || ((l->grad_w || l->grad_w_up) && too_many(y.of_w, l->width, l->depth, false)))
        return mx_fail("linear_backward: more results than one launch makes");
    uint8_t *const d = (uint8_t *)workspace;
    float *const column_sums = (float *)(d + y.column_sums_at), *const partial = (float *)(d + y.partial_at);
    if (some && (y.writes_d || y.sums)) {
        SlopeArgs const s = {(uint8_t const *)l->grad, gated || l->activation ? l->pre : nullptr, l->pre_up, y.writes_d ? d : nullptr, y.sums ? column_sums : nullptr, l->grad_stride,
                             l->pre_stride, y.d_stride, (uint32_t)l->height, (uint32_t)l->width, (uint32_t)y.padded, (uint32_t)y.padded, kind_of(l->grad_dtype), (uint32_t)l->activation,
                             (uint32_t)y.rows_each, gated};
        dim3 const grid((uint32_t)((y.padded + 511) / 512), (uint32_t)y.partials);
        if (l->dtype == nk_f16_k) hipLaunchKernelGGL(slope_kernel<_Float16>, grid, dim3(256), 0, stream, s);
        else hipLaunchKernelGGL(slope_kernel<__bf16>, grid, dim3(256), 0, stream, s);
        hipError_t const e = hipGetLastError();
        if (e != hipSuccess) return mx_fail(e, "slope_kernel");
    }
    if (y.sums && l->width)
        if (int const status = launch_column_sum(column_sums, y.partials, l->width, kind_of(l->bias_dtype), l->grad_bias, stream)) return status;
    uint8_t const *const of_p = y.writes_d ? d : (uint8_t const *)l->grad, *const of_q = d + y.padded * 2;
    uint64_t const d_stride = y.writes_d ? y.d_stride : l->grad_stride;
    auto const kind = kind_of(l->dtype);
    if (!some || !l->depth) { // gradients of empty sums
        for (int i = 0; i < 3; ++i) {
            uint64_t const rows = i ? l->width : l->height, stride = i == 0 ? l->grad_a_stride : i == 1 ? l->grad_w_stride : l->grad_w_up_stride;
            void *const to = i == 0 ? l->grad_a : i == 1 ? l->grad_w : l->grad_w_up;
            if (!to || !rows || !l->depth) continue;
            for (uint64_t first = 0; first < rows; first += 1u << 20) { // (a grid is at most 65535 high)
                FewArgs p = {};                                          // (no depth: zeros)
                p.m = (uint32_t)(rows - first < 1u << 20 ? rows - first : 1u << 20), p.n = (uint32_t)l->depth;
                p.e.c = (uint8_t *)to + first * stride, p.e.c_stride = stride, p.e.c_kind = kind;
                if (int const status = launch_few<__bf16, 2, 1, false, 8>(p, stream)) return status;
            }
        }
        return 0;
    }
    uint8_t const *a = (uint8_t const *)l->a, *w[2] = {(uint8_t const *)l->w, (uint8_t const *)l->w_up};
    uint64_t a_stride = l->a_stride, w_stride[2] = {l->w_stride, l->w_up_stride};
    Preparation before = {};
    auto const move = [&](uint8_t const *&values, uint64_t &stride, uint64_t rows, uint64_t at) {
        before.add(values, stride, rows, l->depth * 2, d + at, y.moved_stride);
        values = d + at, stride = y.moved_stride;
    };
    if (y.moves_a) move(a, a_stride, l->height, y.a_at);
    if (y.moves_w) move(w[0], w_stride[0], l->width, y.w_at);
    if (y.moves_up) move(w[1], w_stride[1], l->width, y.up_at);
    if (int const status = launch_preparation(before, stream)) return status;
    if (l->grad_a) { // rows of d times columns of W
        TileArgs p = {};
        p.m = (uint32_t)l->height, p.n = (uint32_t)l->depth, p.stages = (uint32_t)y.stages, p.first_stages = (uint32_t)y.first_stages;
        p.a.values[0] = of_p, p.a.stride[0] = d_stride, p.a.extent = p.m, p.a.k = (uint32_t)(y.writes_d ? y.d_stride / 2 : l->width);
        p.b = {{w[0], w[1]}, {w_stride[0], w_stride[1]}, {}, 0, p.n, (uint32_t)l->width};
        p.e.c = (uint8_t *)l->grad_a, p.e.c_stride = l->grad_a_stride, p.e.c_kind = kind;
        if (int const status = launch_tiles(l->dtype, {0, false, true, false}, y.of_a, p, partial, stream)) return status;
    }
    for (int i = 0; i < 2; ++i) { // columns of d times columns of A
        void *const to = i ? l->grad_w_up : l->grad_w;
        if (!to) continue;
        TileArgs p = {};
        p.m = (uint32_t)l->width, p.n = (uint32_t)l->depth, p.stages = p.first_stages = (uint32_t)((l->height + 63) / 64);
        p.a = {{i ? of_q : of_p}, {d_stride}, {}, 0, p.m, (uint32_t)l->height};
        p.b = {{a}, {a_stride}, {}, 0, p.n, (uint32_t)l->height};
        p.e.c = (uint8_t *)to, p.e.c_stride = i ? l->grad_w_up_stride : l->grad_w_stride, p.e.c_kind = kind;
        if (int const status = launch_tiles(l->dtype, {0, true, true, false}, y.of_w, p, partial, stream)) return status;
    }
    return 0;
}

} // extern "C"
