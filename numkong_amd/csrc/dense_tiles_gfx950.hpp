/**
 *  @brief Dense products of many rows in tiles: operands straight into LDS, both of them, results through it.
 *  @file numkong_amd/csrc/dense_tiles_gfx950.hpp
 *
 *  A workgroup of four wavefronts (two by two) makes a tile of C. A stage is 128 bytes of depth of each of its rows and columns (64 values of
 *  16 bits, 128 of 8), brought by loads that write LDS themselves, one stage on its way while another is multiplied. Two layouts of operands:
 *
 *      rows     the depth runs along a row: LDS holds rows of 128 bytes, and position p of row r the 16 bytes p ^ (r / 2 % 8), so that the
 *               lanes of a fragment, which read as many rows, meet no bank twice
 *      columns  the depth runs from row to row (the gradients' operands): LDS holds 64 rows of the tile's columns, and the reads that
 *               transpose (ds_read_b64_tr_b16: of 16 lanes, four rows of 16 columns) give each lane its column; position p of row r holds
 *               the 16 bytes p ^ 4 (r % 4), or, in rows of 64 columns, p ^ 4 (r / 2 % 2)
 *
 *  Which depth is in which place of a fragment is the same for both, 8 adjacent values a lane, so either kind meets either. Of 8-bit values the
 *  instruction takes 64 of the depth, a lane 16 of its first 32 and 16 of its second, and the scale of row or column l % 32 for block l / 32
 *  from lane l: two fragments one behind the other.
 *
 *  The products are made transposed (the matrix instruction's rows are C's columns), so that a lane has four adjacent results of one
 *  row; 64 rows at a time they go through LDS, where adjacent ones of a row come together: bias, activation and residual are
 *  added there, in 32 bits, and whole lines are written.
 *
 *  Measured: 256 x 256 bf16 8192 x 8192 x 4096 416 us (1.32 PFLOP/s), 8192^3 797 us (1.38), gated 8192 x 8192 x 4096 868 to 880 us; columns 8192 x 4096 x 4096 206 us (both operands)
 *  and 216 (one); 8 bits 8192^3 400 us (2.75). Power bounds them: matrix instructions take 65 % of the cycles at 1.6 to 1.9 GHz, waits 10 to 14 %.
 */
#ifndef NUMKONG_AMD_DENSE_TILES_GFX950_HPP
#define NUMKONG_AMD_DENSE_TILES_GFX950_HPP

#include "dense_gfx950.hpp"

namespace nk_gfx950 {

/** What becomes of a product's sums. */
struct Epilogue {
    void const *bias;
    uint8_t const *residual;
    uint8_t *c;
    float *pre, *pre_up;
    uint64_t residual_stride, c_stride, pre_stride;
    uint32_t bias_kind, residual_kind, c_kind, activation;
};

/**
 *  One operand: `extent` rows (columns) of tiles and a depth of `k`; rows 4-byte aligned and at most 2^24 bytes apart. Two addresses: the matrices of a gated product, or (columns) of two depths one behind the other. Scales of mx8: a word, four blocks, for each stage and
 *  row, [stage][pitch rows].
 */
struct TileSide {
    uint8_t const *values[2];
    uint64_t stride[2];
    uint32_t const *scales[2];
    uint32_t pitch, extent, k;
};
struct TileArgs {
    TileSide a, b;
    uint32_t m, n;
    uint32_t stages, first_stages; // all; those of the first depth, where there are two
    uint32_t splits, split_stages; // of the stages
    uint32_t tiles_m, tiles_n;
    float *partial;                // splits x (gated: 2 x) m x n sums, if there is more than one split
    Epilogue e;
};
/** Which kernel: tiles of 64, 128 or 256 rows (shape 0 to 2), the layouts, gated or not. */
struct TileForm {
    int shape;
    bool a_columns, b_columns, gated;
};
constexpr uint64_t kTileStride = 1ull << 24;

/** 8-bit values with scales. */
struct Mx8 {};
template <class T>
inline constexpr int kValueBytes = 2;
template <>
inline constexpr int kValueBytes<Mx8> = 1;

typedef short v8s __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

/** c += x y for fragments of 16-bit values: rows of c are those of x. */
template <class T>
__device__ __forceinline__ v16f multiply_32(v4u x, v4u y, v16f c) {
#ifdef NK_MX_DEVICE_BUILTINS
    if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, x), __builtin_bit_cast(v8bf, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0, 0);
#else
    return c;
#endif
}
/** The same for 64 8-bit values; byte U of the scale words. */
template <int U>
__device__ __forceinline__ v16f multiply_mx8(v4u const (&x)[2], v4u const (&y)[2], v16f c, uint32_t x_scale, uint32_t y_scale) {
#ifdef NK_MX_DEVICE_BUILTINS
    v8i const p = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], (int)x[1][0], (int)x[1][1], (int)x[1][2], (int)x[1][3]};
    v8i const q = {(int)y[0][0], (int)y[0][1], (int)y[0][2], (int)y[0][3], (int)y[1][0], (int)y[1][1], (int)y[1][2], (int)y[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(p, q, c, 0, 0, U, (int)x_scale, U, (int)y_scale);
#else
    return c;
#endif
}

constexpr uint32_t kNowhere = 0xFFFFFFF0u; // past the end of every buffer: zeros arrive
/** `bytes` from `base` on as a buffer; what is read past them is zero, four bytes at a time. */
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(uint8_t const *base, uint64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (uint32_t)(bytes < 0xFFFF0000u ? bytes : 0xFFFF0000u), 0x00020000);
}

/** What brings one operand's stages: WIDTH rows (columns) of a tile; PAIR: gated, 32 rows of the one matrix and 32 of the other in turn. */
template <class T, int WIDTH, bool COLUMNS, bool PAIR>
struct Bringer {
    static constexpr int kLoads = WIDTH / 32; // of a wavefront for a stage
    static constexpr uint32_t kEachLoad = 512 / WIDTH, kChunks = WIDTH / 8; // columns: rows of a load, 16-byte pieces of a row
    uint8_t const *base[2];
    uint64_t left[2]; // bytes from there to the end of what may be read
    uint32_t lane;    // offset of the lane in its row
    uint32_t row;     // of the lane's first load in a stage
    uint32_t beyond;  // rows: all ones where the lane's 16 bytes are past the end of the depth in its last stage
    TileSide const &side;

    __device__ __forceinline__ Bringer(TileSide const &its, uint32_t first, uint32_t wave) : side(its) {
        uint32_t const l = threadIdx.x & 63;
        if constexpr (!COLUMNS) {
            uint32_t const chunk = (l & 7) ^ ((wave * 4 + l / 16) & 7), bytes = its.k * kValueBytes<T>, tail = bytes % 128;
            row = wave * 8 + l / 8, lane = chunk * 16;
            beyond = tail && chunk * 16 >= tail ? kNowhere : 0;
#pragma unroll
            for (int i = 0; i < (PAIR ? 2 : 1); ++i) {
                base[i] = its.values[i] + first * its.stride[i];
                left[i] = (uint64_t)(its.extent - 1 - first) * its.stride[i] + (bytes + 3) / 4 * 4;
            }
        } else {
            row = wave * kEachLoad + l / kChunks, lane = ((l % kChunks) ^ swizzle(row)) * 16, beyond = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                base[i] = its.values[i] + first * 2;
                left[i] = (uint64_t)(its.k - 1) * its.stride[i] + ((uint64_t)(its.extent - first) * 2 + 3) / 4 * 4;
            }
        }
    }
    /** Columns: what row r's pieces are moved by, so that eight reads that run at one time (four rows, two times 32 bytes) meet no bank twice. */
    __device__ static __forceinline__ uint32_t swizzle(uint32_t r) { return WIDTH >= 128 ? (r & 3) * 4 : (r >> 1 & 1) * 4; }

    /** Begins to bring stage `s` (all four wavefronts bring a share) to `to`: zeros from `stages` on. */
    __device__ __forceinline__ void bring(uint8_t *to, uint32_t s, uint32_t stages, uint32_t first_stages, uint32_t wave) const {
        if constexpr (!COLUMNS) {
            uint64_t const at = (uint64_t)s * 128;
            uint32_t const nowhere = s + 1 >= stages ? beyond : 0;
#pragma unroll
            for (int which = 0; which < (PAIR ? 2 : 1); ++which) {
                __amdgpu_buffer_rsrc_t const from = buffer_of(base[which] + at, s < stages ? left[which] - at : 0);
                uint32_t const step = (uint32_t)side.stride[which];
#pragma unroll
                for (int i = which; i < kLoads; i += PAIR ? 2 : 1) {
                    uint32_t const r = row + (PAIR ? i / 2 : i) * 32;
                    fetch_16(from, to + (i * 4 + wave) * 1024, (lane + r * step) | nowhere, 0);
                }
            }
        } else {
            bool const second = s >= first_stages;
            uint32_t const k0 = (second ? s - first_stages : s) * 64;
            uint64_t const stride = second ? side.stride[1] : side.stride[0], at = k0 * stride;
            __amdgpu_buffer_rsrc_t const from = buffer_of((second ? base[1] : base[0]) + at, s < stages ? (second ? left[1] : left[0]) - at : 0);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint32_t const r = row + i * 4 * kEachLoad;
                fetch_16(from, to + (i * 4 + wave) * 1024, k0 + r >= side.k ? kNowhere : lane + r * (uint32_t)stride, 0);
            }
        }
    }
    /** Makes zeros, in the last stage of a depth that runs along the rows, of what stands between its end and the next 16 bytes: a thread a row. */
    __device__ __forceinline__ void clear_tail(uint8_t *at) const {
        if constexpr (!COLUMNS) {
            uint32_t const tail = side.k * kValueBytes<T> % 128;
            if (tail % 16 == 0) return;
#pragma unroll
            for (uint32_t r = threadIdx.x; r < WIDTH; r += 256) {
                uint32_t *const piece = (uint32_t *)(at + r * 128 + ((tail / 16) ^ (r / 2 & 7)) * 16);
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    uint32_t const from = tail % 16;
                    if (from <= i * 4) piece[i] = 0;
                    else if (from < i * 4 + 4) piece[i] &= (1u << (from % 4 * 8)) - 1;
                }
            }
        }
    }
    /** 16 bytes of step `j` of the stage at `from` for rows (columns) 32 `block` and so on of the wavefront's, which begin at `begin`. */
    __device__ static __forceinline__ v4u fragment(uint8_t const *from, uint32_t begin, int block, int j) {
        uint32_t const l = threadIdx.x & 63;
        if constexpr (!COLUMNS) {
            uint32_t const at = (begin + l % 32) * 128 + (((l / 32) ^ ((l % 32) / 2 & 7)) * 16 ^ (uint32_t)j * 32);
            return *(v4u const *)(from + at + block * 4096);
        } else {
#ifdef NK_MX_DEVICE_BUILTINS
            typedef short v4s __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) v4s lds_v4s;
            uint32_t const r = 8 * (l / 32) + l % 16 / 4, chunk = begin / 8 + (l / 16 % 2) * 2 + l % 4 / 2;
            uint32_t const at = r * WIDTH * 2 + ((chunk ^ swizzle(r)) * 16 ^ (uint32_t)block * 64) + l % 2 * 8;
            v4s const low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(from + at + j * 16 * WIDTH * 2));
            v4s const high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(from + at + (j * 16 + 4) * WIDTH * 2));
            v2u const x = __builtin_bit_cast(v2u, low), y = __builtin_bit_cast(v2u, high);
            return v4u {x[0], x[1], y[0], y[1]};
#else
            return v4u {0, 0, 0, 0};
#endif
        }
    }
};

template <class T>
struct Bytes {
    typedef uint8_t type;
};
template <class T>
struct Bytes<T const> {
    typedef uint8_t const type;
};
/** Where N rows of V adjacent results lie: row `row + i step` of the matrix for i < N, of which the lane's own part, `lane` rows and `col` columns further on,
 *  is added last: all else is the same in all lanes. WHOLE: all of them are within m x n. */
template <int N, int V, bool WHOLE>
struct Rows {
    uint32_t row, step, m, lane, col, n;
    template <class T>
    __device__ __forceinline__ T *at(T *base, uint64_t stride, uint64_t of_lane, int i) const {
        typedef typename Bytes<T>::type B;
        return (T *)((B *)base + (uint64_t)(row + i * step) * stride + of_lane);
    }
    template <class T>
    __device__ __forceinline__ uint64_t of_lane(T const *, uint64_t stride) const { return lane * stride + (uint64_t)col * sizeof(T); }
    __device__ __forceinline__ bool inside(int i) const { return WHOLE || (row + i * step + lane < m && col < n); }
    __device__ __forceinline__ uint32_t end() const { return WHOLE ? ~0u : n - col; }
    template <class T>
    __device__ __forceinline__ void store(T *base, uint64_t stride, float const (&v)[N][V]) const {
        uint64_t const its = of_lane(base, stride);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (inside(i)) store_some(at(base, stride, its, i), v[i], end());
    }
    template <class T>
    __device__ __forceinline__ void load(T const *base, uint64_t stride, float (&v)[N][V]) const {
        uint64_t const its = of_lane(base, stride);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (inside(i)) load_adjacent(at(base, stride, its, i), 0, end(), v[i]);
    }
};
/** V adjacent values of a residual as they lie in memory. */
template <int V>
struct RawPiece {
    v4u words[V / 4];
    __device__ __forceinline__ void load(uint32_t kind, uint8_t const *at) {
        if (kind == kF32) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) words[i] = *(v4u_anywhere const *)(at + 16 * i);
        } else if constexpr (V == 8) words[0] = *(v4u_anywhere const *)at;
        else {
            typedef v2u __attribute__((aligned(1))) v2u_anywhere;
            v2u const half = *(v2u_anywhere const *)at;
            words[0] = v4u {half[0], half[1], 0, 0};
        }
    }
    __device__ __forceinline__ void widen_to(uint32_t kind, float (&v)[V]) const {
        if (kind == kF32) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = __uint_as_float(words[i / 4][i % 4]);
            return;
        }
        float all[8];
        if (kind == kBF16) widen<__bf16>(words[0], all);
        else widen<_Float16>(words[0], all);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = all[i];
    }
};
/** N rows of V adjacent results from their sums; `q`: gated, the other product's. `bias` and `rest`, the residual, are looked at only where there are such. */
template <bool GATED, int N, int V, bool WHOLE>
__device__ __forceinline__ void finish(Epilogue const &e, Rows<N, V, WHOLE> const &rows, float (&p)[N][V], float const (&q)[N][V], float const (&bias)[V], float const (&rest)[N][V]) {
    if (!GATED && e.bias) {
#pragma unroll
        for (int i = 0; i < N * V; ++i) p[i / V][i % V] += bias[i % V];
    }
    if (e.pre) {
        rows.store(e.pre, e.pre_stride, p);
        if (GATED) rows.store(e.pre_up, e.pre_stride, q);
    }
    activate(e.activation, p);
    if constexpr (GATED) {
#pragma unroll
        for (int i = 0; i < N * V; ++i) p[i / V][i % V] *= q[i / V][i % V];
    }
    if (!GATED && e.residual) {
#pragma unroll
        for (int i = 0; i < N * V; ++i) p[i / V][i % V] += rest[i / V][i % V];
    }
    if (e.c_kind == kF32) rows.store((float *)e.c, e.c_stride, p);
    else if (e.c_kind == kBF16) rows.store((__bf16 *)e.c, e.c_stride, p);
    else rows.store((_Float16 *)e.c, e.c_stride, p);
}
/** A residual's. */
template <int N, int V, bool WHOLE>
__device__ __forceinline__ void load_rest(Epilogue const &e, Rows<N, V, WHOLE> const &rows, float (&rest)[N][V]) {
    if (e.residual_kind == kF32) rows.load((float const *)e.residual, e.residual_stride, rest);
    else if (e.residual_kind == kBF16) rows.load((__bf16 const *)e.residual, e.residual_stride, rest);
    else rows.load((_Float16 const *)e.residual, e.residual_stride, rest);
}
/** `finish` of one row with what it needs of the bias and the residual. */
template <bool GATED>
__device__ __forceinline__ void finish(Epilogue const &e, uint32_t row, uint32_t m, uint32_t col, uint32_t n, float (&p)[1][8], float const (&q)[1][8]) {
    Rows<1, 8, false> const rows = {0, 0, m, row, col, n};
    float bias[8], rest[1][8];
    if (!GATED && e.bias) load_adjacent(e.bias_kind, e.bias, col, n, bias);
    if (!GATED && e.residual) load_rest(e, rows, rest);
    finish<GATED>(e, rows, p, q, bias, rest);
}

/** Nothing that reads or writes LDS moves across; what this wavefront has begun to load into LDS, and read from it, is there. */
__device__ __forceinline__ void arrive_and_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070); // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

/**
 *  A tile of 64 WM x 64 WN results (columns of both matrices, where gated). Loop over the stages: fragments of a step are read while the one before is
 *  multiplied; before the last step of a stage, whose fragments are in registers then, the wavefronts meet, the next stage has to be there, and the
 *  one after that is asked for into the array that has become free. TAIL: a depth along rows may end at any byte, not only at multiples of 16 (256 x 256
 *  would spill with it: their operands are moved to where it does).
 */
template <class T, int WM, int WN, bool A_COLUMNS, bool B_COLUMNS, bool GATED, bool TAIL>
__global__ __launch_bounds__(256, WM * WN > 8 ? 1 : 2) void tile_kernel(TileArgs p) {
    constexpr int kRows = 64 * WM, kColumns = 64 * WN, kValues = 128 / kValueBytes<T>;
    constexpr bool kScaled = __is_same(T, Mx8);
    constexpr int kSteps = kScaled ? 2 : 4, kParts = 4 / kSteps;
    static_assert(!GATED || WN % 2 == 0, "a wavefront has columns of both matrices");
    __shared__ __attribute__((aligned(1024))) uint8_t a0[kRows * 128], a1[kRows * 128], b0[kColumns * 128], b1[kColumns * 128];
    uint32_t const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;

    // Workgroups go to the eight XCDs in turn; each gets adjacent tiles, in bands of eight rows of tiles, so that those that run at one
    // time share their operands in its L2.
    uint32_t const tiles = p.tiles_m * p.tiles_n, xcd = blockIdx.x % 8, each = gridDim.x / 8, more = gridDim.x % 8;
    uint32_t const at = xcd * each + (xcd < more ? xcd : more) + blockIdx.x / 8;
    uint32_t const split = at / tiles, tile = at - split * tiles;
    uint32_t const band = tile / (8 * p.tiles_n), in_band = tile - band * 8 * p.tiles_n, high = p.tiles_m - band * 8 < 8 ? p.tiles_m - band * 8 : 8;
    uint32_t const row0 = (band * 8 + in_band % high) * kRows, col0 = in_band / high * (GATED ? kColumns / 2 : kColumns);
    uint32_t const begin = split * p.split_stages, end = begin + p.split_stages < p.stages ? begin + p.split_stages : p.stages;

    typedef Bringer<T, kRows, A_COLUMNS, false> A;
    typedef Bringer<T, kColumns, B_COLUMNS, GATED> B;
    A const a(p.a, row0, wave);
    B const b(p.b, col0, wave);

    v16f sum[WM][WN] = {};
    v4u x[2][WM][kParts], y[2][WN][kParts];
    uint32_t x_words[2][WM], y_words[2][WN], x_scale[WM], y_scale[WN]; // mx8: of two stages as they were read, of this one as the lane needs it
    uint32_t const a_begin = (wave & 1) * WM * 32, b_begin = (wave >> 1) * WN * 32;

    auto const bring = [&](uint8_t *to_a, uint8_t *to_b, uint32_t s, auto slot) {
        constexpr int kSlot = decltype(slot)::value;
        if constexpr (kScaled) {
            uint32_t const at = s < end ? s : end - 1; // (codes past the end are zeros)
            uint32_t const *const of_a = p.a.scales[0] + (uint64_t)at * p.a.pitch + row0 + a_begin + l % 32;
#pragma unroll
            for (int i = 0; i < WM; ++i) x_words[kSlot][i] = of_a[i * 32];
            uint64_t const of_b = (uint64_t)at * p.b.pitch + col0 + (GATED ? b_begin / 2 : b_begin) + l % 32;
#pragma unroll
            for (int i = 0; i < WN; ++i) y_words[kSlot][i] = p.b.scales[GATED ? i & 1 : 0][of_b + (GATED ? i / 2 : i) * 32];
        }
        uint32_t const stages = s < end ? p.stages : 0;
        a.bring(to_a, s, stages, p.first_stages, wave);
        b.bring(to_b, s, stages, p.first_stages, wave);
    };
    auto const clear = [&](uint8_t *at_a, uint8_t *at_b, uint32_t s) { // stage `s` is there
        if (!TAIL || s + 1 != p.stages) return;
        a.clear_tail(at_a), b.clear_tail(at_b);
        __syncthreads();
    };
    auto const read = [&](int to, uint8_t const *at_a, uint8_t const *at_b, int j) {
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
#pragma unroll
            for (int i = 0; i < WM; ++i) x[to][i][part] = A::fragment(at_a, a_begin, i, j * kParts + part);
#pragma unroll
            for (int i = 0; i < WN; ++i) y[to][i][part] = B::fragment(at_b, b_begin, i, j * kParts + part);
        }
    };
    auto const multiply = [&](auto from) { // step `from` of a stage, or one that differs from it by a multiple of two
        constexpr int kFrom = decltype(from)::value;
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
            for (int j = 0; j < WN; ++j) {
                if constexpr (kScaled) sum[i][j] = multiply_mx8<2 * kFrom>(y[kFrom][j], x[kFrom][i], sum[i][j], y_scale[j], x_scale[i]);
                else sum[i][j] = multiply_32<T>(y[kFrom][j][0], x[kFrom][i][0], sum[i][j]);
            }
    };
    // The instructions of a step in turn, reads (and what brings the next stage) between the products: left to itself, the compiler puts each read
    // right before the product that waits for it.
    auto const in_turn = [&](auto brings) {
#ifdef NK_MX_DEVICE_BUILTINS
        constexpr int kReads = kParts * (WM * (A_COLUMNS ? 2 : 1) + WN * (B_COLUMNS ? 2 : 1)), kLoads = decltype(brings)::value ? A::kLoads + B::kLoads : 0;
        constexpr int kAll = kReads | kLoads | WM * WN, kTurns = kAll % 8 == 0 ? 8 : kAll % 4 == 0 ? 4 : kAll % 2 == 0 ? 2 : 1; // (divides all three)
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, kReads / kTurns, 0);
            if constexpr (kLoads > 0) __builtin_amdgcn_sched_group_barrier(0x10, kLoads / kTurns, 0);
            __builtin_amdgcn_sched_group_barrier(0x8, WM * WN / kTurns, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
#endif
    };
    auto const stage = [&](uint8_t *at_a, uint8_t *at_b, uint8_t *next_a, uint8_t *next_b, uint32_t s, auto slot) {
        if constexpr (kScaled) { // (a step's two blocks are bytes 0 and 1, then 2 and 3; the lane's half of the wavefront says which of the two)
            constexpr int kSlot = decltype(slot)::value;
#pragma unroll
            for (int i = 0; i < WM; ++i) x_scale[i] = x_words[kSlot][i] >> (l / 32 * 8);
#pragma unroll
            for (int i = 0; i < WN; ++i) y_scale[i] = y_words[kSlot][i] >> (l / 32 * 8);
        }
        read(1, at_a, at_b, 1);
        multiply(Number<0>());
        in_turn(Number<0>());
        if constexpr (kSteps == 4) {
            read(0, at_a, at_b, 2);
            multiply(Number<1>());
            in_turn(Number<0>());
            read(1, at_a, at_b, 3);
            multiply(Number<0>());
            in_turn(Number<0>());
        }
        arrive_and_meet();
        clear(next_a, next_b, s + 1);
        read(0, next_a, next_b, 0);
        bring(at_a, at_b, s + 2, slot);
        multiply(Number<1>());
        in_turn(Number<1>());
    };

    if (begin < end) {
        bring(a0, b0, begin, Number<0>());
        arrive_and_meet();
        clear(a0, b0, begin);
        bring(a1, b1, begin + 1, Number<1>());
        read(0, a0, b0, 0);
        for (uint32_t s = begin; s < end; s += 2) { // (an odd number of stages ends with one of zeros)
            stage(a0, b0, a1, b1, s, Number<0>());
            stage(a1, b1, a0, b0, s + 1, Number<1>());
        }
    }

    // 64 rows at a time (32, if there are no more) through LDS, each wavefront in an array of its own: piece p (four results) of row r at p ^ r. A lane
    // has the same columns in all of them: eight, or four where C is of 32 bits and so written in whole lines (8192 x 8192 x 64 to f32: 82 us, and
    // 93 with eight, two stores with gaps; to bf16 72 and 57; with the sums for the gradients beside bf16 eight again, 8192 x 4096 x 4096 282 and 328).
    // Two or four rows are finished at a time.
    // (The arrays are free once every wavefront's loads into them have arrived: those of the stages past the end bring zeros.)
    arrive_and_meet();
    constexpr int kHigh = WM < 2 ? WM : 2;
    constexpr uint32_t kWidth = WN * 32, kPieces = kWidth / 4, kOut = GATED ? kWidth / 2 : kWidth; // kOut: results of a row
    float *const room = (float *)(wave == 0 ? a0 : wave == 1 ? a1 : wave == 2 ? b0 : b1);
    uint32_t const out0 = col0 + (GATED ? b_begin / 2 : b_begin);
    bool const last = p.splits == 1;
    auto const put = [&](int i, auto from) {
        constexpr int kFrom = decltype(from)::value;
        uint32_t const r = l % 32;
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int t = 0; t < 4; ++t)
                *(v4f *)(room + (i * 32 + r) * kWidth + ((j * 8 + t * 2 + l / 32) ^ (r % kPieces)) * 4) =
                    v4f {sum[kFrom][j][4 * t], sum[kFrom][j][4 * t + 1], sum[kFrom][j][4 * t + 2], sum[kFrom][j][4 * t + 3]};
    };
    auto const finish_part = [&](auto values, auto whole, auto part, uint32_t first) __attribute__((always_inline)) {
        constexpr int V = decltype(values)::value;
        constexpr bool kWhole = decltype(whole)::value != 0;
        constexpr uint32_t kLanes = kOut / V, kStep = 64 / kLanes, kTurns = kHigh * 32 / kStep, kAhead = !kWhole ? 1 : kTurns < 16 / V ? kTurns : 16 / V;
        uint32_t const c = l % kLanes * V, col = out0 + c, piece = (GATED ? c / 32 * 64 + c % 32 : c) / 4;
        float bias[V];
        if (!GATED && last && p.e.bias && (kWhole || col < p.n)) load_adjacent(p.e.bias_kind, p.e.bias, col, p.n, bias);
        // Of whole tiles the residual is asked for before the sums are put down, eight groups of rows (of 32-bit results four) ahead.
        bool const rests = !GATED && last && p.e.residual;
        constexpr int kRing = !kWhole || GATED ? 1 : V == 8 ? 8 : 4;
        RawPiece<V> ring[kRing][kAhead];
        auto const ask = [&](uint32_t turn, RawPiece<V> (&to)[kAhead]) {
            uint64_t const of_lane = l / kLanes * p.e.residual_stride + (uint64_t)col * bytes_of(p.e.residual_kind);
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) to[i].load(p.e.residual_kind, p.e.residual + (uint64_t)(first + (turn + i) * kStep) * p.e.residual_stride + of_lane);
        };
        if (kRing > 1 && rests) {
#pragma unroll
            for (int i = 0; i < kRing; ++i)
                if (i * kAhead < kTurns) ask(i * kAhead, ring[i]);
        }
        put(0, Number<decltype(part)::value * kHigh>());
        if constexpr (kHigh > 1) put(1, Number<decltype(part)::value * kHigh + 1>());
        wave_fence();
#pragma unroll 1
        for (uint32_t turn = 0; turn < kTurns; turn += kAhead) {
            Rows<kAhead, V, kWhole> const rows = {first + turn * kStep, kStep, p.m, l / kLanes, col, p.n};
            float rest[kAhead][V], v[kAhead][V], q[kAhead][V];
            if (rests) {
                if constexpr (kRing > 1) {
#pragma unroll
                    for (uint32_t i = 0; i < kAhead; ++i) {
                        ring[0][i].widen_to(p.e.residual_kind, rest[i]);
#pragma unroll
                        for (int j = 0; j + 1 < kRing; ++j) ring[j][i] = ring[j + 1][i];
                    }
                    if (turn + kRing * kAhead < kTurns) ask(turn + kRing * kAhead, ring[kRing - 1]);
                } else load_rest(p.e, rows, rest);
            }
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) {
                uint32_t const r = turn * kStep + l / kLanes + i * kStep;
#pragma unroll
                for (uint32_t t = 0; t < V / 4; ++t) {
                    v4f const four = *(v4f const *)(room + r * kWidth + ((piece + t) ^ (r % kPieces)) * 4);
                    v[i][4 * t] = four[0], v[i][4 * t + 1] = four[1], v[i][4 * t + 2] = four[2], v[i][4 * t + 3] = four[3];
                    if constexpr (GATED) {
                        v4f const its = *(v4f const *)(room + r * kWidth + ((piece + 8 + t) ^ (r % kPieces)) * 4);
                        q[i][4 * t] = its[0], q[i][4 * t + 1] = its[1], q[i][4 * t + 2] = its[2], q[i][4 * t + 3] = its[3];
                    }
                }
            }
            if (last) finish<GATED>(p.e, rows, v, q, bias, rest);
            else {
                float *const to = p.partial + (uint64_t)split * (GATED ? 2 : 1) * p.m * p.n;
                rows.store(to, (uint64_t)p.n * 4, v);
                if (GATED) rows.store(to + (uint64_t)p.m * p.n, (uint64_t)p.n * 4, q);
            }
        }
    };
    auto const finish_rows = [&](auto part, uint32_t first) __attribute__((always_inline)) {
        bool const whole = first + kHigh * 32 <= p.m && out0 + kOut <= p.n;
        if (!whole) finish_part(Number<4>(), Number<0>(), part, first);
        else if (!last || p.e.c_kind == kF32) finish_part(Number<4>(), Number<1>(), part, first);
        else finish_part(Number<8>(), Number<1>(), part, first);
        wave_fence();
    };
    uint32_t const first = row0 + a_begin;
    if (first >= p.m) return;
    finish_rows(Number<0>(), first);
    if constexpr (WM > kHigh) {
        if (first + kHigh * 32 < p.m) finish_rows(Number<1>(), first + kHigh * 32);
    }
}

/** Queues the kernel of a form; the grid is a workgroup for each tile and split. */
template <class T, int WM, int WN, bool A_COLUMNS, bool B_COLUMNS, bool GATED, bool TAIL>
int launch_tile(TileArgs const &p, hipStream_t stream) {
    hipLaunchKernelGGL((tile_kernel<T, WM, WN, A_COLUMNS, B_COLUMNS, GATED, TAIL>), dim3(p.tiles_m * p.tiles_n * p.splits), dim3(256), 0, stream, p);
    hipError_t const e = hipGetLastError();
    return e == hipSuccess ? 0 : mx_fail(e, "tile_kernel");
}
template <class T, bool A_COLUMNS, bool B_COLUMNS, bool GATED, bool TAIL>
int launch_shape(int shape, TileArgs const &p, hipStream_t stream) {
    if (shape == 0) return launch_tile<T, 1, GATED ? 2 : 1, A_COLUMNS, B_COLUMNS, GATED, TAIL>(p, stream);
    if (shape == 1) return launch_tile<T, 2, 2, A_COLUMNS, B_COLUMNS, GATED, TAIL>(p, stream);
    if constexpr (TAIL) return mx_fail("tile_kernel: no such form");
    else return launch_tile<T, 4, 4, A_COLUMNS, B_COLUMNS, GATED, false>(p, stream);
}
template <class T>
int launch_tiles_of(TileForm const &f, TileArgs const &p, hipStream_t stream) {
    if (!f.b_columns) {
        bool const tail = p.a.k * kValueBytes<T> % 16 || p.b.k * kValueBytes<T> % 16;
        if (f.gated) return tail ? launch_shape<T, false, false, true, true>(f.shape, p, stream) : launch_shape<T, false, false, true, false>(f.shape, p, stream);
        return tail ? launch_shape<T, false, false, false, true>(f.shape, p, stream) : launch_shape<T, false, false, false, false>(f.shape, p, stream);
    }
    if constexpr (!__is_same(T, Mx8)) return f.a_columns ? launch_shape<T, true, true, false, false>(f.shape, p, stream) : launch_shape<T, false, true, false, false>(f.shape, p, stream);
    return mx_fail("tile_kernel: no such form");
}
int launch_tiles_bf16(TileForm const &, TileArgs const &, hipStream_t);
int launch_tiles_f16(TileForm const &, TileArgs const &, hipStream_t);
int launch_tiles_mx8(TileForm const &, TileArgs const &, hipStream_t);

} // namespace nk_gfx950

#endif // NUMKONG_AMD_DENSE_TILES_GFX950_HPP
