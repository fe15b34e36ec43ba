/**
 *  @brief Routing to experts on gfx950: the choice, its gradient, the plan of the products.
 *  @file numkong_amd/csrc/experts_gfx950.hip
 *
 *  Implements the experts half of <numkong_amd/mx.h> but for the products (mx_gfx950.hip).
 */
#include "mx_gfx950.hpp"

namespace nk_gfx950 {
namespace {

// ---- reductions over a wavefront ----------------------------------------------------------------------------------

/** The value of the lane that stands across: in pairs, fours, eights (within each the same already), sixteens and so on, for
 *  reductions whose every lane gets the result. Moves within 16 lanes come with the instruction that uses them, others are
 *  swaps of rows: a maximum over the wavefront costs six instructions (and six round trips to LDS by shuffles). */
template <int STEP>
__device__ __forceinline__ v2u swapped(uint32_t x) { // what the lower and the upper of two rows (halves) of lanes hold
#ifdef NK_MX_DEVICE_BUILTINS
    auto const both = STEP == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false) : __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return v2u {both[0], both[1]};
#else
    return v2u {x, x};
#endif
}
template <int STEP>
__device__ __forceinline__ uint32_t across(uint32_t x) {
#ifdef NK_MX_DEVICE_BUILTINS
    if constexpr (STEP == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true);       // lanes 1 0 3 2
    else if constexpr (STEP == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true);  // lanes 2 3 0 1
    else if constexpr (STEP == 4) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, true); // eights mirrored
    else if constexpr (STEP == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xF, 0xF, true); // sixteens mirrored
    else {
        v2u const both = swapped<STEP>(x);
        return threadIdx.x & STEP ? both[0] : both[1];
    }
#else
    return x;
#endif
}
/** `join` of what two lanes that stand across hold, in both. */
template <int STEP, class F>
__device__ __forceinline__ uint32_t joined(uint32_t x, F &&join) {
    if constexpr (STEP < 16) return join(x, across<STEP>(x));
    else {
        v2u const both = swapped<STEP>(x);
        return join((uint32_t)both[0], (uint32_t)both[1]);
    }
}
/** `join` over groups of `lanes` (a power of two) adjacent lanes. */
template <class F>
__device__ __forceinline__ void reduce_steps(uint32_t lanes, F &&join) {
    if (lanes > 1) join(Number<1>());
    if (lanes > 2) join(Number<2>());
    if (lanes > 4) join(Number<4>());
    if (lanes > 8) join(Number<8>());
    if (lanes > 16) join(Number<16>());
    if (lanes > 32) join(Number<32>());
}
template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
    auto const sum = [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); };
    uint32_t bits = __float_as_uint(x);
    reduce_steps(L, [&](auto step) __attribute__((always_inline)) { bits = joined<decltype(step)::value>(bits, sum); });
    return __uint_as_float(bits);
}
template <int L>
__device__ __forceinline__ float lanes_max(float x) {
    auto const most = [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); };
    uint32_t bits = __float_as_uint(x);
    reduce_steps(L, [&](auto step) __attribute__((always_inline)) { bits = joined<decltype(step)::value>(bits, most); });
    return __uint_as_float(bits);
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
    reduce_steps(L, [&](auto step) __attribute__((always_inline)) { x = joined<decltype(step)::value>(x, larger); });
    return x;
}
/** The lowest of L lanes for which `is` holds; L and more where it does for none. */
template <int L>
__device__ __forceinline__ uint32_t first_lane(bool is) {
    uint64_t const all = __ballot(is);
    if constexpr (L == 64) return all ? (uint32_t)__builtin_ctzll(all) : 64u;
    else return (uint32_t)__builtin_ctz(((uint32_t)(all >> (threadIdx.x & 63 & ~(L - 1))) & ((1u << L) - 1)) | 1u << L);
}
/** Numbers in the order of unsigned integers: larger number, larger key; every NaN above them all, both zeros the same.
 *  Zero is below every key: what is taken already. */
__device__ __forceinline__ uint32_t key_of(float x) {
    uint32_t const bits = __float_as_uint(x + 0.0f), key = bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
    return x != x ? 0xFFFFFFFFu : key;
}
constexpr uint32_t kMaskedKey = 0x007FFFFFu; // of -inf

__device__ __forceinline__ float number_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

/** What one lane holds of a row: experts lane * J ... lane * J + J - 1, -inf past the end. */
template <class T, int J>
__device__ __forceinline__ void load_row(T const *row, uint32_t lane, uint32_t experts, float (&l)[J]) {
    if (lane * J + J <= experts) {
        struct __attribute__((packed, aligned(sizeof(T)))) Several {
            T x[J];
        } several;
        __builtin_memcpy(&several, row + lane * J, sizeof(several));
#pragma unroll
        for (int j = 0; j < J; ++j) l[j] = (float)several.x[j];
        return;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        uint32_t const e = lane * J + j;
        l[j] = e < experts ? (float)row[e] : -__builtin_inff();
    }
}

template <class T, int J>
__device__ __forceinline__ void store_row(T *row, uint32_t lane, uint32_t experts, float const (&l)[J]) {
    if (lane * J + J <= experts) {
        struct __attribute__((packed, aligned(sizeof(T)))) Several {
            T x[J];
        } several;
#pragma unroll
        for (int j = 0; j < J; ++j) several.x[j] = (T)l[j];
        __builtin_memcpy(row + lane * J, &several, sizeof(several));
        return;
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
        if (lane * J + j < experts) row[lane * J + j] = (T)l[j];
}

/** What scores are made of besides the logit: the row's largest logit and the sum of exponentials (softmax). */
struct ScoreOf {
    int sigmoid;
    float top, sum;
    template <int J>
    __device__ __forceinline__ void operator()(float const (&l)[J], float (&s)[J]) const {
        if (sigmoid) {
#pragma unroll
            for (int j = 0; j < J; ++j) s[j] = 1.0f / (1.0f + expf(-l[j]));
            return;
        }
#pragma unroll
        for (int j = 0; j < J; ++j) { // -inf has score 0, also where the whole row is -inf
            float const e = expf(l[j] - top);
            s[j] = l[j] == -__builtin_inff() || e == 0.0f ? 0.0f : e / sum;
        }
    }
};
template <int L, int J>
__device__ __forceinline__ ScoreOf score_of_row(float const (&l)[J], int sigmoid) {
    if (sigmoid) return {sigmoid, 0.0f, 0.0f};
    float top = l[0];
#pragma unroll
    for (int j = 1; j < J; ++j) top = fmaxf(top, l[j]);
    top = lanes_max<L>(top);
    float sum = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        float const e = expf(l[j] - top);
        sum += l[j] == -__builtin_inff() ? 0.0f : e;
    }
    return {sigmoid, top, lanes_sum<L>(sum)};
}

/** Takes the largest key of L lanes out, the first of equal ones: its place in the lane that held it, -1 in others and where
 *  none is above `floor`. */
template <int L, int J>
__device__ __forceinline__ int take_largest(uint32_t (&key)[J], uint32_t lane, uint32_t floor, bool &any) {
    uint32_t mine = key[0];
#pragma unroll
    for (int j = 1; j < J; ++j) mine = larger(mine, key[j]);
    uint32_t const top = lanes_max<L>(mine);
    any = top > floor;
    bool here = first_lane<L>(mine == top) == lane && any;
    int at = -1;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        bool const hit = here && key[j] == top;
        at = hit ? j : at, key[j] = hit ? 0u : key[j], here = here && !hit;
    }
    return at;
}

struct RouteArgs {
    void const *logits;
    uint64_t stride;
    uint32_t tokens, experts, top_k;
    float const *bias;
    nk_amd_route_t how;
    float *weights;
    int32_t *chosen;
};

/**
 *  L lanes for a token: its row stays in registers, J experts a lane, adjacent ones, so that of equal keys the lowest lane's
 *  lowest is the lowest expert. A choice is a maximum over each lane's keys and over the lanes; the lane that holds it takes it
 *  out and notes it. What bounds this is the number of instructions, which 16 lanes to a token share among four of them, and for few
 *  tokens the time that they take one after the other (with_row). 16,384 tokens of 256 experts, sigmoid and bias, 4 of 8 groups,
 *  8 chosen: 14.6 us, at 3 us for the traffic; 8192 tokens of 128 experts, 8 chosen: 5.5 us. Groups of whole lanes are found in
 *  registers, others through LDS (the same 16,384 tokens through LDS, a lane for four groups: 23.6 us).
 */
template <class T, int L, int J>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs p) {
    constexpr uint32_t kTokens = 256 / L;
    constexpr int kOfLane = 64 / L; // groups, and choices, that a lane looks after
    __shared__ uint32_t keys[kTokens][L * J];
    __shared__ int32_t notes[kTokens][64];
    uint32_t const lane = threadIdx.x % L, local = threadIdx.x / L, token = blockIdx.x * kTokens + local;
    if (token >= p.tokens) return; // (with all lanes that it exchanges anything with)
    T const *const row = (T const *)((uint8_t const *)p.logits + token * p.stride);
    float l[J];
    load_row<T, J>(row, lane, p.experts, l);
    ScoreOf const score = score_of_row<L, J>(l, p.how.sigmoid);
    uint32_t key[J];
    if (p.bias) {
        float bias[J], s[J];
        load_row<float, J>(p.bias, lane, p.experts, bias);
        score(l, s);
#pragma unroll
        for (int j = 0; j < J; ++j) key[j] = key_of(l[j] == -__builtin_inff() ? l[j] : s[j] + bias[j]);
    }
    else
#pragma unroll
        for (int j = 0; j < J; ++j) key[j] = key_of(l[j]);
    bool any;
    if (p.how.groups > 1) {
        uint32_t const groups = (uint32_t)p.how.groups, size = p.experts / groups, lanes = size / J;
        bool const two = p.how.group_top == 2 && size > 1;
        // (a masked expert adds nothing to its group, and a group with one that can be chosen stands before those without, also where
        // a sum of the lowest numbers overflows: what cannot be chosen never keeps out what can)
        auto const group_key = [&](uint32_t first, uint32_t second) {
            return two && second > kMaskedKey ? larger(key_of(number_of(first) + number_of(second)), kMaskedKey + 1) : first;
        };
        auto const best_two = [&](uint32_t lanes, uint32_t &first, uint32_t &second) __attribute__((always_inline)) { // of adjacent lanes, in all
            reduce_steps(lanes, [&](auto step) __attribute__((always_inline)) {
                uint32_t const other = across<decltype(step)::value>(first), next = across<decltype(step)::value>(second);
                uint32_t const lesser = other < first ? other : first;
                first = larger(first, other), second = larger(larger(second, next), lesser);
            });
        };
        if (size % J == 0 && (lanes & (lanes - 1)) == 0) { // a group is some whole lanes, side by side, and stays in registers
            uint32_t first = key[0], second = 0;
#pragma unroll
            for (int j = 1; j < J; ++j) {
                uint32_t const lesser = key[j] < first ? key[j] : first;
                first = larger(first, key[j]), second = larger(second, lesser);
            }
            best_two(lanes, first, second);
            uint32_t mine = lane >= groups * lanes ? 0 : group_key(first, second);
            bool stays = false;
            for (int i = 0; i < p.how.top_groups; ++i)
                if ((lane ^ first_lane<L>(mine == lanes_max<L>(mine))) < lanes) stays = true, mine = 0;
#pragma unroll
            for (int j = 0; j < J; ++j) key[j] = stays ? key[j] : kMaskedKey;
        }
        else { // the keys go through LDS, and some lanes (or one, which may have several groups) find the best of each group
            uint32_t const per_lane = (groups + L - 1) / L;
            uint32_t share = 1;
            while (share * 2 * groups <= L) share *= 2;
            uint32_t const part = lane & (share - 1);
#pragma unroll
            for (int j = 0; j < J; ++j) keys[local][lane * J + j] = key[j];
            wave_fence();
            uint32_t of_group[kOfLane], stay = 0;
#pragma unroll
            for (int q = 0; q < kOfLane; ++q) {
                uint32_t const group = lane / share * per_lane + q;
                bool const has = q < per_lane && group < groups;
                uint32_t first = 0, second = 0;
                of_group[q] = 0;
                if (q >= per_lane) continue;
#pragma unroll 4
                for (uint32_t i = part; has && i < size; i += share) {
                    uint32_t const k = keys[local][group * size + i], lesser = k < first ? k : first;
                    first = larger(first, k), second = larger(second, lesser);
                }
                best_two(share, first, second);
                if (has && part == 0) of_group[q] = group_key(first, second);
            }
            for (int i = 0; i < p.how.top_groups; ++i) {
                int const at = take_largest<L, kOfLane>(of_group, lane, 0u, any);
                stay |= at < 0 ? 0u : 1u << at;
            }
#pragma unroll
            for (int q = 0; q < kOfLane; ++q)
                if (q < per_lane && part == 0 && lane / share * per_lane + q < 64) notes[local][lane / share * per_lane + q] = (int32_t)(stay >> q & 1);
            wave_fence();
            uint32_t group = lane * J / size, left = size - (lane * J - group * size);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (group >= groups || !notes[local][group]) key[j] = kMaskedKey;
                if (--left == 0) left = size, ++group;
            }
            wave_fence();
        }
    }
    for (uint32_t i = 0; i < p.top_k; ++i) {
        int const at = take_largest<L, J>(key, lane, kMaskedKey, any);
        if (any ? at >= 0 : lane == 0) notes[local][i] = any ? (int32_t)(lane * J) + at : -1;
    }
    wave_fence();
    float weight[kOfLane], sum = 0;
    int32_t chosen[kOfLane];
#pragma unroll
    for (int q = 0; q < kOfLane; ++q) {
        uint32_t const i = q * L + lane;
        chosen[q] = -1, weight[q] = 0;
        if (q * L >= p.top_k) continue;
        if (i < p.top_k) chosen[q] = notes[local][i];
        float const its[1] = {chosen[q] < 0 ? -__builtin_inff() : (float)row[chosen[q]]}; // (-inf: of both kinds the score is 0)
        float of_it[1];
        score(its, of_it);
        weight[q] = of_it[0], sum += weight[q];
    }
    if (p.how.renormalize) sum = lanes_sum<L>(sum) + 1e-20f;
#pragma unroll
    for (int q = 0; q < kOfLane; ++q) {
        uint32_t const i = q * L + lane;
        if (i >= p.top_k) continue;
        if (p.how.renormalize) weight[q] /= sum;
        p.weights[(uint64_t)token * p.top_k + i] = chosen[q] < 0 ? 0.0f : weight[q] * p.how.scale;
        p.chosen[(uint64_t)token * p.top_k + i] = chosen[q];
    }
}

/**
 *  With s the scores, S the chosen, D = sum_S s + 1e-20:  ds_j = scale (g_j - sum_S g s / D) / D where weights are
 *  renormalised, scale g_j where not, 0 outside S; then dl_j = ds_j s_j (1 - s_j) for sigmoid scores, and
 *  dl_i = s_i (ds_i - sum_S ds s) for softmax. Not its bytes bound it (8192 tokens of 128 experts in bf16: 5.7 us for 4.2 MB) but one
 *  token's work after the other: two wavefronts to a SIMD, 711 vector instructions in each, 57 % of whose time is waiting for loads and LDS.
 */
template <class T, int L, int J>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteArgs p, float const *grad, T *out, uint64_t out_stride) {
    constexpr uint32_t kTokens = 256 / L;
    __shared__ uint32_t choice_of[kTokens][L * J]; // of each expert, 1 for the first; 0: it was not chosen
    __shared__ float grads[kTokens][64];
    uint32_t const lane = threadIdx.x % L, local = threadIdx.x / L, token = blockIdx.x * kTokens + local;
    if (token >= p.tokens) return; // (with all lanes that it exchanges anything with)
    float l[J], s[J], g[J];
    load_row<T, J>((T const *)((uint8_t const *)p.logits + token * p.stride), lane, p.experts, l);
#pragma unroll
    for (int j = 0; j < J; ++j) choice_of[local][lane * J + j] = 0;
    wave_fence();
    for (uint32_t i = lane; i < p.top_k; i += L) {
        uint32_t const e = (uint32_t)p.chosen[(uint64_t)token * p.top_k + i];
        grads[local][i] = grad[(uint64_t)token * p.top_k + i];
        if (e < p.experts) choice_of[local][e] = i + 1;
    }
    ScoreOf const score = score_of_row<L, J>(l, p.how.sigmoid);
    wave_fence();
    bool in[J];
    float total = 0, along = 0;
    score(l, s);
#pragma unroll
    for (int j = 0; j < J; ++j) {
        uint32_t const choice = choice_of[local][lane * J + j];
        in[j] = choice != 0, g[j] = in[j] ? grads[local][choice - 1] : 0.0f;
        if (in[j]) total += s[j], along += g[j] * s[j];
    }
    total = lanes_sum<L>(total) + 1e-20f, along = lanes_sum<L>(along);
    float ds[J], inner = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        ds[j] = !in[j] ? 0.0f : p.how.scale * (p.how.renormalize ? (g[j] - along / total) / total : g[j]);
        inner += in[j] ? ds[j] * s[j] : 0.0f;
    }
    inner = lanes_sum<L>(inner);
#pragma unroll
    for (int j = 0; j < J; ++j) {
        // (1 - s of a sigmoid is the score of the opposite logit, without its cancellation)
        float const slope = p.how.sigmoid ? (in[j] ? ds[j] * s[j] / (1.0f + expf(l[j])) : 0.0f) : s[j] * (ds[j] - inner);
        g[j] = l[j] == -__builtin_inff() ? 0.0f : slope;
    }
    store_row<T, J>((T *)((uint8_t *)out + token * out_stride), lane, p.experts, g);
}

// ---- the plan -----------------------------------------------------------------------------------------------------

constexpr int kPlanWaves = 4, kPlanThreads = 64 * kPlanWaves;
static_assert(kPlanBlockSlots == 4 * kPlanThreads, "what plan_geometry leaves room for");
/** So many workgroups of plan_kernel add up one another's counts themselves; of more a launch of its own does, whose time grows with the
 *  slots and not with their square (whole plans, us, by themselves and by that launch: 2^15 slots of 128 experts 10.0 and 11.8, 2^16 11.4 and
 *  12.4, 2^17 14.4 and 12.7, 2^18 20.2 and 13.7; of 1,024 experts 20.7 and 19.9, 27.5 and 21.3, 41.7 and 22.0, 69.5 and 23.8). 2^20 slots
 *  take 20 us and 37. */
constexpr uint32_t kPlanCountBlocks = 64;
/** Lanes of the wavefront that hold the same bucket, by one ballot for each bit. */
__device__ __forceinline__ uint64_t same_bucket(uint32_t bucket, int bits, bool active) {
    uint64_t mask = __ballot(active);
    for (int bit = 0; bit < bits; ++bit) {
        bool const set = bucket >> bit & 1;
        uint64_t const with = __ballot(active && set);
        mask &= set ? with : ~with;
    }
    return mask;
}

/** The slots of one lane: `BATCH` of its wavefront's stretch of 64 BATCH, which starts at `begin`; `experts` for none. */
template <int BATCH>
__device__ __forceinline__ void load_stretch(int32_t const *chosen, uint32_t begin, uint32_t slots, uint32_t experts, uint32_t (&mine)[BATCH]) {
    uint32_t const lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) mine[i] = begin + i * 64 + lane < slots ? (uint32_t)chosen[begin + i * 64 + lane] : 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) mine[i] = mine[i] < experts ? mine[i] : experts;
}

/** How many slots of each bucket each workgroup of plan_kernel will have: table[workgroup][bucket]. */
__global__ __launch_bounds__(kPlanThreads) void plan_count_kernel(int32_t const *chosen, uint32_t slots, uint32_t experts, uint32_t *table) {
    extern __shared__ uint32_t plan_lds[];
    constexpr int BATCH = 4;
    uint32_t const buckets = experts + 1, lane = threadIdx.x & 63, begin = (blockIdx.x * kPlanWaves + (threadIdx.x >> 6)) * 64 * BATCH;
    uint32_t mine[BATCH];
    load_stretch(chosen, begin, slots, experts, mine);
    for (uint32_t i = threadIdx.x; i < buckets; i += kPlanThreads) plan_lds[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
        if (begin + i * 64 + lane < slots) atomicAdd(plan_lds + mine[i], 1u);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < buckets; i += kPlanThreads) table[blockIdx.x * buckets + i] = plan_lds[i];
}

constexpr uint32_t kScanBuckets = 16, kScanParts = 64, kScanBatch = 8;
/**
 *  Of each bucket's counts in `table` the sums over the workgroups before each, and over all of them in the row behind the last, so that a
 *  workgroup of plan_kernel reads two words for a bucket however many there are. A workgroup takes 16 adjacent buckets; of a
 *  bucket's column each of 64 threads adds up one stretch, learns from LDS what stands before it, and goes over it again.
 */
__global__ __launch_bounds__(kScanBuckets * kScanParts) void plan_scan_kernel(uint32_t buckets, uint32_t blocks, uint32_t *table) {
    __shared__ uint32_t sums[kScanParts][kScanBuckets];
    uint32_t const column = threadIdx.x % kScanBuckets, part = threadIdx.x / kScanBuckets, bucket = blockIdx.x * kScanBuckets + column;
    uint32_t const stretch = (blocks + kScanParts - 1) / kScanParts, from = part * stretch < blocks ? part * stretch : blocks;
    uint32_t const to = bucket >= buckets ? from : from + stretch < blocks ? from + stretch : blocks;
    uint32_t sum = 0;
#pragma unroll 8
    for (uint32_t at = from; at < to; ++at) sum += table[at * buckets + bucket];
    sums[part][column] = sum;
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t earlier = 0; earlier < part; ++earlier) before += sums[earlier][column];
    for (uint32_t at = from; at < to; at += kScanBatch) {
        uint32_t its[kScanBatch];
#pragma unroll
        for (uint32_t i = 0; i < kScanBatch; ++i) its[i] = at + i < to ? table[(at + i) * buckets + bucket] : 0;
#pragma unroll
        for (uint32_t i = 0; i < kScanBatch; ++i) {
            if (at + i < to) table[(at + i) * buckets + bucket] = before;
            before += its[i];
        }
    }
    if (part == kScanParts - 1 && bucket < buckets) table[blocks * buckets + bucket] = before;
}

/**
 *  Counting sort of the slots by expert. A wavefront has a stretch of them in registers; it counts them, learns where its slots
 *  of each bucket go (behind those of the wavefronts before it, whose counts are in LDS, and of the workgroups before, in
 *  `table`; NULL where there is one workgroup), and goes over them again in order, so that no atomic decides an order. `scanned`:
 *  the table holds sums (plan_scan_kernel), not counts. The first workgroup also writes the header and the slots of rows that
 *  stand between experts; the tiles are written by all in turn, as one expert may have most of them. Its time is that of a few loads
 *  and LDS round trips one after the other: 32 slots 3.6 us, 1,024 5.5, 4,004 6.1 and the launch that counts 2.0, 32,768 7.3 and 2.6,
 *  2^20 11.1, 3.7 and the sums 6.5 (back to back 8.4, 9.6 and 20).
 */
template <int BATCH, bool SCANNED>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(int32_t const *chosen, uint32_t slots, uint32_t experts, PlanHeader header,
                                                            uint32_t offsets, uint32_t order, uint32_t place, uint32_t tiles, int bits,
                                                            uint32_t const *table, uint32_t blocks, uint32_t *plan) {
    extern __shared__ uint32_t plan_lds[]; // [wave][bucket] counts, then where the wave's next slot of the bucket goes
    __shared__ uint32_t wave_total[2][kPlanWaves];
    uint32_t const buckets = experts + 1, thread = threadIdx.x, lane = thread & 63;
    uint32_t const wave = __builtin_amdgcn_readfirstlane(thread >> 6), begin = (blockIdx.x * kPlanWaves + wave) * 64 * BATCH;
    uint32_t mine[BATCH];
    load_stretch(chosen, begin, slots, experts, mine);
    for (uint32_t i = thread; i < buckets * kPlanWaves; i += kPlanThreads) plan_lds[i] = 0;
    __syncthreads();
    uint32_t *counts = plan_lds + wave * buckets;
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
        if (begin + i * 64 + lane < slots) atomicAdd(counts + mine[i], 1u);
    __syncthreads();
    uint32_t rows_before = 0, tiles_before = 0;
    for (uint32_t base = 0; base < buckets; base += kPlanThreads) { // a thread for a bucket
        uint32_t const bucket = base + thread;
        uint32_t here[kPlanWaves] = {}, size = 0, earlier = 0;
        if (bucket < buckets) {
#pragma unroll
            for (int w = 0; w < kPlanWaves; ++w) here[w] = plan_lds[w * buckets + bucket], size += here[w];
            if (SCANNED) earlier = table[blockIdx.x * buckets + bucket], size = table[blocks * buckets + bucket];
            else if (table) {
                size = 0;
#pragma unroll 8
                for (uint32_t block = 0; block < blocks; ++block) {
                    uint32_t const its = table[block * buckets + bucket];
                    size += its, earlier += block < blockIdx.x ? its : 0;
                }
            }
        }
        uint32_t const its_tiles = (size + header.tile_rows - 1) / header.tile_rows, its_rows = (size + 15) / 16 * 16;
        uint32_t rows = its_rows, tiles_upto = its_tiles; // inclusive sums over the wavefront, then over wavefronts
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) {
            uint32_t const r = (uint32_t)__shfl_up((int)rows, step), t = (uint32_t)__shfl_up((int)tiles_upto, step);
            if (lane >= (uint32_t)step) rows += r, tiles_upto += t;
        }
        if (lane == 63) wave_total[0][wave] = rows, wave_total[1][wave] = tiles_upto;
        __syncthreads();
        uint32_t first = rows_before + rows - its_rows, first_tile = tiles_before + tiles_upto - its_tiles;
#pragma unroll
        for (uint32_t w = 0; w < (uint32_t)kPlanWaves; ++w) {
            if (w < wave) first += wave_total[0][w], first_tile += wave_total[1][w];
            rows_before += wave_total[0][w], tiles_before += wave_total[1][w];
        }
        if (bucket < buckets) {
            uint32_t next = first + earlier;
#pragma unroll
            for (int w = 0; w < kPlanWaves; ++w) plan_lds[w * buckets + bucket] = next, next += here[w];
            for (uint32_t t = blockIdx.x; t < its_tiles; t += blocks) {
                uint32_t const from = first + t * header.tile_rows, to = from + header.tile_rows;
                PlanTile const tile = {(int32_t)bucket, (int32_t)from, (int32_t)(to < first + size ? to : first + size), 0};
                *(PlanTile *)(plan + tiles + (first_tile + t) * 4) = tile;
            }
            if (blockIdx.x == 0) {
                plan[offsets + bucket] = first;
                for (uint32_t at = first + size; at < first + its_rows; ++at) plan[order + at] = 0xFFFFFFFFu;
                if (bucket == experts) {
                    header.tile_count = first_tile, header.zero_tiles = its_tiles;
                    header.first_zero = first, header.end_zero = first + size;
                    plan[offsets + buckets] = first + size;
                    *(PlanHeader *)plan = header;
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
        uint32_t const at = begin + i * 64 + lane, bucket = mine[i];
        if (begin + i * 64 >= slots) break;
        bool const active = at < slots;
        uint64_t const same = same_bucket(bucket, bits, active);
        uint32_t const rank = (uint32_t)__popcll(same & ((1ull << lane) - 1));
        if (active) {
            uint32_t const row = counts[bucket] + rank;
            plan[order + row] = at;
            plan[place + at] = bucket < experts ? row : 0xFFFFFFFFu;
        }
        wave_fence(); // (every lane has read its count before the first of each bucket moves it on)
        if (active && !rank) counts[bucket] += (uint32_t)__popcll(same);
        wave_fence();
    }
}

int check_route(nk_dtype_t dtype, void const *logits, nk_size_t stride, nk_size_t tokens, nk_size_t experts, nk_size_t top_k,
                nk_amd_route_t const *how) {
    int const bytes = dtype == nk_f32_k ? 4 : dtype == nk_bf16_k || dtype == nk_f16_k ? 2 : 0;
    if (!bytes) return mx_fail("experts_route: logits have to be f32, bf16 or f16");
    if (!how) return mx_fail("experts_route: NULL operand");
    if (!experts || experts > kMaxExperts || !top_k || top_k > kMaxTopK || top_k > experts) return mx_fail("experts_route: 1 to 1024 experts, top_k at most 64 and no more than there are");
    if (tokens >= (1ull << 31)) return mx_fail("experts_route: too many tokens");
    if (how->groups < 1 || how->groups > (int)kMaxGroups || experts % how->groups || how->top_groups < 1 || how->top_groups > how->groups ||
        how->group_top < 1 || how->group_top > 2)
        return mx_fail("experts_route: groups have to divide the experts, at most 64, top_groups 1 to groups, group_top 1 or 2");
    if (tokens && (!logits || (((uintptr_t)logits | stride) & (bytes - 1)))) return mx_fail("experts_route: logits are NULL or not aligned to their elements");
    return 0;
}

/**
 *  Calls `f` with a value of the logits' type, and with how many lanes a token has and how many experts a lane holds. A wavefront
 *  for a token (`wide`) is done sooner, 16 lanes take fewer instructions in all: with 64 lanes and with 16, 128 experts took 3.6 and
 *  4.5 us for up to 1,024 tokens, 4.2 and 4.7 for 2,048, 5.3 and 4.9 for 4,096, 12.7 and 8.3 for 16,384; 256 experts in groups 4.4 and 6.1,
 *  4.9 and 6.2, 6.5 and 6.3, 17.1 and 13.3. The gradient, 128 experts: 2.5 and 3.9, 3.0 and 4.0, 3.9 and 4.2, 8.7 and 7.5; 256 experts:
 *  3.1 and 6.8, 3.5 and 6.9, 4.6 and 7.5, 12.6 and 14.6, so there a wavefront it is for any number. (Up to 64 experts: no difference.)
 */
template <bool ALL_WIDE_PAST_128, class F>
int with_row(nk_dtype_t dtype, bool wide, size_t experts, F &&f) {
    auto const of_type = [&](auto value) {
        if (experts <= 64) return f(value, Number<16>(), Number<4>());
        if (experts <= 128) return wide ? f(value, Number<64>(), Number<2>()) : f(value, Number<16>(), Number<8>());
        if constexpr (!ALL_WIDE_PAST_128)
            if (experts <= 256 && !wide) return f(value, Number<16>(), Number<16>());
        if (experts <= 256) return f(value, Number<64>(), Number<4>());
        if (experts <= 512) return f(value, Number<64>(), Number<8>());
        return f(value, Number<64>(), Number<16>());
    };
    if (dtype == nk_f32_k) return of_type(float());
    if (dtype == nk_bf16_k) return of_type(__bf16());
    return of_type(_Float16());
}

} // namespace
} // namespace nk_gfx950

using namespace nk_gfx950;

extern "C" {

int nk_amd_experts_route_async(nk_dtype_t dtype, void const *logits, nk_size_t logits_stride, nk_size_t tokens, nk_size_t experts,
                               nk_size_t top_k, float const *bias, nk_amd_route_t const *how, float *weights, nk_i32_t *chosen,
                               void *stream) {
    if (int const status = check_route(dtype, logits, logits_stride, tokens, experts, top_k, how)) return status;
    if ((size_t)how->top_groups * (experts / how->groups) < top_k) return mx_fail("experts_route: the groups that stay hold fewer than top_k experts");
    if (!tokens) return 0;
    if (!weights || !chosen) return mx_fail("experts_route: NULL operand");
    return with_row<false>(dtype, tokens <= (experts > 128 ? 4096 : 2048), experts, [&](auto value, auto lanes, auto per_lane) {
        typedef decltype(value) T;
        constexpr int L = decltype(lanes)::value, J = decltype(per_lane)::value;
        for (uint64_t first = 0; first < tokens; first += kMostThreads / L) {
            uint64_t const here = tokens - first < kMostThreads / L ? tokens - first : kMostThreads / L;
            RouteArgs const p = {(uint8_t const *)logits + first * logits_stride, logits_stride, (uint32_t)here, (uint32_t)experts, (uint32_t)top_k,
                                 bias, *how, weights + first * top_k, chosen + first * top_k};
            hipLaunchKernelGGL((route_kernel<T, L, J>), dim3((uint32_t)((here + 256 / L - 1) / (256 / L))), dim3(256), 0, (hipStream_t)stream, p);
            hipError_t const e = hipGetLastError();
            if (e != hipSuccess) return mx_fail(e, "route_kernel");
        }
        return 0;
    });
}

int nk_amd_experts_route_backward_async(nk_dtype_t dtype, void const *logits, nk_size_t logits_stride, nk_size_t tokens,
                                        nk_size_t experts, nk_size_t top_k, nk_amd_route_t const *how, nk_i32_t const *chosen,
                                        float const *grad_weights, void *grad_logits, nk_size_t grad_stride, void *stream) {
    if (int const status = check_route(dtype, logits, logits_stride, tokens, experts, top_k, how)) return status;
    if (!tokens) return 0;
    if (!chosen || !grad_weights || !grad_logits) return mx_fail("experts_route_backward: NULL operand");
    int const bytes = dtype == nk_f32_k ? 4 : 2;
    if (((uintptr_t)grad_logits | grad_stride) & (bytes - 1)) return mx_fail("experts_route_backward: grad_logits is not aligned to its elements");
    return with_row<true>(dtype, tokens <= 4096, experts, [&](auto value, auto lanes, auto per_lane) {
        typedef decltype(value) T;
        constexpr int L = decltype(lanes)::value, J = decltype(per_lane)::value;
        for (uint64_t first = 0; first < tokens; first += kMostThreads / L) {
            uint64_t const here = tokens - first < kMostThreads / L ? tokens - first : kMostThreads / L;
            RouteArgs const p = {(uint8_t const *)logits + first * logits_stride, logits_stride, (uint32_t)here, (uint32_t)experts, (uint32_t)top_k,
                                 nullptr, *how, nullptr, (int32_t *)chosen + first * top_k};
            hipLaunchKernelGGL((route_backward_kernel<T, L, J>), dim3((uint32_t)((here + 256 / L - 1) / (256 / L))), dim3(256), 0,
                               (hipStream_t)stream, p, grad_weights + first * top_k, (T *)((uint8_t *)grad_logits + first * grad_stride), (uint64_t)grad_stride);
            hipError_t const e = hipGetLastError();
            if (e != hipSuccess) return mx_fail(e, "route_backward_kernel");
        }
        return 0;
    });
}

nk_size_t nk_amd_experts_plan_size(nk_size_t slots, nk_size_t experts) {
    PlanGeometry g;
    return plan_geometry(slots, experts, g) ? g.total_words * 4 : 0;
}

int nk_amd_experts_plan_async(nk_i32_t const *chosen, nk_size_t slots, nk_size_t experts, void *plan, void *stream) {
    PlanGeometry g;
    if (!plan_geometry(slots, experts, g)) return mx_fail("experts_plan: 1 to 1024 experts, fewer than 2^30 slots");
    if (!plan || ((uintptr_t)plan & 15)) return mx_fail("experts_plan: the plan has to be 16-byte aligned");
    if (slots && (!chosen || ((uintptr_t)chosen & 3))) return mx_fail("experts_plan: chosen is NULL or misaligned");
    PlanHeader const header = {kPlanMagic, (uint32_t)slots, (uint32_t)experts, g.tile_rows, 0, 0, 0, 0};
    int bits = 0;
    while (experts >> bits) ++bits;
    uint32_t const blocks = slots ? (uint32_t)((slots + kPlanBlockSlots - 1) / kPlanBlockSlots) : 1, lds = (uint32_t)((experts + 1) * 4);
    uint32_t *const table = blocks > 1 ? (uint32_t *)plan + g.table : nullptr;
    if (table) hipLaunchKernelGGL(plan_count_kernel, dim3(blocks), dim3(kPlanThreads), lds, (hipStream_t)stream, chosen, (uint32_t)slots, (uint32_t)experts, table);
    bool const scanned = blocks > kPlanCountBlocks;
    if (scanned)
        hipLaunchKernelGGL(plan_scan_kernel, dim3((uint32_t)(experts / kScanBuckets + 1)), dim3(kScanBuckets * kScanParts), 0, (hipStream_t)stream,
                           (uint32_t)experts + 1, blocks, table);
    // Slots that fit one a lane are not followed by three more. (Up to 4,096 slots without the launch that counts, each workgroup
    // counting all slots: 7.3 us instead of 8.5 by itself, but 11.0 instead of 9.4 where `chosen` is not in the caches any more; eight
    // slots a lane: 15.5 us for 32,768.)
    auto *const kernel = slots <= kPlanThreads ? plan_kernel<1, false> : scanned ? plan_kernel<4, true> : plan_kernel<4, false>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kPlanThreads), lds * kPlanWaves, (hipStream_t)stream, chosen, (uint32_t)slots, (uint32_t)experts,
                       header, (uint32_t)g.offsets, (uint32_t)g.order, (uint32_t)g.place, (uint32_t)g.tiles, bits, table, blocks, (uint32_t *)plan);
    hipError_t const e = hipGetLastError();
    return e == hipSuccess ? 0 : mx_fail(e, "plan_kernel");
}

} // extern "C"
