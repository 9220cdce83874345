// The kernels behind attention.hip, instantiated by type in attention_half.hip and attention_float.hip.
//
//   s(r, p) = scale q[r] . k[p];   y[r] = sum_p 2^(s'(r, p) - m) v[p] / sum_p 2^(s'(r, p) - m),   s' = s log2(e)
//
// over the places p that row r sees, in one pass with a running maximum m.  Rows are the queries of all heads that share a head of k and v, so that
// those are read once for them.  Products are matrix instructions of 32 x 32 results, scores as k q^T: a lane then holds scores of one row, whose maximum and sum are two
// lanes' business, and the weights lie as the second product, v^T w^T, takes them: its sum runs over places in whichever order, so that v's are taken in
// the order in which the first product left them.
#pragma once

#include <cfloat>
#include <cmath>
#include <cstddef>
#include <type_traits>

#include "attention.h"

namespace chx {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at any address of an element

template <bool kHalf, int kSize>
struct Head {
    static constexpr int kElement = kHalf ? 2 : 4;
    static constexpr int kRow = kSize * kElement;  // bytes
    static constexpr int kChunks = kRow / 16;
    static constexpr int kSteps = kChunks / 2;     // of the first product: two chunks of 16 bytes, one to each half of the wavefront
    static constexpr int kBlocks = kSize / 32;     // of results of the second
    static constexpr int kWide = kSize / 32 < 4 ? kSize / 32 : 4;  // float32: elements of v that a lane reads at once
    // Chunk c of a row lies at place c ^ turned(row): the rows of an instruction (32 of k, a lane each; 4 of v, 64 bytes each) meet all banks.
    static __device__ __forceinline__ int turned(int row) {
        return kChunks == 8 ? ((row >> 1) & 1) << 2 | ((row >> 2) & 3) : (row & 3) << 2 | ((row >> 2) & 3);
    }
    // Calls f(element of the head, kVector results of a lane next to each other from it on) for all of them.
    static constexpr int kVector = kHalf ? 4 : kWide;
    typedef float Vector __attribute__((ext_vector_type(kVector)));
    template <typename F>
    static __device__ __forceinline__ void in_vectors(const f32x16 (&acc)[kBlocks], int half, F f) {
        if constexpr (kHalf) {
#pragma unroll
            for (int n = 0; n < kBlocks; ++n)
#pragma unroll
                for (int i = 0; i < 16; i += 4) f(element(n, i, half), Vector{acc[n][i], acc[n][i + 1], acc[n][i + 2], acc[n][i + 3]});
        } else {
#pragma unroll
            for (int n = 0; n < kBlocks; n += kWide)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    Vector v;
#pragma unroll
                    for (int j = 0; j < kWide; ++j) v[j] = acc[n + j][i];
                    f(element(n, i, half), v);
                }
        }
    }
    // Element of the head that result (block, i) of a lane is; i = 0..15.
    static __device__ __forceinline__ int element(int block, int i, int half) {
        const int r = 8 * (i >> 2) + 4 * half + (i & 3);
        return kHalf ? 32 * block + r : kWide * r + block % kWide + 32 * kWide * (block / kWide);
    }
};

__device__ const u32x4 kZeros[1] = {{0, 0, 0, 0}};  // what is not there is read from here

// What lies in memory at an address that has been chosen: said to be global memory's, which the compiler no longer sees then (it would ask whether it is LDS's, and wait for both).
template <typename T>
__device__ __forceinline__ T load_global(const char* p) {
    return *(const __attribute__((address_space(1))) T*)(uintptr_t)p;
}

// 16 bytes of a row of `bytes` bytes from byte `at` on (a multiple of 16), zeros behind its end and of a row that is not there.  The last ones of a row that is not whole pieces are its last 16, moved
// down.  (Addresses and values are chosen, here and below, where a branch that lanes take by themselves would do: where registers are short, the compiler puts moves of live ones before the point at which the
// others come back, and those lose what they held.)
template <bool kHalf>
__device__ __forceinline__ u32x4 chunk_of(const char* row, int32_t at, int32_t bytes, bool whole, bool there = true) {
    const char* none = reinterpret_cast<const char*>(kZeros);
    const bool any = there & (at < bytes);
    if (whole) return load_global<u32x4>(any ? row + at : none);
    if (bytes >= 16) {
        const u32x4 v = load_global<u32x4_any>(any ? row + min(at, bytes - 16) : none);
        const int32_t more = max(at + 16 - bytes, 0), bits = 8 * (more & 7);  // bytes of these that the row does not have
        uint64_t lower = (uint64_t)v[1] << 32 | v[0], upper = (uint64_t)v[3] << 32 | v[2];
        lower = more & 8 ? upper : lower;
        upper = more & 8 ? 0 : upper;
        lower = lower >> bits | (upper << 1) << (63 - bits);
        upper >>= bits;
        return u32x4{(uint32_t)lower, (uint32_t)(lower >> 32), (uint32_t)upper, (uint32_t)(upper >> 32)};
    }
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < (kHalf ? 8 : 4); ++j) {
        const int32_t b = j * (kHalf ? 2 : 4);
        const char* from = (any & (b < bytes)) ? row + b : none;  // (at is 0, or there is none of it)
        if constexpr (kHalf) v[j / 2] |= (uint32_t)load_global<uint16_t>(from) << (16 * (j & 1));
        else v[j] = load_global<uint32_t>(from);
    }
    return v;
}

// A number that all lanes of a wavefront have, where the compiler goes by memory or a division for it.
__device__ __forceinline__ int32_t uniform(int32_t v) {
    return __builtin_amdgcn_readfirstlane(v);
}
// (Of a work-group's sequence: the same for all its lanes, and through the scalar cache.)
__device__ __forceinline__ int32_t number_at(const int32_t* p, int64_t i) {
    return uniform(((const __attribute__((address_space(4))) int32_t*)(uintptr_t)p)[i]);
}
__device__ __forceinline__ int32_t length_of(const AttentionArgs& a, int32_t b) {
    return a.lengths ? max(0, min(number_at(a.lengths, b), a.places)) : a.places;
}
__device__ __forceinline__ int32_t count_of(const AttentionArgs& a, int32_t b) {
    return a.counts ? max(0, min(number_at(a.counts, b), a.T)) : a.T;
}

__device__ __forceinline__ Place place_in(const AttentionArgs& a, int32_t b, int32_t p) {
    return a.tables ? place_of(a, b, p) : Place{b, p};
}

// Which nodes each node of a tree sees: words of 32 bits, of all nodes, in LDS.  Every step doubles the ancestors that a node knows of.
struct Nodes {
    int16_t up[kMostNodes];
    uint32_t sees[kMostNodes][kMostNodes / 32];  // (of T nodes: a launch has memory for no more)
};
inline int nodes_bytes(const AttentionArgs& a) {
    return a.kind == kTree ? (int)offsetof(Nodes, sees) + a.T * (kMostNodes / 8) : 0;
}
template <int kThreads>
__device__ __forceinline__ void find_ancestors(Nodes* nodes, const int32_t* parents, int32_t T) {
    constexpr int kOf = kThreads < kMostNodes ? kMostNodes / kThreads : 1;  // nodes of a lane
    const int words = (T + 31) / 32;
    for (int i = threadIdx.x; i < T; i += kThreads) {
        const int32_t p = parents[i];
        nodes->up[i] = (int16_t)(p >= 0 && p < i ? p : -1);
        for (int w = 0; w < words; ++w) nodes->sees[i][w] = w == i / 32 ? 1u << (i & 31) : 0;
    }
    __syncthreads();
    for (int reach = 1; reach < T; reach *= 2) {
        uint32_t more[kOf][kMostNodes / 32];
        int32_t up[kOf], next[kOf];
#pragma unroll
        for (int j = 0; j < kOf; ++j) {
            const int i = j * kThreads + threadIdx.x;
            up[j] = i < T ? nodes->up[i] : -1;
            next[j] = up[j] >= 0 ? nodes->up[up[j]] : -1;
#pragma unroll
            for (int w = 0; w < kMostNodes / 32; ++w) more[j][w] = w < words && up[j] >= 0 ? nodes->sees[up[j]][w] : 0;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kOf; ++j) {
            const int i = j * kThreads + threadIdx.x;
            if (up[j] < 0) continue;
            nodes->up[i] = (int16_t)next[j];
#pragma unroll
            for (int w = 0; w < kMostNodes / 32; ++w)
                if (w < words) nodes->sees[i][w] |= more[j][w];
        }
        __syncthreads();
    }
}

// What a row sees: places below `limit`, and of a tree's nodes, which lie from `length` on, those that its own node does.
struct Sight {
    int32_t limit, length, count;
    int32_t node;  // -1: none
    bool trees;    // whether any row has one
};
__device__ __forceinline__ Sight sight_of(const AttentionArgs& a, int32_t t, int32_t length, int32_t count) {
    const int32_t limit = a.kind == kChain ? length + t + 1 : length;
    return {t < count ? limit : 0, length, count, a.kind == kTree && t < count ? t : -1, a.kind == kTree};
}
// Which of the places p0 to p0 + 31 a row sees, a bit each.  (A node's words have only nodes before it and itself, all below count.)
__device__ __forceinline__ uint32_t seen_of(const Sight& s, const Nodes* nodes, int32_t p0) {
    const int32_t below = s.limit - p0;
    uint32_t seen = below >= 32 ? ~0u : below > 0 ? (1u << below) - 1 : 0;
    const int32_t i = p0 - s.length;  // the node that lies at p0
    if (s.trees && i > -32 && i < s.count) {
        const uint32_t* words = nodes->sees[max(s.node, 0)];
        const uint64_t lower = i < 0 ? 0 : words[max(i >> 5, 0)], upper = words[min((i >> 5) + 1, kMostNodes / 32 - 1)];
        const uint32_t seen_nodes = (uint32_t)((lower | upper << 32) >> (i & 31));
        seen |= s.node >= 0 ? seen_nodes : 0;
    }
    return seen;
}

// Tiles that the maximum may lag behind by: weights are then up to 2^kLag, and kept that much and kRaise higher than they are in relation to the largest, so that few of those
// of float16 fall below its normal numbers (2^-14): 2^-20 of the largest does.
constexpr float kLag = 8.f;
template <bool kHalf>
constexpr float kRaise = kHalf ? 6.f : 0.f;
constexpr float kNoMaximum = -3e38f;

// A lane's value and that of the one with the row's other scores, in both.
struct Halves {
    float lower, upper;
};
__device__ __forceinline__ Halves both_halves(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto both = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const uint32_t lower = both[0], upper = both[1];  // (numbers of their own: the compiler takes the first element's bits for those of any that is cast in place)
    return {__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper)};
}
__device__ __forceinline__ float sum_of_halves(float v) {
    const Halves h = both_halves(v);
    return h.lower + h.upper;
}
__device__ __forceinline__ float largest_of_halves(float v) {
    const Halves h = both_halves(v);
    return fmaxf(h.lower, h.upper);
}

// The scores of 32 places and 32 rows, of one step's elements.
template <bool kHalf>
__device__ __forceinline__ f32x16 score_of(u32x4 k, u32x4 q, f32x16 score) {
    if constexpr (kHalf) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, k), __builtin_bit_cast(half8, q), score, 0, 0, 0);
    const f32x4 kf = __builtin_bit_cast(f32x4, k), qf = __builtin_bit_cast(f32x4, q);
#pragma unroll
    for (int j = 0; j < 4; ++j) score = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], qf[j], score, 0, 0, 0);
    return score;
}

// The scores of places that are seen, -inf in the others' place.  (Chosen without branches.)
__device__ __forceinline__ f32x16 hide(f32x16 score, uint32_t seen) {
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = (seen >> (8 * (i >> 2) + (i & 3))) & 1 ? score[i] : -INFINITY;
    return s;
}

// log2 of a row's sum of weights; +inf where it has none, so that each of them is 0.
template <bool kHalf>
__device__ __forceinline__ float sum_of(float m, float l) {
    return l == 0.f ? INFINITY : m - kRaise<kHalf> + log2f(l);
}

// Rounding to float16 of a weighted mean.  What is finite stays so: the weights were rounded to float16 before the products and their sum was not, so that a mean of 65504 and the like may come out up to
// 2^-11 of it higher, which is infinity from 2^-12 on.
__device__ __forceinline__ _Float16 to_half(float v) {
    const float within = __builtin_amdgcn_fmed3f(v, -65504.f, 65504.f);
    return (_Float16)(fabsf(v) <= FLT_MAX ? within : v);
}

// Elements of a result next to each other.
template <int kCount, typename V>
__device__ __forceinline__ void store(const AttentionArgs& a, char* row, int32_t element, V v) {
    using E = std::remove_reference_t<decltype(v[0])>;
    E* to = reinterpret_cast<E*>(row) + element;
    if (a.y_whole) {
        if (element < a.D) *reinterpret_cast<V*>(to) = v;
        return;
    }
#pragma unroll
    for (int j = 0; j < kCount; ++j)
        if (element + j < a.D) to[j] = v[j];
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
template <typename V>
__device__ __forceinline__ __attribute__((address_space(3))) V* lds_pointer(uint32_t at) {
    return (__attribute__((address_space(3))) V*)(uintptr_t)at;
}

// ---- a wavefront's work on a block of places: 32 rows, a lane's row is lane & 31 ---------------------------------

// Steps of products whose operands come from LDS: load(i) asks for step i's, use(i) multiplies them, kAhead steps later.  The compiler alone puts each load right in front of its use and waits for it.
template <int kSteps, int kAhead, typename Load, typename Use>
__device__ __forceinline__ void in_steps(Load load, Use use) {
#pragma unroll
    for (int i = 0; i < kAhead && i < kSteps; ++i) load(i);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        if (i + kAhead < kSteps) load(i + kAhead);
        __builtin_amdgcn_sched_barrier(6);  // (vector and scalar arithmetic may cross)
        use(i);
    }
}

// Scores of blocks of 32 places, whose keys lie in LDS from `keys` on; 32 rows to a lane's column.
template <bool kHalf, int kSize, int kCount>
__device__ __forceinline__ void find_scores(const char* keys, const u32x4 (&q)[Head<kHalf, kSize>::kSteps], f32x16 (&score)[kCount]) {
    using H = Head<kHalf, kSize>;
    const int lane = threadIdx.x & 63, row = lane & 31;
    // (chunk 2 s + half of row, its place turned: s comes in by one more exclusive or; 32 rows on, all is the same)
    uint32_t at = lds_address(keys) + row * H::kRow + (((lane >> 5) ^ H::turned(row)) << 4);
    asm volatile("" : "+v"(at));  // (the others are made from it where they are used)
#pragma unroll
    for (int n = 0; n < kCount; ++n) score[n] = f32x16{};
    constexpr int kAhead = kHalf ? 4 : 2;
    u32x4 k[kAhead + 1][kCount];
    in_steps<H::kSteps, kAhead>(
            [&](int s) __attribute__((always_inline)) {
#pragma unroll
                for (int n = 0; n < kCount; ++n) k[s % (kAhead + 1)][n] = *lds_pointer<u32x4>((at ^ (s << 5)) + n * 32 * H::kRow);
            },
            [&](int s) __attribute__((always_inline)) {
#pragma unroll
                for (int n = 0; n < kCount; ++n) score[n] = score_of<kHalf>(k[s % (kAhead + 1)][n], q[s], score[n]);
            });
}

// The rows' maxima with these scores; the sums so far are brought to them.
template <bool kHalf, int kBlocks, int kCount>
__device__ __forceinline__ void find_maxima(float scale2, const f32x16 (&score)[kCount], f32x16 (&acc)[kBlocks], float& m, float& l) {
    float of[4] = {score[0][0], score[0][1], score[0][2], score[0][3]};  // (four chains, below for the sum too)
#pragma unroll
    for (int n = 0; n < kCount; ++n)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
#pragma unroll
            for (int j = 0; j < 4; ++j) of[j] = fmaxf(of[j], score[n][i + j]);
    const float most = largest_of_halves(fmaxf(fmaxf(of[0], of[1]), fmaxf(of[2], of[3]))) * scale2;
    if (__builtin_amdgcn_ballot_w64(most > m + kLag)) {
        const float next = fmaxf(m, most), f = __builtin_amdgcn_exp2f(m - next);
        l *= f;
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) acc[n] *= f;
        m = next;
    }
}

// Weights in the scores' place.
template <bool kHalf, int kCount>
__device__ __forceinline__ void find_weights(float scale2, f32x16 (&score)[kCount], float m, float& l) {
    const float less = m - kRaise<kHalf>;
    float sum[4] = {};
#pragma unroll
    for (int n = 0; n < kCount; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            score[n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[n][i], scale2, -less));
            sum[i & 3] += score[n][i];
        }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// How often what is finite is halved where results are made again, in float32: weights are up to 2^kLag, there are fewer than 2^(32 - clz) places, and the sums of all of them are then below float32's
// largest number whatever the values are.  (float16's values and weights are below 2^16 and 2^14, and 2^30 places of those no problem.)
template <bool kHalf>
__device__ __forceinline__ int halvings(const AttentionArgs& a) {
    return kHalf ? 0 : (int)kLag + 32 - __builtin_clz(a.places | 1);
}

// What is added up in place of v, all of it in LDS: itself, or (where results are made again) ones for what is inf, -inf and NaN, or what is finite, times `less`.
enum { kAll, kInfinities, kNegativeInfinities, kNans, kFinite };
template <bool kHalf>
__device__ __forceinline__ void replace_values(char* values, int32_t bytes, int32_t special, float less, int32_t thread, int32_t threads) {
    using E = std::conditional_t<kHalf, _Float16, float>;
#pragma unroll 1
    for (int32_t i = thread; i < bytes / (int32_t)sizeof(E); i += threads) {
        const float v = (float)reinterpret_cast<const E*>(values)[i];
        const bool finite = v - v == 0.f, marked = special == kNans ? v != v : v == (special == kInfinities ? INFINITY : -INFINITY);
        reinterpret_cast<E*>(values)[i] = (E)(special == kFinite ? (finite ? v * less : 0.f) : marked ? 1.f : 0.f);
    }
}

// acc += v^T weights^T, v's rows in LDS from `values` on.  float16: weights are rounded to float16, which is what lets float16 matrix instructions take them (1431 TFLOP/s where float32's reach 150; as two
// float16 numbers each, the second product would cost twice as much).  Each is off by up to 2^-11 of itself, as much as the result's rounding is, and they average out: over 4096 places results are off by 2.9e-4 of their norm
// against 2.1e-4 with weights in float32.  Their sum, which divides, is of the weights before that.
template <bool kHalf, int kSize, int kCount>
__device__ __forceinline__ void add_values(const char* values, const f32x16 (&weight)[kCount], f32x16 (&acc)[kSize / 32]) {
    using H = Head<kHalf, kSize>;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    if constexpr (kHalf) {
        // 16 lanes read 4 rows of 16 elements, which are transposed on the way: a lane gets 4 rows of one element.  Two such reads make a fragment; 16 rows on, all is the same, and
        // 32 elements on one more exclusive or
        uint32_t at[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = e * 8 + 4 * half + ((lane & 15) >> 2), c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            at[e] = lds_address(values) + row * H::kRow + ((c ^ H::turned(row)) << 4) + 8 * (lane & 1);
            asm volatile("" : "+v"(at[e]));
        }
        half8 w[2 * kCount];
#pragma unroll
        for (int kb = 0; kb < 2 * kCount; ++kb)
#pragma unroll
            for (int j = 0; j < 8; ++j) w[kb][j] = (_Float16)weight[kb >> 1][8 * (kb & 1) + j];
        constexpr int kAhead = 6;
        union {
            short4v part[2];
            half8 whole;
        } v[kAhead + 1];
        in_steps<2 * kCount * H::kBlocks, kAhead>(
                [&](int i) __attribute__((always_inline)) {
                    const int kb = i / H::kBlocks, n = i % H::kBlocks;
#pragma unroll
                    for (int e = 0; e < 2; ++e) v[i % (kAhead + 1)].part[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_pointer<short4v>((at[e] ^ (n << 6)) + kb * 16 * H::kRow));
                },
                [&](int i) __attribute__((always_inline)) {
                    acc[i % H::kBlocks] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i % (kAhead + 1)].whole, w[i / H::kBlocks], acc[i % H::kBlocks], 0, 0, 0);
                });
    } else {
        // a lane reads kWide elements of one row; row i of a block is turned by what 16 rows have in common
        constexpr int kWide = H::kWide, kReads = H::kBlocks / kWide, kAhead = 3;
        typedef float Wide __attribute__((ext_vector_type(kWide)));
        uint32_t at = lds_address(values) + 4 * half * H::kRow + 4 * kWide * (lane & 31);
        asm volatile("" : "+v"(at));
        const uint32_t turn = half << 4;  // of row 4 half
        Wide v[kAhead + 1];
        in_steps<kCount * 16 * kReads, kAhead>(
                [&](int i) __attribute__((always_inline)) {
                    const int of = i / kReads, row = 8 * (of >> 2) + (of & 3);  // (16 to a block of 32)
                    v[i % (kAhead + 1)] = *lds_pointer<Wide>((at ^ (H::turned(row) << 4) ^ turn) + row * H::kRow + 128 * kWide * (i % kReads));
                },
                [&](int i) __attribute__((always_inline)) {
                    const int of = i / kReads, w = i % kReads;
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
                        acc[w * kWide + j] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[i % (kAhead + 1)][j], weight[of / 16][of % 16], acc[w * kWide + j], 0, 0, 0);
                });
    }
}

// Whether a lane has a sum that is not finite.
template <int kBlocks>
__device__ __forceinline__ bool not_finite(const f32x16 (&acc)[kBlocks]) {
    float zero = 0.f;
#pragma unroll
    for (int n = 0; n < kBlocks; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) zero = __builtin_fmaf(acc[n][i], 0.f, zero);
    return zero != 0.f;
}

// The sums of a row, added up again where one of them is not finite: then v is not, or it is the product of 0 and something infinite, and places of no weight add nothing, whatever they hold; or the
// sum is more than float32 holds, which the mean is not.  `pass` goes over the places once, with what stands for v.  `any`: of all that make the passes together.  Returns what the sums are to be
// multiplied by (after the division by the weights' sum): 1, or a power of 2 where they were made of smaller values.
template <int kBlocks, typename Pass, typename Any>
__device__ __forceinline__ float add_up(f32x16 (&acc)[kBlocks], int halved, Pass pass, Any any) {
    uint32_t marks[3][kBlocks / 2];  // a bit for each sum: whether it has an inf, -inf, NaN
#pragma unroll 1
    for (int32_t special = kAll; special <= kFinite; ++special) {
        pass(special);
        if (special == kAll) {
            if (!any(not_finite(acc))) return 1.f;
        } else if (special < kFinite) {
#pragma unroll
            for (int n = 0; n < kBlocks; n += 2) {
                uint32_t found = 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) found |= (uint32_t)(acc[n + i / 16][i & 15] > 0.f) << i;
#pragma unroll
                for (int k = 0; k < 3; ++k) marks[k][n / 2] = special == k + 1 ? found : marks[k][n / 2];
            }
        }
    }
#pragma unroll
    for (int n = 0; n < kBlocks; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int bit = 16 * (n & 1) + i;
            float v = acc[n][i];
            v += (marks[0][n / 2] >> bit) & 1 ? INFINITY : 0.f;
            v -= (marks[1][n / 2] >> bit) & 1 ? INFINITY : 0.f;
            acc[n][i] = (marks[2][n / 2] >> bit) & 1 ? NAN : v;
        }
    return ldexpf(1.f, halved);
}

// ---- rows of k and v into LDS ---------------------------------------------------------------------------------------

// Asynchronous copies of 16 bytes a lane into LDS, lane i's to lds + 16 i (the same for all lanes), counted like loads.  (The base goes through a scalar instruction: where the compiler has it from a vector
// one, as a v_readlane, five cycles would have to pass before a memory instruction reads it, and it does not see that this is one.  Waiting them out in each copy: 599 us of 2048 x 4096 rows, so 594.)
__device__ __forceinline__ void copy_to_lds(uint32_t offset, const char* base, uint32_t lds) {
    const char* from;
    asm volatile("s_mov_b32 m0, %3\n\ts_mov_b64 %0, %2\n\tglobal_load_lds_dwordx4 %1, %0" : "=&s"(from) : "v"(offset), "s"(base), "s"(uniform(lds)) : "memory", "m0");
}
// (Of some lanes only.)
__device__ __forceinline__ void copy_to_lds(uint32_t offset, const char* base, uint32_t lds, uint64_t lanes) {
    const char* from;
    uint64_t all;
    asm volatile("s_mov_b32 m0, %4\n\ts_mov_b64 %0, %3\n\ts_and_saveexec_b64 %1, %5\n\tglobal_load_lds_dwordx4 %2, %0\n\ts_mov_b64 exec, %1"
                 : "=&s"(from), "=&s"(all) : "v"(offset), "s"(base), "s"(uniform(lds)), "s"(lanes) : "memory", "m0", "scc");
}
__device__ __forceinline__ void copy_to_lds(const char* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(uniform(lds)) : "memory", "m0");
}
// (4 bytes a lane, lane i's to lds + 4 i.)
__device__ __forceinline__ void copy_number_to_lds(uint32_t offset, const char* base, uint32_t lds, uint64_t lanes) {
    const char* from;
    uint64_t all;
    asm volatile("s_mov_b32 m0, %4\n\ts_mov_b64 %0, %3\n\ts_and_saveexec_b64 %1, %5\n\tglobal_load_lds_dword %2, %0\n\ts_mov_b64 exec, %1"
                 : "=&s"(from), "=&s"(all) : "v"(offset), "s"(base), "s"(uniform(lds)), "s"(lanes) : "memory", "m0", "scc");
}
__device__ __forceinline__ void copy_number_to_lds(const float* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(from), "s"(uniform(lds)) : "memory", "m0");
}

// What a lane knows of kPlaces places from p0 on, some of them before end: of place p0 + lane % kPlaces, where it lies; of all, which are there.
template <int kPlaces>
struct Places {
    Place at;
    uint64_t there;
    __device__ __forceinline__ Places(const AttentionArgs& a, int32_t b, int32_t p0, int32_t end) {
        const int32_t p = p0 + (int)(threadIdx.x & (kPlaces - 1));
        at = place_in(a, b, min(p, end - 1));
        at.page = p < end ? at.page : -1;
        there = __builtin_amdgcn_ballot_w64(at.page >= 0);
    }
};

// One of the arrays that is copied from.
struct From {
    const char* base;  // of the group's head
    int64_t page, row;
    uint32_t of_lane;  // how far the lane's row is from the first one of an instruction
    bool near;         // every row is less than 4 GB behind base
    uint32_t bytes;    // of a row
    bool whole;        // rows and their distances are whole pieces of 16 bytes
};
template <typename H>
__device__ __forceinline__ From from_of(const AttentionArgs& a, const char* base, int64_t page, int64_t row, int32_t b) {
    const uint32_t of_lane = (uint32_t)((threadIdx.x & 63) / H::kChunks * row);
    if (a.tables == nullptr) return {base + b * page, 0, row, of_lane, row >= 0 && a.places * row < (int64_t(1) << 31), (uint32_t)(a.D * H::kElement), a.k_whole};
    return {base, page, row, of_lane, page >= 0 && row >= 0 && page < (int64_t(1) << 31) && row < (int64_t(1) << 31) && (int64_t)a.pages * page + a.page_rows * row < (int64_t(1) << 32), (uint32_t)(a.D * H::kElement), a.k_whole};
}

// Whether the rows of every instruction's copies (of four, where it has fewer) lie in one page, at distances that 32 bits hold: then their address is one of the wavefront's and an offset.
template <typename H>
__device__ __forceinline__ bool in_runs(const AttentionArgs& a) {
    constexpr int32_t kRows = 64 / H::kChunks < 4 ? 4 : 64 / H::kChunks;
    return (a.k_whole || H::kElement == 4) && (a.tables == nullptr || a.page_rows % kRows == 0) && a.k_row >= 0 && a.k_row < (1 << 24) && a.v_row >= 0 && a.v_row < (1 << 24);
}

// kCount copies from the first-th of the tile on, for places anywhere.  What is not there, and what a row has less than the kernel's, is 0.
template <typename H, int kPlaces, int kCount>
__device__ __forceinline__ void copy_rows(const AttentionArgs& a, const From& f, const Places<kPlaces>& places, uint32_t lds, char* to, int32_t first) {
    constexpr int kRows = 64 / H::kChunks, kAtOnce = 2;
    static_assert(kCount % kAtOnce == 0 || kCount < kAtOnce, "whole rounds");
    const int lane = threadIdx.x & 63;
    const int32_t row_bytes = a.D * H::kElement;
#pragma unroll 1
    for (int j0 = 0; j0 < kCount; j0 += kAtOnce) {
        const char* from[kAtOnce];
        int32_t c[kAtOnce];
        bool there[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce && j < kCount; ++j) {
            const int32_t row = (first + j0 + j) * kRows + lane / H::kChunks, page = __shfl(places.at.page, row), at = __shfl(places.at.row, row);
            c[j] = ((lane % H::kChunks) ^ H::turned(row)) << 4;
            there[j] = page >= 0;
            from[j] = f.base + page * f.page + at * f.row;
        }
        if (a.k_whole) {
#pragma unroll
            for (int j = 0; j < kAtOnce && j < kCount; ++j) copy_to_lds((there[j] & (c[j] < row_bytes)) ? from[j] + c[j] : reinterpret_cast<const char*>(kZeros), lds + (first + j0 + j) * 1024);
        } else {
            u32x4 v[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce && j < kCount; ++j) v[j] = chunk_of<H::kElement == 2>(from[j], c[j], row_bytes, false, there[j]);
#pragma unroll
            for (int j = 0; j < kAtOnce && j < kCount; ++j) *reinterpret_cast<u32x4*>(to + (first + j0 + j) * 1024 + lane * 16) = v[j];
        }
    }
}

// Where a tile's places lie whose rows come in runs of kRun, all of them there: known to the wavefront, and asked for through the scalar cache, so that nobody waits for copies
// that are on their way to have it.  (Tables do not change while a kernel runs.)  A wavefront keeps what it copies itself: kOwn places from own on.
template <typename H, int kPlaces, int kOwn>
struct Runs {
    static constexpr int kRun = 64 / H::kChunks < 4 ? 4 : 64 / H::kChunks, kCount = kOwn / kRun;
    int32_t page[kCount], row[kCount];
    bool good;
    __device__ __forceinline__ void look_up(const AttentionArgs& a, int32_t b, int32_t p0, int32_t own, int32_t end, bool runs) {
        good = runs && p0 + kPlaces <= end;
        if (!good) return;
        if (a.tables == nullptr) {
#pragma unroll
            for (int i = 0; i < kCount; ++i) page[i] = 0, row[i] = p0 + own + i * kRun;
            return;
        }
        const auto* table = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(a.tables + b * a.table_row);
        if constexpr (kOwn < kPlaces) good = all_there(a, table, p0, kPlaces);
        int32_t at = over(p0 + own, a.by_page), r = p0 + own - at * a.page_rows;
        uint32_t outside = 0;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            page[i] = table[at];
            row[i] = r;
            r += kRun;
            if (r >= a.page_rows) r = 0, ++at;
        }
#pragma unroll
        for (int i = 0; i < kCount; ++i) outside |= (uint32_t)page[i] >= (uint32_t)a.pages;
        good = good && outside == 0;
    }
    static __device__ __forceinline__ bool all_there(const AttentionArgs& a, const __attribute__((address_space(4))) int32_t* table, int32_t p0, int32_t places) {
        const int32_t first = over(p0, a.by_page), last = over(p0 + places - 1, a.by_page);
        uint32_t outside = 0;
        for (int32_t i = first; i <= last; ++i) outside |= (uint32_t)table[i] >= (uint32_t)a.pages;
        return outside == 0;
    }
};

// The copies of a wavefront's own places: kCount of them from the first-th of the tile on.
template <typename H, int kCount, typename R>
__device__ __forceinline__ void copy_runs(const From& f, const R& runs, uint32_t lds, int32_t first) {
    constexpr int kRows = 64 / H::kChunks;
    int32_t lane = threadIdx.x & 63;
    // (Where a row is one copy and a wavefront has many, what differs from one to the next is made where it is used.  Made ahead it is 16 registers, and the kernel for few rows of 256 elements, which has none
    // left, kept 21 in memory: a token of 8 sequences of up to 4000 places, 32 heads over 8, 226 us, so 177.)
    if constexpr (H::kRow > 512 && kCount > 8) asm volatile("" : "+v"(lane));
    auto all = [&](auto simple) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) {
            const int32_t row = (first + j) * kRows + lane / H::kChunks, page = runs.page[j * kRows / R::kRun], at = runs.row[j * kRows / R::kRun] + j * kRows % R::kRun;
            const uint32_t c = ((lane % H::kChunks) ^ H::turned(row)) << 4;
            // (rows that are shorter than the kernel's leave the rest as it is, which is 0)
            if constexpr (decltype(simple)::value) copy_to_lds(f.of_lane + c + ((uint32_t)page * (uint32_t)f.page + (uint32_t)at * (uint32_t)f.row), f.base, lds + (first + j) * 1024);
            else copy_to_lds(f.of_lane + c, f.base + page * f.page + at * f.row, lds + (first + j) * 1024, __builtin_amdgcn_ballot_w64(c < f.bytes));
        }
    };
    if (f.near && f.whole && f.bytes == H::kRow) all(std::true_type());
    else if (H::kElement == 2 || f.whole) all(std::false_type());
    else {
        // Rows of float32 that are not whole pieces, by their elements: the same bytes in four times the copies.
        int32_t place = lane;
        asm volatile("" : "+v"(place));  // (the addresses are made where they are used, and not kept in registers)
#pragma unroll
        for (int j = 0; j < 4 * kCount; ++j) {
            const int32_t row = first * kRows + j * 256 / H::kRow;
            const uint32_t c = ((place >> 2 | (j * 16 & (H::kChunks - 1))) ^ H::turned(row)) << 4 | (place & 3) << 2;
            copy_number_to_lds(c, f.base + runs.page[j * 256 / H::kRow / R::kRun] * f.page + (runs.row[j * 256 / H::kRow / R::kRun] + j * 256 / H::kRow % R::kRun) * f.row, lds + first * 1024 + j * 256, __builtin_amdgcn_ballot_w64(c < f.bytes));
        }
    }
}

// Zeros where rows that are shorter than the kernel's do not come.
template <typename H>
__device__ __forceinline__ void clear_rest(const AttentionArgs& a, char* lds, int32_t bytes, int32_t thread, int32_t threads) {
    if (a.D * H::kElement == H::kRow) return;
    for (int32_t i = thread; i < bytes / 16; i += threads) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// ---- results ----------------------------------------------------------------------------------------------------------

// A row's results, or its mean over one part: 16 elements of it in blocks of 32 to a lane.
template <bool kHalf, int kSize>
__device__ __forceinline__ void finish_row(const AttentionArgs& a, f32x16 (&acc)[kSize / 32], float more, float m, float l, int32_t b, int32_t group, int32_t r, int64_t part_row, bool any) {
    using H = Head<kHalf, kSize>;
    const int half = (threadIdx.x & 63) >> 5;
    const int32_t rows = a.T * a.fan;
    l = sum_of_halves(l);
    const float share = l == 0.f ? 0.f : more / l;
#pragma unroll
    for (int n = 0; n < H::kBlocks; ++n) acc[n] *= share;
    if (a.parts > 1) {
        if (half == 0) *reinterpret_cast<f32x2*>(a.part_stats + 2 * part_row) = f32x2{m, l};
        if (!any || r >= rows) return;
        float* to = a.part_sums + part_row * kSize;
        H::in_vectors(acc, half, [&](int element, typename H::Vector v) __attribute__((always_inline)) { *reinterpret_cast<typename H::Vector*>(to + element) = v; });
        return;
    }
    if (r >= rows) return;
    if (a.sums != nullptr && half == 0) a.sums[((int64_t)b * a.groups + group) * rows + r] = sum_of<kHalf>(m, l);
    const int32_t t = over(r, a.by_fan), head = group * a.fan + (r - t * a.fan);
    char* y = a.y + b * a.y_batch + t * a.y_token + head * a.y_head;
    H::in_vectors(acc, half, [&](int element, typename H::Vector v) __attribute__((always_inline)) {
        if constexpr (kHalf) store<4>(a, y, element, half4{to_half(v[0]), to_half(v[1]), to_half(v[2]), to_half(v[3])});
        else store<H::kVector>(a, y, element, v);
    });
}

// What a work-group works on.
struct Job {
    int32_t b, group, part, row_tile;
    int32_t rows, length, count, end;  // end: of the places that any of its rows sees
    int32_t begin_tile, end_tile;      // of its part
    int64_t at;                        // where its part's sums go, in tiles
};
__device__ __forceinline__ Job job_of(const AttentionArgs& a, int32_t tile_rows, int32_t tile_places) {
    Job j;
    // Work-groups go to the eight XCDs in turn.  Neighbours read neighbouring heads' rows of the same places; the tiles of rows that read the same part of k and v follow each other on one XCD,
    // whose L2 they share; those of the last parts, fewer than eight, are dealt out evenly.
    const int32_t whole_sets = a.B * a.groups * a.parts / 8 * 8;
    const uint32_t whole = whole_sets * a.row_tiles, turn = blockIdx.x < whole ? blockIdx.x >> 3 : blockIdx.x - whole, of_turn = over(turn, a.by_row_tiles);
    const int32_t set = blockIdx.x < whole ? of_turn * 8 + (blockIdx.x & 7) : whole_sets + of_turn, of_group = over(set, a.by_groups);
    // (of a chain, the tiles with the most places first)
    j.row_tile = a.row_tiles - 1 - (int32_t)(turn - of_turn * a.row_tiles);
    j.group = set - of_group * a.groups;
    j.b = over(of_group, a.by_parts);
    j.part = of_group - j.b * a.parts;
    j.at = (((int64_t)j.b * a.groups + j.group) * a.row_tiles + j.row_tile) * a.parts + j.part;
    j.rows = a.T * a.fan;
    j.length = length_of(a, j.b);
    j.count = count_of(a, j.b);
    const int32_t first_t = over(j.row_tile * tile_rows, a.by_fan), last_t = min(over(min((j.row_tile + 1) * tile_rows, j.rows) - 1, a.by_fan), j.count - 1);
    j.end = last_t < first_t ? 0 : a.kind == kCross ? j.length : a.kind == kChain ? j.length + last_t + 1 : j.length + j.count;
    j.end = min(j.end, a.places);
    const int32_t tiles = (j.end + tile_places - 1) / tile_places, each = over(tiles + a.parts - 1, a.by_parts);
    j.begin_tile = j.part * each;
    j.end_tile = min(j.begin_tile + each, tiles);
    return j;
}

// A lane's row, and what the rows of its wavefront see.
struct Row {
    int32_t r, t, head;
    Sight sight;
    int32_t plain;  // places below this are seen by all of them
};
__device__ __forceinline__ Row row_of(const AttentionArgs& a, const Job& j, int32_t first) {  // first: of the wavefront's 32
    Row row;
    row.r = first + (int)(threadIdx.x & 31);
    // (rows behind the last do what the last one does; their results go nowhere)
    const int32_t r = min(row.r, j.rows - 1);
    row.t = over(r, a.by_fan);
    row.head = j.group * a.fan + (r - row.t * a.fan);
    row.sight = sight_of(a, row.t, j.length, j.count);
    const int32_t first_t = over(min(first, j.rows - 1), a.by_fan), last_t = over(min(first + 31, j.rows - 1), a.by_fan);
    row.plain = last_t >= j.count ? 0 : a.kind == kChain ? j.length + first_t + 1 : j.length;
    return row;
}
// The rows of a wavefront; those that are not whole pieces go through `space` in LDS, of 32 rows.
template <bool kHalf, int kSize>
__device__ __forceinline__ void load_rows(const AttentionArgs& a, const Job& j, const Row& row, char* space, u32x4 (&q)[Head<kHalf, kSize>::kSteps]) {
    using H = Head<kHalf, kSize>;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int32_t row_bytes = a.D * H::kElement;
    const char* at = a.q + j.b * a.q_batch + row.t * a.q_token + row.head * a.q_head;
    if (a.q_whole) {
#pragma unroll
        for (int s = 0; s < H::kSteps; ++s) q[s] = chunk_of<kHalf>(at, (2 * s + half) * 16, row_bytes, true);
    } else {
        u32x4* mine = reinterpret_cast<u32x4*>(space) + (lane & 31) * H::kChunks;
#pragma unroll 1
        for (int c = half; c < H::kChunks; c += 2) mine[c] = chunk_of<kHalf>(at, c * 16, row_bytes, false);
#pragma unroll
        for (int s = 0; s < H::kSteps; ++s) q[s] = mine[2 * s + half];  // (what this lane has written itself)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (before the copies that come there: they write LDS past the order of its own instructions)
    }
}
// They are waited for here, behind the first copies: a first use inside a loop would wait for everything that is under way, in every round of it.
template <int kSteps>
__device__ __forceinline__ void wait_for(u32x4 (&q)[kSteps]) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(q[s]));
}

// ---- many rows --------------------------------------------------------------------------------------------------------
//
// A work-group has 128 rows, its four wavefronts 32 each, and goes over the places of one part in tiles that it copies into LDS together: two of them, the next one on its way while this one
// is worked on.
// Where a head of k has thousands of rows, bound by the matrix cores and the vector units, which the two wavefronts of a SIMD use in turn: 4 x 2048 tokens over 4096 states, 32 heads over 8 of 128 elements,
// float16: 573 us, 960 TFLOP/s.  Its products alone are 267 us of the matrix cores, its exponentials, maxima, sums and roundings 208 of the vector units, and what LDS gives 198; with one work-group to
// a compute unit it is 712.  Tried, and slower: the next block's scores during this one's softmax, with a ring of blocks of 32 places (674) or interleaved by hand (589); eight wavefronts to a
// work-group (632); values read ahead of the weights (the same).  Where there are few rows, bound by the bytes of k and v: 4 x 24 tokens over 32768 places, 105 us, 5.1 TB/s.
template <bool kHalf, int kSize>
struct Tile {
    static constexpr int kWaves = 4, kRows = kWaves * 32;
    static constexpr int kBlocksOf = Head<kHalf, kSize>::kRow <= 512 ? 2 : 1;  // of 32 places
    static constexpr int kPlaces = 32 * kBlocksOf;
    static constexpr int kBytes = kPlaces * Head<kHalf, kSize>::kRow;  // of k or v
    static constexpr int kCopies = kBytes / 1024 / kWaves;
    static constexpr int kLds = 4 * kBytes;  // two tiles of k and v (and nodes)
};

template <bool kHalf, int kSize>
__global__ __launch_bounds__(256, (Tile<kHalf, kSize>::kLds <= 80 * 1024 ? 2 : 1)) void attention_rows_kernel(AttentionArgs a) {
    using H = Head<kHalf, kSize>;
    using W = Tile<kHalf, kSize>;
    extern __shared__ __attribute__((aligned(1024))) char attention_lds[];
    Nodes* nodes = reinterpret_cast<Nodes*>(attention_lds + 4 * W::kBytes);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
    const Job job = job_of(a, W::kRows, W::kPlaces);
    if (a.kind == kTree && job.begin_tile < job.end_tile && job.end_tile * W::kPlaces > job.length) find_ancestors<256>(nodes, a.parents + (int64_t)job.b * a.T, a.T);
    const Row row = row_of(a, job, job.row_tile * W::kRows + wave * 32);
    u32x4 q[H::kSteps];
    load_rows<kHalf, kSize>(a, job, row, attention_lds + wave * 32 * H::kRow, q);
    if (!a.q_whole) __syncthreads();  // (the tiles come where they lay)
    if (a.D * H::kElement != H::kRow) {
        clear_rest<H>(a, attention_lds, W::kLds, threadIdx.x, 256);
        __syncthreads();
    }
    const From k = from_of<H>(a, a.k + job.group * a.k_head, a.k_page, a.k_row, job.b), v = from_of<H>(a, a.v + job.group * a.v_head, a.v_page, a.v_row, job.b);
    const bool runs = in_runs<H>(a);
    const uint32_t lds = lds_address(attention_lds);
    const bool idle = job.row_tile * W::kRows + wave * 32 >= job.rows;  // (copies, and meets the others)
    f32x16 acc[H::kBlocks];
    float m, l;

    auto pass = [&](int32_t special) __attribute__((always_inline)) {
        m = kNoMaximum;
        l = 0.f;
#pragma unroll
        for (int n = 0; n < H::kBlocks; ++n) acc[n] = f32x16{};
        if (job.begin_tile >= job.end_tile) return;
        Runs<H, W::kPlaces, W::kPlaces / W::kWaves> next;
        uint64_t there = 0, there_next = 0;
        auto copy = [&](int32_t tile) __attribute__((always_inline)) {
            const int32_t at = (tile & 1) * 2 * W::kBytes;
            if (next.good) {
                copy_runs<H, W::kCopies>(k, next, lds + at, wave * W::kCopies);
                copy_runs<H, W::kCopies>(v, next, lds + at + W::kBytes, wave * W::kCopies);
                there_next = ~0ull;
            } else {
                const Places<W::kPlaces> places(a, job.b, tile * W::kPlaces, job.end);
                copy_rows<H, W::kPlaces, W::kCopies>(a, k, places, lds + at, attention_lds + at, wave * W::kCopies);
                copy_rows<H, W::kPlaces, W::kCopies>(a, v, places, lds + at + W::kBytes, attention_lds + at + W::kBytes, wave * W::kCopies);
                there_next = W::kPlaces == 64 ? places.there : places.there | ~0ull << 32;
            }
        };
        auto look_up = [&](int32_t tile) __attribute__((always_inline)) { next.look_up(a, job.b, tile * W::kPlaces, wave * (W::kPlaces / W::kWaves), job.end, runs); };
        look_up(job.begin_tile);
        copy(job.begin_tile);
        wait_for(q);
        look_up(job.begin_tile + 1);
        for (int32_t tile = job.begin_tile; tile < job.end_tile; ++tile) {
            there = there_next;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (tile + 1 < job.end_tile) {
                copy(tile + 1);
                look_up(tile + 2);
            }
            if (special == kAll && idle) continue;
            char* keys = attention_lds + (tile & 1) * 2 * W::kBytes;
            if (special != kAll) {
                replace_values<kHalf>(keys + W::kBytes, W::kBytes, special, ldexpf(1.f, -halvings<kHalf>(a)), threadIdx.x, 256);
                __syncthreads();
            }
            const int32_t p0 = tile * W::kPlaces;
            f32x16 score[W::kBlocksOf];
            // (its products go before the softmax of the other work-group's wavefront, which goes on under them, and its first product before the other's second.  2048 x 4096 rows without such an
            // order, with the softmax last, and with both: 571, 555 and 556 us; 2 x 2048 tokens over 4000 places, as a chain, with the softmax last and with both: 328 and 315)
            __builtin_amdgcn_s_setprio(2);
            find_scores<kHalf, kSize>(keys, q, score);
            __builtin_amdgcn_s_setprio(0);
            if (p0 + W::kPlaces > row.plain || there != ~0ull) {
#pragma unroll
                for (int n = 0; n < W::kBlocksOf; ++n) score[n] = hide(score[n], (seen_of(row.sight, nodes, p0 + 32 * n) & (uint32_t)(there >> (32 * n))) >> (4 * half));
            }
            find_maxima<kHalf>(a.scale2, score, acc, m, l);
            find_weights<kHalf>(a.scale2, score, m, l);
            __builtin_amdgcn_s_setprio(1);
            add_values<kHalf, kSize>(keys + W::kBytes, score, acc);
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();
    };
    const float more = add_up(acc, halvings<kHalf>(a), pass, [](bool mine) { return __syncthreads_or(mine) != 0; });
    finish_row<kHalf, kSize>(a, acc, more, m, l, job.b, job.group, row.r, job.at * W::kRows + wave * 32 + (lane & 31), job.begin_tile < job.end_tile);
}

// ---- few rows -----------------------------------------------------------------------------------------------------------
//
// A work-group has 32 rows, and its wavefronts share out the places of its part, 32 at a time, each with copies, maxima and sums of its own; those are joined at the end, in one order.  Bound by the
// bytes of k and v: a wavefront has a block of one of them on its way while it works on the other's, without waiting for the rest.  One token of 8 sequences of up to 2000 places, 8 heads of 128 elements,
// float16: 14 us (37 MB; a launch that does nothing takes 3, and copies, products and the join each wait for what is before them); one of 32768 places, with the join, 38 us (134 MB); of 16 to up to 1500
// states, 16 heads of 64, 16 us (53 MB).  float32, 3 x 197 tokens to up to 577 states, 12 heads of 64: 21 us, 9 of them the products'.
template <bool kHalf, int kSize>
struct Few {
    static constexpr int kBytes = 32 * Head<kHalf, kSize>::kRow;  // of a block of k or v
    static constexpr int kWaves = kBytes <= 16 * 1024 ? 4 : 2;
    static constexpr int kPlaces = 32 * kWaves;                    // of a round
    static constexpr int kCopies = kBytes / 1024;
    static constexpr int kJoin = kWaves * 32 * (kSize + 4) * 4;    // the wavefronts' sums, rows not in the same banks
    static constexpr int kRing = kWaves * 2 * kBytes;
    static constexpr int kWork = kRing > kJoin ? kRing : kJoin;
    static constexpr int kLds = kWork + kWaves * 64 * 4;  // (and nodes)
};

template <bool kHalf, int kSize>
__global__ __launch_bounds__((64 * Few<kHalf, kSize>::kWaves), (Few<kHalf, kSize>::kLds <= 80 * 1024 ? 2 : 1)) void attention_places_kernel(AttentionArgs a) {
    using H = Head<kHalf, kSize>;
    using W = Few<kHalf, kSize>;
    constexpr int kWaves = W::kWaves;
    extern __shared__ __attribute__((aligned(1024))) char attention_lds[];
    float* stats = reinterpret_cast<float*>(attention_lds + W::kWork);  // [wave][m of 32 rows, l of 32 rows]
    Nodes* nodes = reinterpret_cast<Nodes*>(attention_lds + W::kWork + kWaves * 64 * 4);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
    const Job job = job_of(a, 32, W::kPlaces);
    if (a.kind == kTree && job.begin_tile < job.end_tile && job.end_tile * W::kPlaces > job.length) find_ancestors<64 * kWaves>(nodes, a.parents + (int64_t)job.b * a.T, a.T);
    const Row row = row_of(a, job, job.row_tile * 32);
    u32x4 q[H::kSteps];
    load_rows<kHalf, kSize>(a, job, row, attention_lds + wave * 2 * W::kBytes, q);
    clear_rest<H>(a, attention_lds + wave * 2 * W::kBytes, 2 * W::kBytes, lane, 64);
    const From k = from_of<H>(a, a.k + job.group * a.k_head, a.k_page, a.k_row, job.b), v = from_of<H>(a, a.v + job.group * a.v_head, a.v_page, a.v_row, job.b);
    const bool runs = in_runs<H>(a);
    char *keys = attention_lds + wave * 2 * W::kBytes, *values = keys + W::kBytes;
    const uint32_t keys_at = lds_address(keys), values_at = keys_at + W::kBytes;
    // this wavefront's blocks of 32 places: every kWaves-th, as far as there are places
    const int32_t first = job.begin_tile * kWaves + wave, last = min(job.end_tile * kWaves, (job.end + 31) / 32);
    f32x16 acc[H::kBlocks];
    float m, l;

    auto pass = [&](int32_t special) __attribute__((always_inline)) {
        m = kNoMaximum;
        l = 0.f;
#pragma unroll
        for (int n = 0; n < H::kBlocks; ++n) acc[n] = f32x16{};
        if (first >= last) return;
        Runs<H, 32, 32> next;
        uint64_t there = 0;
        auto copy = [&](const From& f, int32_t block, uint32_t lds, char* to) __attribute__((always_inline)) {
            if (next.good) {
                copy_runs<H, W::kCopies>(f, next, lds, 0);
                there = ~0ull;
            } else {
                const Places<32> places(a, job.b, block * 32, job.end);
                copy_rows<H, 32, W::kCopies>(a, f, places, lds, to, 0);
                there = places.there;
            }
        };
        next.look_up(a, job.b, first * 32, 0, job.end, runs);
        copy(k, first, keys_at, keys);
        copy(v, first, values_at, values);
        wait_for(q);
#pragma unroll 1
        for (int32_t block = first; block < last; block += kWaves) {
            const bool more = block + kWaves < last;
            const uint32_t seen_there = (uint32_t)there;
            next.look_up(a, job.b, (block + kWaves) * 32, 0, job.end, runs && more);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(W::kCopies) : "memory");  // (v's copies came behind)
            f32x16 score[1];
            find_scores<kHalf, kSize>(keys, q, score);
            const int32_t p0 = block * 32;
            if (p0 + 32 > row.plain || seen_there != ~0u) score[0] = hide(score[0], (seen_of(row.sight, nodes, p0) & seen_there) >> (4 * half));
            if (more) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                copy(k, block + kWaves, keys_at, keys);
            }
            find_maxima<kHalf>(a.scale2, score, acc, m, l);
            find_weights<kHalf>(a.scale2, score, m, l);
            if (more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(W::kCopies) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            if (special != kAll) replace_values<kHalf>(values, W::kBytes, special, ldexpf(1.f, -halvings<kHalf>(a)), lane, 64);
            add_values<kHalf, kSize>(values, score, acc);
            if (more) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                copy(v, block + kWaves, values_at, values);
            }
        }
    };
    const float more = add_up(acc, halvings<kHalf>(a), pass, [](bool mine) { return __builtin_amdgcn_ballot_w64(mine) != 0; });

    // The wavefronts' sums, relative to the largest of their maxima and divided by the sum of all weights; of those with an infinite one, what weighs nothing adds nothing.
    l = sum_of_halves(l);
    if (half == 0) {
        stats[wave * 64 + lane] = m;
        stats[wave * 64 + 32 + lane] = l;
    }
    __syncthreads();
    float most = kNoMaximum, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) most = fmaxf(most, stats[w * 64 + (lane & 31)]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += stats[w * 64 + 32 + (lane & 31)] * __builtin_amdgcn_exp2f(stats[w * 64 + (lane & 31)] - most);
    const float f = __builtin_amdgcn_exp2f(m - most), share = total == 0.f ? 0.f : more / total;
    constexpr int kPitch = kSize + 4;
    float* sums = reinterpret_cast<float*>(attention_lds);
#pragma unroll
    for (int n = 0; n < H::kBlocks; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] = f == 0.f || l == 0.f ? 0.f : acc[n][i] * f * share;
    H::in_vectors(acc, half, [&](int element, typename H::Vector v) __attribute__((always_inline)) { *reinterpret_cast<typename H::Vector*>(sums + (wave * 32 + (lane & 31)) * kPitch + element) = v; });
    __syncthreads();
    const int64_t part_row = job.at * 32;
    if (a.parts > 1 && threadIdx.x < 32) *reinterpret_cast<f32x2*>(a.part_stats + 2 * (part_row + lane)) = f32x2{most, total};
    if (a.parts > 1 && job.begin_tile >= job.end_tile) return;
    if (a.parts == 1 && a.sums != nullptr && threadIdx.x < 32 && row.r < job.rows) a.sums[((int64_t)job.b * a.groups + job.group) * job.rows + row.r] = sum_of<kHalf>(most, total);
    const int32_t rows = min(32, job.rows - job.row_tile * 32);
#pragma unroll 2
    for (int i = threadIdx.x; i < rows * (kSize / 4); i += 64 * kWaves) {
        const int r = i / (kSize / 4), e = i % (kSize / 4) * 4;
        f32x4 sum = *reinterpret_cast<const f32x4*>(sums + r * kPitch + e);
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += *reinterpret_cast<const f32x4*>(sums + (w * 32 + r) * kPitch + e);
        if (a.parts > 1) {
            *reinterpret_cast<f32x4*>(a.part_sums + (part_row + r) * kSize + e) = sum;
            continue;
        }
        const int32_t all = job.row_tile * 32 + r, t = over(all, a.by_fan), head = job.group * a.fan + (all - t * a.fan);
        char* y = a.y + job.b * a.y_batch + t * a.y_token + head * a.y_head;
        if constexpr (kHalf) store<4>(a, y, e, half4{to_half(sum[0]), to_half(sum[1]), to_half(sum[2]), to_half(sum[3])});
        else store<4>(a, y, e, sum);
    }
}

// A row's parts, by a wavefront (8 parts of 256 rows 4 us, 16 of those of 4 x 24 tokens and 32 heads 7.4): y = sum_i w_i y_i with w_i = l_i 2^(m_i - m) over the sum of those and y_i the part's own mean, in the order of the parts.
template <bool kHalf, int kSize>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a) {
    constexpr int kOf = kSize / 64;  // elements of a lane, next to each other
    const int lane = threadIdx.x & 63;
    const int32_t rows = a.T * a.fan;
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= (int64_t)a.B * a.groups * rows) return;
    const int32_t of = (int32_t)(row / rows), r = (int32_t)(row % rows), t = over(r, a.by_fan), b = over(of, a.by_groups), head = (of - b * a.groups) * a.fan + (r - t * a.fan);
    const int32_t tile = r / a.tile_rows;
    const int64_t first = (((int64_t)of * a.row_tiles + tile) * a.parts) * a.tile_rows + (r - tile * a.tile_rows);
    f32x2 stat = {kNoMaximum, 0.f};
    if (lane < a.parts) stat = *reinterpret_cast<const f32x2*>(a.part_stats + 2 * (first + (int64_t)lane * a.tile_rows));
    float m = stat[1] != 0.f ? stat[0] : kNoMaximum;
#pragma unroll
    for (int d = 32; d; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
    const float weight = stat[1] != 0.f ? __builtin_amdgcn_exp2f(stat[0] - m) : 0.f;
    // (A part whose sum is no number has a score that is none, which its maximum does not show: the row has no result, whatever that part would weigh.)
    float l = weight == 0.f && stat[1] == stat[1] ? 0.f : stat[1] * weight;
#pragma unroll
    for (int d = 32; d; d /= 2) l += __shfl_xor(l, d);
    const float part = weight == 0.f || l == 0.f ? 0.f : stat[1] * weight / l;
    float sum[kOf] = {};
    typedef float Of __attribute__((ext_vector_type(kOf)));
    // (eight parts' loads under way at once; a part without weight may hold anything)
    const float* from = a.part_sums + first * kSize + lane * kOf;
    const int64_t next = (int64_t)a.tile_rows * kSize;
    constexpr int kAtOnce = 8;
    for (int p = 0; p < a.parts; p += kAtOnce) {
        Of v[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) v[i] = *reinterpret_cast<const Of*>(from + min(p + i, a.parts - 1) * next);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const float w = p + i < a.parts ? __shfl(part, (p + i) & 63) : 0.f;
#pragma unroll
            for (int j = 0; j < kOf; ++j) sum[j] = w == 0.f ? sum[j] : __builtin_fmaf(w, v[i][j], sum[j]);
        }
    }
    if (a.sums != nullptr && lane == 0) a.sums[row] = sum_of<kHalf>(m, l);
    char* y = a.y + b * a.y_batch + t * a.y_token + head * a.y_head;
#pragma unroll
    for (int j = 0; j < kOf; ++j) {
        if (lane * kOf + j >= a.D) break;
        if constexpr (kHalf) reinterpret_cast<_Float16*>(y)[lane * kOf + j] = to_half(sum[j]);
        else reinterpret_cast<float*>(y)[lane * kOf + j] = sum[j];
    }
}

// The weights that each place is given, over a group's rows, of which the first pass has left m + log2(l).  The scores are made again, here as q k^T: a lane has one place, and
// its weights add up without another lane's.  Rows lie in LDS, 128 at a time; a wavefront goes over blocks of 32 places with copies of its own.  Bound by the bytes of k and the wait for them:
// 4 x 24 tokens over 32768 places, 32 heads over 8 of 128 elements, float16, 66 us, 4.1 TB/s.  (With the last places first, of which the last level of cache has some from the first pass, the same.)
template <bool kHalf, int kSize>
struct Mass {
    static constexpr int kBytes = 32 * Head<kHalf, kSize>::kRow;  // of a block of k
    static constexpr int kRows = kBytes <= 16 * 1024 ? 128 : 64;
    static constexpr int kWaves = kBytes <= 16 * 1024 ? 4 : 2, kThreads = 64 * kWaves;
    static constexpr int kCopies = kBytes / 1024;
    static constexpr int kOfRows = kRows * Head<kHalf, kSize>::kRow;
    static constexpr int kLds = kOfRows + kWaves * (kBytes + 256) + kRows * 12;  // (and nodes)
};

template <bool kHalf, int kSize>
__global__ __launch_bounds__((Mass<kHalf, kSize>::kThreads)) void attention_mass_kernel(AttentionArgs a, int32_t runs_of_places) {
    using H = Head<kHalf, kSize>;
    using W = Mass<kHalf, kSize>;
    extern __shared__ __attribute__((aligned(1024))) char attention_lds[];
    float* before = reinterpret_cast<float*>(attention_lds + W::kOfRows + W::kWaves * W::kBytes);  // what the places have already: [wave][64]
    float* less = before + W::kWaves * 64;  // of the rows: m + log2(l)
    int32_t* limits = reinterpret_cast<int32_t*>(less + W::kRows);                                               // what they see, as in Sight
    int32_t* sees = limits + W::kRows;
    Nodes* nodes = reinterpret_cast<Nodes*>(sees + W::kRows);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    Job job;
    const int32_t of = uniform(blockIdx.x / runs_of_places), run = blockIdx.x - of * runs_of_places;
    job.b = over(of, a.by_groups);
    job.group = of - job.b * a.groups;
    job.rows = a.T * a.fan;
    job.length = length_of(a, job.b);
    job.count = count_of(a, job.b);
    job.end = min(job.length + job.count, a.places);
    // a run of blocks of 32 places, of which the wavefronts have every kWaves-th
    const int32_t blocks = (job.end + 31) / 32, each = uniform(((blocks + runs_of_places - 1) / runs_of_places + W::kWaves - 1) / W::kWaves * W::kWaves), last = min((run + 1) * each, blocks);
    if (run * each >= last) return;
    if (a.kind == kTree && last * 32 > job.length) find_ancestors<W::kThreads>(nodes, a.parents + (int64_t)job.b * a.T, a.T);
    const From k = from_of<H>(a, a.k + job.group * a.k_head, a.k_page, a.k_row, job.b);
    const bool runs = in_runs<H>(a);
    char* keys = attention_lds + W::kOfRows + wave * W::kBytes;
    clear_rest<H>(a, keys, W::kBytes, lane, 64);
    const uint32_t keys_at = lds_address(keys), before_at = lds_address(before) + wave * 256;
    const int32_t row_bytes = a.D * H::kElement, used = job.count * a.fan;
    for (int32_t r0 = 0; r0 < used; r0 += W::kRows) {
        __syncthreads();
        for (int32_t i = threadIdx.x; i < W::kRows * H::kChunks; i += W::kThreads) {
            const int32_t r = r0 + i / H::kChunks, c = i % H::kChunks, t = over(r, a.by_fan), head = job.group * a.fan + (r - t * a.fan);
            reinterpret_cast<u32x4*>(attention_lds)[i / H::kChunks * H::kChunks + (c ^ H::turned(i / H::kChunks))] =
                chunk_of<kHalf>(a.q + job.b * a.q_batch + t * a.q_token + head * a.q_head, c * 16, row_bytes, a.q_whole, r < used);
        }
        static_assert(W::kRows <= W::kThreads, "a lane to a row");
        if (threadIdx.x < W::kRows) {
            const int32_t r = r0 + threadIdx.x, t = over(r, a.by_fan);
            const Sight sight = sight_of(a, t, job.length, job.count);
            less[threadIdx.x] = r < used ? a.sums[(int64_t)of * job.rows + r] : INFINITY;
            limits[threadIdx.x] = sight.limit;
            sees[threadIdx.x] = sight.node;
        }
        __syncthreads();
        const int32_t row_blocks = (min(used - r0, W::kRows) + 31) / 32;
        // (the rows of a chain do not see places behind the last of them)
        const int32_t seen_end = a.kind == kChain ? min(job.end, job.length + over(min(r0 + W::kRows, used) - 1, a.by_fan) + 1) : job.end;
        Runs<H, 32, 32> next;
        uint64_t there = 0, there_next = 0;
        float* mass = a.mass + job.b * a.mass_batch + job.group * a.mass_head;
        auto copy = [&](int32_t block) __attribute__((always_inline)) {
            if (next.good) {
                copy_runs<H, W::kCopies>(k, next, keys_at, 0);
                there_next = ~0ull;
            } else {
                const Places<32> places(a, job.b, block * 32, job.end);
                copy_rows<H, 32, W::kCopies>(a, k, places, keys_at, keys, 0);
                there_next = places.there;
            }
            // (tokens' own places are set by the first of the rows)
            const int32_t p = block * 32 + (lane & 31);
            copy_number_to_lds(p < job.length || (r0 > 0 && p < job.end) ? mass + p : reinterpret_cast<const float*>(kZeros), before_at);
        };
        const int32_t first = run * each + wave;
        if (first >= last) continue;
        next.look_up(a, job.b, first * 32, 0, job.end, runs);
        copy(first);
#pragma unroll 1
        for (int32_t block = first; block < last; block += W::kWaves) {
            const bool more = block + W::kWaves < last;
            const int32_t p0 = block * 32, p = p0 + (lane & 31);
            there = there_next;
            next.look_up(a, job.b, (block + W::kWaves) * 32, 0, job.end, runs && more);
            const bool mine = ((there >> lane) & 1) && half == 0;
            // the block goes into registers, and the next one's copies into its place are on their way while it is worked on
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            const float so_far = before[wave * 64 + lane];
            u32x4 kf[H::kSteps];
            {
                uint32_t at = keys_at + (lane & 31) * H::kRow + ((half ^ H::turned(lane & 31)) << 4);
#pragma unroll
                for (int s = 0; s < H::kSteps; ++s) kf[s] = *lds_pointer<u32x4>(at ^ (s << 5));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (more) copy(block + W::kWaves);
            float total = 0.f;
            const bool plain = p0 + 32 <= job.length;
#pragma unroll 1
            for (int rb = 0; rb < (p0 < seen_end ? row_blocks : 0); ++rb) {
                f32x16 score = {};
                uint32_t at = lds_address(attention_lds) + (rb * 32 + (lane & 31)) * H::kRow + ((half ^ H::turned(lane & 31)) << 4);
                asm volatile("" : "+v"(at));
                constexpr int kAhead = kHalf ? 4 : 2;
                u32x4 q[kAhead + 1];
                in_steps<H::kSteps, kAhead>([&](int s) __attribute__((always_inline)) { q[s % (kAhead + 1)] = *lds_pointer<u32x4>(at ^ (s << 5)); },
                                            [&](int s) __attribute__((always_inline)) { score = score_of<kHalf>(q[s % (kAhead + 1)], kf[s], score); });
                const int row = rb * 32 + 4 * half;
                auto add = [&](uint32_t seen, auto some) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const f32x4 l = *reinterpret_cast<const f32x4*>(less + row + 2 * i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(score[i + j], a.scale2, -l[j]));
                            total += !decltype(some)::value || ((seen >> (i + j)) & 1) ? w : 0.f;
                        }
                    }
                };
                if (plain && r0 + rb * 32 + 32 <= used) {
                    add(~0u, std::false_type());
                } else {  // (a weight that is not seen is none, also of a row that has no number for its sum)
                    uint32_t seen = 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) seen |= (uint32_t)(p < limits[row + 8 * (i >> 2) + (i & 3)]) << i;
                    if (a.kind == kTree && p0 + 32 > job.length) {
                        const int32_t other = max(0, min(p - job.length, job.count - 1));  // the node that lies there
                        const uint32_t is = (p >= job.length) & (p < job.end);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int32_t node = sees[row + 8 * (i >> 2) + (i & 3)];
                            seen |= (((nodes->sees[max(node, 0)][other >> 5] >> (other & 31)) & is & (uint32_t)(node >= 0)) << i);
                        }
                    }
                    add(seen, std::true_type());
                }
            }
            total = sum_of_halves(total);
            if (mine) mass[p] = so_far + total;
        }
    }
    // (places of a sequence without tokens stay as they are)
}

// The same of many rows: a work-group has the keys of a few blocks of places in LDS, and its wavefronts go over the rows, every fourth 32 of them, with scores as in the first pass: a lane has one row, whose
// m + log2(l) is one number, and adds up the places' weights over its rows in registers; lanes and wavefronts are added at the end, in one order.  2 x 2048 tokens over up to 4000 places, 32 heads over 8 of 128 elements, float16,
// 188 us (by places, whose lanes read each row's number from LDS, 608).  Bound by vector and matrix instructions, which take turns: by counters (a launch of 206 us) the vector units are busy for 51 % of the time (5.4 instructions to a
// score; its exponential alone 16 %) and the matrix units for 32 %, with up to two wavefronts to a SIMD, which wait 19 % of their time, for the next rows of q among others.  float32, 2 x 512 tokens: 295 us, matrix units busy for 60 %.
template <bool kHalf, int kSize, int kBlocks>
struct MassRows {
    static constexpr int kWaves = 4, kPlaces = 32 * kBlocks;
    static constexpr int kBytes = kPlaces * Head<kHalf, kSize>::kRow;
    static constexpr int kLookUp = kPlaces < 64 ? kPlaces : 64;   // places that a wavefront looks up at once, where they do not come in runs
    static constexpr int kSums = kWaves * kPlaces * 4;
    static constexpr int kLds = kBytes + kSums;  // (and nodes)
};
// Blocks of a work-group: rows of q are read once for all of them.
template <bool kHalf, int kSize>
constexpr int kMassBlocks = Head<kHalf, kSize>::kRow <= 256 ? 4 : Head<kHalf, kSize>::kRow <= 512 ? 2 : 1;

template <bool kHalf, int kSize, int kBlocks>
__global__ __launch_bounds__(256, (Head<kHalf, kSize>::kRow <= 512 ? 2 : 1)) void attention_mass_rows_kernel(AttentionArgs a, int32_t tiles) {
    using H = Head<kHalf, kSize>;
    using W = MassRows<kHalf, kSize, kBlocks>;
    constexpr int kOfWave = W::kPlaces / W::kWaves, kParts = W::kPlaces / W::kLookUp;
    extern __shared__ __attribute__((aligned(1024))) char attention_lds[];
    float* sums = reinterpret_cast<float*>(attention_lds + W::kBytes);  // [wave][place]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    Nodes* nodes = reinterpret_cast<Nodes*>(attention_lds + W::kLds);
    // (all tiles of a head of k on one XCD, whose L2 then has its rows of q)
    const int32_t whole_sets = a.B * a.groups / 8 * 8;
    const uint32_t whole = (uint32_t)whole_sets * (uint32_t)tiles, turn = blockIdx.x < whole ? blockIdx.x >> 3 : blockIdx.x - whole, of_turn = uniform(turn / (uint32_t)tiles);
    const int32_t of = blockIdx.x < whole ? of_turn * 8 + (blockIdx.x & 7) : whole_sets + of_turn, p0 = (int32_t)(turn - of_turn * tiles) * W::kPlaces;
    Job job;
    job.b = over(of, a.by_groups);
    job.group = of - job.b * a.groups;
    job.rows = a.T * a.fan;
    job.length = length_of(a, job.b);
    job.count = count_of(a, job.b);
    job.end = min(job.length + job.count, a.places);
    if (p0 >= job.end || job.count == 0) return;
    if (a.kind == kTree && p0 + W::kPlaces > job.length) find_ancestors<256>(nodes, a.parents + (int64_t)job.b * a.T, a.T);
    if (a.D * H::kElement != H::kRow) {
        clear_rest<H>(a, attention_lds, W::kBytes, threadIdx.x, 256);
        __syncthreads();
    }
    const From k = from_of<H>(a, a.k + job.group * a.k_head, a.k_page, a.k_row, job.b);
    const uint32_t lds = lds_address(attention_lds);
    uint64_t there[kParts];
    Runs<H, W::kPlaces, kOfWave> keys;
    keys.look_up(a, job.b, p0, wave * kOfWave, job.end, in_runs<H>(a));
    if (keys.good) {
        constexpr int kCopies = W::kBytes / 1024 / W::kWaves;
        copy_runs<H, kCopies>(k, keys, lds, wave * kCopies);
#pragma unroll
        for (int i = 0; i < kParts; ++i) there[i] = ~0ull;
    } else {
        constexpr int kCopies = W::kLookUp * H::kRow / 1024 / W::kWaves;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            const int32_t at = i * W::kLookUp * H::kRow;
            const Places<W::kLookUp> places(a, job.b, p0 + i * W::kLookUp, job.end);
            copy_rows<H, W::kLookUp, kCopies>(a, k, places, lds + at, attention_lds + at, wave * kCopies);
            there[i] = places.there;
        }
    }
    const int32_t used = job.count * a.fan, row_bytes = a.D * H::kElement;
    // (the rows of a chain that come before the first of these places do not see them)
    int32_t first = (a.kind == kChain ? max(0, p0 - job.length) : 0) * a.fan / 32 * 32 + wave * 32;
    f32x16 total[kBlocks];
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) total[n] = f32x16{};
    struct Rows {
        float less;  // m + log2(l)
        u32x4 q[H::kSteps];
    };
    auto load = [&](Rows& r, int32_t at) __attribute__((always_inline)) {
        const Row row = row_of(a, job, at);
        r.less = a.sums[(int64_t)of * job.rows + min(row.r, job.rows - 1)];
        const char* from = a.q + job.b * a.q_batch + row.t * a.q_token + row.head * a.q_head;
        if (a.q_whole) {
#pragma unroll
            for (int s = 0; s < H::kSteps; ++s) r.q[s] = chunk_of<kHalf>(from, (2 * s + half) * 16, row_bytes, true);
        } else {
#pragma unroll
            for (int s = 0; s < H::kSteps; ++s) r.q[s] = chunk_of<kHalf>(from, (2 * s + half) * 16, row_bytes, false);
        }
    };
    auto add = [&](const Rows& r, int32_t at) __attribute__((always_inline)) {
        constexpr int kAtOnce = kBlocks < 2 ? 1 : 2;
        const Row row = row_of(a, job, at);
#pragma unroll
        for (int n0 = 0; n0 < kBlocks; n0 += kAtOnce) {
            f32x16 score[kAtOnce];
            __builtin_amdgcn_s_setprio(1);
            find_scores<kHalf, kSize>(attention_lds + n0 * 32 * H::kRow, r.q, score);
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) {
                const int32_t p = p0 + 32 * (n0 + n);
                const uint32_t here = (uint32_t)(there[(n0 + n) / 2 % kParts] >> (32 * ((n0 + n) & 1)));
                uint32_t seen = ~0u;
                if (p + 32 > row.plain || at + 32 > used || here != ~0u) {
                    seen = (seen_of(row.sight, nodes, p) & here) >> (4 * half);
                    seen = row.r < used ? seen : 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {  // (a weight that is not seen is none, also of a row that has no number for its sum)
                        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(score[n][i], a.scale2, -r.less));
                        total[n0 + n][i] += (seen >> (8 * (i >> 2) + (i & 3))) & 1 ? w : 0.f;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) total[n0 + n][i] += __builtin_amdgcn_exp2f(__builtin_fmaf(score[n][i], a.scale2, -r.less));
                }
            }
        }
    };
    Rows now;
    load(now, min(first, used - 1));
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll 1
    for (; first < used; first += W::kWaves * 32) {
        add(now, first);
        load(now, min(first + W::kWaves * 32, used - 1));  // (a second set of registers, for the next rows under these, gained nothing)
    }
    // Lanes of a half have the same places: eight of their sixteen go to the lane 16 on and come from it, four to the one 8 on, and so on, until each has one.
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = total[n][i];
#pragma unroll
        for (int w = 8; w; w /= 2) {
            const bool upper = lane & (2 * w);
#pragma unroll
            for (int i = 0; i < w; ++i) {
                const float mine = upper ? v[i + w] : v[i], other = upper ? v[i] : v[i + w];
                v[i] = mine + __shfl_xor(other, 2 * w);
            }
        }
        v[0] += __shfl_xor(v[0], 1);
        const int i = (lane >> 1) & 15;
        if ((lane & 1) == 0) sums[wave * W::kPlaces + 32 * n + 8 * (i >> 2) + 4 * half + (i & 3)] = v[0];
    }
    __syncthreads();
    const int32_t p = p0 + (int)threadIdx.x;
    if (threadIdx.x >= W::kPlaces || p >= job.end || place_in(a, job.b, p).page < 0) return;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < W::kWaves; ++w) sum += sums[w * W::kPlaces + threadIdx.x];
    float* to = a.mass + job.b * a.mass_batch + job.group * a.mass_head + p;
    *to = (p < job.length ? *to : 0.f) + sum;
}

// More than 64 KB has to be asked for, on every device: always for the largest tree, so that threads that call at once ask for the same.
inline int ask_for_lds(const void* kernel, int lds) {
    if (lds + (int)sizeof(Nodes) > 65536) CHX_HIP_CALL(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds + (int)sizeof(Nodes)));
    return CHX_HIP_OK;
}

template <bool kHalf, int kSize>
int attend_of(const AttentionArgs& a, hipStream_t s) {
    using W = Tile<kHalf, kSize>;
    using F = Few<kHalf, kSize>;
    const bool few = a.tile_rows == 32;
    auto kernel = few ? attention_places_kernel<kHalf, kSize> : attention_rows_kernel<kHalf, kSize>;
    const int lds = few ? F::kLds : W::kLds;
    CHX_PROPAGATE(ask_for_lds(reinterpret_cast<const void*>(kernel), lds));
    kernel<<<(unsigned)((int64_t)a.B * a.groups * a.parts * a.row_tiles), few ? 64 * F::kWaves : 256, lds + nodes_bytes(a), s>>>(a);
    return launch_check(few ? "attention_places_kernel" : "attention_rows_kernel");
}
template <bool kHalf, int kSize>
int join_of(const AttentionArgs& a, hipStream_t s) {
    attention_join_kernel<kHalf, kSize><<<(unsigned)(((int64_t)a.B * a.groups * a.T * a.fan + 3) / 4), 256, 0, s>>>(a);
    return launch_check("attention_join_kernel");
}
template <bool kHalf, int kSize, int kBlocks>
int mass_rows_of(const AttentionArgs& a, int64_t groups, int64_t tiles, hipStream_t s) {
    using W = MassRows<kHalf, kSize, kBlocks>;
    auto kernel = attention_mass_rows_kernel<kHalf, kSize, kBlocks>;
    CHX_PROPAGATE(ask_for_lds(reinterpret_cast<const void*>(kernel), W::kLds));
    kernel<<<(unsigned)(groups * tiles), 256, W::kLds + nodes_bytes(a), s>>>(a, (int32_t)tiles);
    return launch_check("attention_mass_rows_kernel");
}
template <bool kHalf, int kSize>
int mass_of(const AttentionArgs& a, hipStream_t s) {
    using W = Mass<kHalf, kSize>;
    const int64_t groups = (int64_t)a.B * a.groups, most = ((int64_t)a.places + 127) / 128, blocks = ((int64_t)a.places + 31) / 32;
    // By rows where there are many.  us by places / by rows, 128 elements of float16, 8 heads: 2 x 2048 tokens x 4 rows over 4000 places 608 / 185, 2 x 256 x 4 over 4000 79 / 29, 16 x 64 x 4 over 300
    // 27 / 18, but 40 x 8 over 30000 (whose keys take the time) 55 / 69.
    const int64_t rows = (int64_t)a.T * a.fan;
    if (rows > 384 || (rows > 128 && a.places < 8192)) {
        // Blocks by themselves where there are few work-groups of several.  us of several / one: float16, 160 work-groups of several 33 / 51, 56 of them 40 / 34; float32, 192 of them 47 / 37.
        constexpr int kBlocks = kMassBlocks<kHalf, kSize>;
        const int64_t wide = groups * ((blocks + kBlocks - 1) / kBlocks);
        if (kBlocks > 1 && wide < (kHalf ? 128 : 256)) return mass_rows_of<kHalf, kSize, 1>(a, groups, blocks, s);
        return mass_rows_of<kHalf, kSize, kBlocks>(a, groups, (blocks + kBlocks - 1) / kBlocks, s);
    }
    // By places, in runs of them: as many as give each compute unit two work-groups, of at least 128 places (a block to each wavefront).
    int64_t runs = (512 + groups - 1) / groups;
    runs = runs > most ? most : runs;
    auto kernel = attention_mass_kernel<kHalf, kSize>;
    CHX_PROPAGATE(ask_for_lds(reinterpret_cast<const void*>(kernel), W::kLds));
    kernel<<<(unsigned)(groups * runs), W::kThreads, W::kLds + nodes_bytes(a), s>>>(a, (int32_t)runs);
    return launch_check("attention_mass_kernel");
}

}  // namespace

template <bool kHalf>
int AttentionKernels<kHalf>::attend(const AttentionArgs& a, int size, hipStream_t s) {
    return size == 64 ? attend_of<kHalf, 64>(a, s) : size == 128 ? attend_of<kHalf, 128>(a, s) : attend_of<kHalf, 256>(a, s);
}
template <bool kHalf>
int AttentionKernels<kHalf>::join(const AttentionArgs& a, int size, hipStream_t s) {
    return size == 64 ? join_of<kHalf, 64>(a, s) : size == 128 ? join_of<kHalf, 128>(a, s) : join_of<kHalf, 256>(a, s);
}
template <bool kHalf>
int AttentionKernels<kHalf>::mass(const AttentionArgs& a, int size, hipStream_t s) {
    return size == 64 ? mass_of<kHalf, 64>(a, s) : size == 128 ? mass_of<kHalf, 128>(a, s) : mass_of<kHalf, 256>(a, s);
}

}  // namespace chx

