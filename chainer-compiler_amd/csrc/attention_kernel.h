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
#include <type_traits>

#include "attention.h"

namespace chx {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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
    // Element of the head that result (block, i) of a lane is; i = 0..15.
    static __device__ __forceinline__ int element(int block, int i, int half) {
        const int r = 8 * (i >> 2) + 4 * half + (i & 3);
        return kHalf ? 32 * block + r : kWide * r + block % kWide + 32 * kWide * (block / kWide);
    }
};

// 16 bytes of a row of `bytes` bytes from byte `at` on, zeros behind its end.
template <bool kHalf>
__device__ __forceinline__ u32x4 chunk_of(const char* row, int32_t at, int32_t bytes, bool whole) {
    u32x4 v = {0, 0, 0, 0};
    if (whole) return at < bytes ? *reinterpret_cast<const u32x4*>(row + at) : v;
#pragma unroll
    for (int j = 0; j < (kHalf ? 8 : 4); ++j) {
        const int32_t b = at + j * (kHalf ? 2 : 4);
        if (b >= bytes) break;
        if constexpr (kHalf) v[j / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(row + b) << (16 * (j & 1));
        else v[j] = *reinterpret_cast<const uint32_t*>(row + b);
    }
    return v;
}

__device__ __forceinline__ int32_t length_of(const AttentionArgs& a, int32_t b) {
    return a.lengths ? max(0, min(a.lengths[b], a.places)) : a.places;
}
__device__ __forceinline__ int32_t count_of(const AttentionArgs& a, int32_t b) {
    return a.counts ? max(0, min(a.counts[b], a.T)) : a.T;
}

__device__ __forceinline__ Place place_in(const AttentionArgs& a, int32_t b, int32_t p) {
    return a.tables ? place_of(a, b, p) : Place{b, p};
}

// Which nodes each node of a tree sees: words of 32 bits, of all nodes, in LDS.  Every step doubles the ancestors that a node knows of.
struct Nodes {
    uint32_t sees[kMostNodes][kMostNodes / 32];
    int16_t up[kMostNodes];
};
__device__ __forceinline__ void find_ancestors(Nodes* nodes, const int32_t* parents, int32_t T) {
    const int i = threadIdx.x;
    const int words = (T + 31) / 32;
    if (i < T) {
        const int32_t p = parents[i];
        nodes->up[i] = (int16_t)(p >= 0 && p < i ? p : -1);
        for (int w = 0; w < words; ++w) nodes->sees[i][w] = w == i / 32 ? 1u << (i & 31) : 0;
    }
    __syncthreads();
    for (int reach = 1; reach < T; reach *= 2) {
        uint32_t more[kMostNodes / 32];
        int32_t up = -1, next = -1;
        if (i < T) up = nodes->up[i];
        if (up >= 0) {
            next = nodes->up[up];
#pragma unroll
            for (int w = 0; w < kMostNodes / 32; ++w) more[w] = w < words ? nodes->sees[up][w] : 0;
        }
        __syncthreads();
        if (up >= 0) {
            nodes->up[i] = (int16_t)next;
#pragma unroll
            for (int w = 0; w < kMostNodes / 32; ++w)
                if (w < words) nodes->sees[i][w] |= more[w];
        }
        __syncthreads();
    }
}

// What a row sees: places below `limit`, and of a tree's nodes, which lie from `length` on, those that its own node does.
struct Sight {
    int32_t limit, length, count;
    int32_t node;  // -1: none
};
__device__ __forceinline__ Sight sight_of(const AttentionArgs& a, int32_t t, int32_t length, int32_t count) {
    if (t >= count) return {0, length, count, -1};
    return {a.kind == kChain ? length + t + 1 : length, length, count, a.kind == kTree ? t : -1};
}
// Which of the places p0 to p0 + 31 a row sees, a bit each.  (A node's words have only nodes before it and itself, all below count.)
__device__ __forceinline__ uint32_t seen_of(const Sight& s, const Nodes* nodes, int32_t p0) {
    const int32_t below = s.limit - p0;
    uint32_t seen = below >= 32 ? ~0u : below > 0 ? (1u << below) - 1 : 0;
    const int32_t i = p0 - s.length;  // the node that lies at p0
    if (s.node >= 0 && i > -32 && i < s.count) {
        const uint32_t* words = nodes->sees[s.node];
        const uint64_t two = i < 0 ? (uint64_t)words[0] << 32 : words[i >> 5] | (uint64_t)words[min((i >> 5) + 1, kMostNodes / 32 - 1)] << 32;
        seen |= (uint32_t)(two >> (i & 31));
    }
    return seen;
}

// Tiles that the maximum may lag behind by: weights are then up to 2^kLag, and kept that much and kRaise higher than they are in relation to the largest, so that few of those
// of float16 fall below its normal numbers (2^-14): 2^-20 of the largest does.
constexpr float kLag = 8.f;
template <bool kHalf>
constexpr float kRaise = kHalf ? 6.f : 0.f;
constexpr float kNoMaximum = -3e38f;

// The largest of a lane and the one that has the row's other scores.
__device__ __forceinline__ float with_other_half(float v) {
    return __shfl_xor(v, 32);
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

template <bool kHalf, int kSize>
struct Tile {
    static constexpr int kWaves = 4, kRowsOfWave = 32, kRows = kWaves * kRowsOfWave;
    static constexpr int kKeyBlocks = kHalf || kSize < 256 ? 2 : 1;  // of 32 places
    static constexpr int kKeys = 32 * kKeyBlocks;
    static constexpr int kBytes = kKeys * Head<kHalf, kSize>::kRow;  // of k or v
    static constexpr int kLds = 2 * kBytes + (int)sizeof(Nodes);
};

// One work-group: 128 rows, four wavefronts with 32 each, and the places of one part.  k and v go through LDS.
template <bool kHalf, int kSize>
__global__ __launch_bounds__(256) void attention_kernel(AttentionArgs a) {
    using H = Head<kHalf, kSize>;
    using W = Tile<kHalf, kSize>;
    constexpr int kSteps = H::kSteps, kBlocks = H::kBlocks, kKeyBlocks = W::kKeyBlocks, kKeys = W::kKeys;
    extern __shared__ __attribute__((aligned(128))) char attention_lds[];
    char *k_lds = attention_lds, *v_lds = attention_lds + W::kBytes;
    Nodes* nodes = reinterpret_cast<Nodes*>(attention_lds + 2 * W::kBytes);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int32_t part = blockIdx.x % a.parts, of_tile = blockIdx.x / a.parts, row_tile = of_tile % a.row_tiles;
    const int32_t b = of_tile / a.row_tiles / a.groups, group = of_tile / a.row_tiles % a.groups;
    const int32_t rows = a.T * a.fan, length = length_of(a, b), count = count_of(a, b);
    const int32_t first_row = row_tile * W::kRows, r = first_row + wave * W::kRowsOfWave + (lane & 31);
    const int32_t t = r < rows ? r / a.fan : a.T, head = group * a.fan + (r - t * a.fan);
    // the places that any row of the work-group sees
    const int32_t last_t = min((min(first_row + W::kRows, rows) - 1) / a.fan, count - 1), first_t = first_row / a.fan;
    int32_t end = last_t < first_t ? 0 : a.kind == kCross ? length : a.kind == kChain ? length + last_t + 1 : length + count;
    end = min(end, a.places);
    const int32_t tiles = (end + kKeys - 1) / kKeys, each = (tiles + a.parts - 1) / a.parts;
    const int32_t begin_tile = part * each, end_tile = min(begin_tile + each, tiles);
    const bool any_drafted = a.kind == kTree && end_tile * kKeys > length && begin_tile < end_tile;
    if (any_drafted) find_ancestors(nodes, a.parents + (int64_t)b * a.T, a.T);
    const Sight sight = sight_of(a, t, length, count);
    // places below this are seen by all rows of the wavefront
    int32_t plain = sight.limit;
#pragma unroll
    for (int d = 16; d; d /= 2) plain = min(plain, __shfl_xor(plain, d));
    plain = __builtin_amdgcn_readfirstlane(plain);

    const int32_t row_bytes = a.D * H::kElement;
    u32x4 q[kSteps];
    {
        const char* at = a.q + b * a.q_batch + t * a.q_token + head * a.q_head;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q[s] = r < rows ? chunk_of<kHalf>(at, (2 * s + half) * 16, row_bytes, a.q_whole) : u32x4{0, 0, 0, 0};
    }

    f32x16 acc[kBlocks];
    float m, l;
    uint32_t marks[3][kBlocks / 2];  // a bit for each result: whether inf, -inf, NaN of v have weight in it
    // A result that is not finite has one of v that is not, or 0 times one: places of no weight add nothing, whatever they hold.  Then the sums are made
    // again, first of what is inf, -inf and NaN, as ones, then of the rest.
    for (int special = 0; special < 5; ++special) {
        m = kNoMaximum;
        l = 0.f;
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) acc[n] = f32x16{};
        for (int32_t tile = begin_tile; tile < end_tile; ++tile) {
            const int32_t p0 = tile * kKeys;
            __syncthreads();
            for (int i = threadIdx.x; i < kKeys * H::kChunks; i += 256) {
                const int row = i / H::kChunks, at = (i % H::kChunks ^ H::turned(row)) * 16;
                u32x4 kc = {0, 0, 0, 0}, vc = {0, 0, 0, 0};
                if (p0 + row < end) {
                    const Place p = place_in(a, b, p0 + row);
                    if (p.page >= 0) {
                        kc = chunk_of<kHalf>(a.k + p.page * a.k_page + p.row * a.k_row + group * a.k_head, at, row_bytes, a.k_whole);
                        vc = chunk_of<kHalf>(a.v + p.page * a.v_page + p.row * a.v_row + group * a.v_head, at, row_bytes, a.k_whole);
                    }
                }
                *reinterpret_cast<u32x4*>(k_lds + i * 16) = kc;
                *reinterpret_cast<u32x4*>(v_lds + i * 16) = vc;
            }
            const int32_t mine = p0 + (lane & (kKeys - 1));
            const uint64_t there = __builtin_amdgcn_ballot_w64(mine < end && place_in(a, b, mine).page >= 0);
            __syncthreads();

            f32x16 score[kKeyBlocks];
#pragma unroll
            for (int n = 0; n < kKeyBlocks; ++n) {
                score[n] = f32x16{};
                const int row = n * 32 + (lane & 31);
                const char* at = k_lds + row * H::kRow;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    const u32x4 kc = *reinterpret_cast<const u32x4*>(at + (((2 * s + half) ^ H::turned(row)) << 4));
                    score[n] = score_of<kHalf>(kc, q[s], score[n]);
                }
            }
            constexpr uint64_t kAll = kKeys == 64 ? ~0ull : (1ull << (kKeys & 63)) - 1;
            if (p0 + kKeys > plain || (there & kAll) != kAll) {
#pragma unroll
                for (int n = 0; n < kKeyBlocks; ++n) score[n] = hide(score[n], (seen_of(sight, nodes, p0 + 32 * n) & (uint32_t)(there >> (32 * n))) >> (4 * half));
            }
            float most = score[0][0];
#pragma unroll
            for (int n = 0; n < kKeyBlocks; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) most = fmaxf(most, score[n][i]);
            most = fmaxf(most, with_other_half(most)) * a.scale2;
            if (__builtin_amdgcn_ballot_w64(most > m + kLag)) {
                const float next = fmaxf(m, most), f = __builtin_amdgcn_exp2f(m - next);
                l *= f;
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) acc[n] *= f;
                m = next;
            }
            const float less = m - kRaise<kHalf>;
#pragma unroll
            for (int n = 0; n < kKeyBlocks; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    score[n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[n][i], a.scale2, -less));
                    l += score[n][i];
                }

            auto second = [&](auto replaced) __attribute__((always_inline)) {
                if constexpr (kHalf) {
#pragma unroll
                    for (int kb = 0; kb < 2 * kKeyBlocks; ++kb) {
                        half8 w;
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] = (_Float16)score[kb >> 1][8 * (kb & 1) + j];
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
                            union {
                                short4v part[2];
                                half8 whole;
                            } vf;
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int row = kb * 16 + e * 8 + 4 * half + ((lane & 15) >> 2), c = 4 * n + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                                const char* at = v_lds + row * H::kRow + ((c ^ H::turned(row)) << 4) + 8 * (lane & 1);
                                vf.part[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)at);
                            }
#pragma unroll
                            for (int j = 0; j < 8; ++j) vf.whole[j] = (_Float16)replaced((float)vf.whole[j]);
                            acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf.whole, w, acc[n], 0, 0, 0);
                        }
                    }
                } else {
                    constexpr int kWide = H::kWide;
#pragma unroll
                    for (int n = 0; n < kKeyBlocks; ++n)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int row = n * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
#pragma unroll
                            for (int w = 0; w < kBlocks / kWide; ++w) {
                                const int at = (kWide * (lane & 31) + 32 * kWide * w) * 4;
                                const char* from = v_lds + row * H::kRow + (((at >> 4) ^ H::turned(row)) << 4) + (at & 15);
                                float vf[kWide];
                                __builtin_memcpy(vf, from, sizeof(vf));
#pragma unroll
                                for (int j = 0; j < kWide; ++j) acc[w * kWide + j] = __builtin_amdgcn_mfma_f32_32x32x2f32(replaced(vf[j]), score[n][i], acc[w * kWide + j], 0, 0, 0);
                            }
                        }
                }
            };
            if (special == 0) second([](float v) { return v; });
            else second([special](float v) { return special == 4 ? (v - v == 0.f ? v : 0.f) : special == 3 ? (v != v ? 1.f : 0.f) : v == (special == 1 ? INFINITY : -INFINITY) ? 1.f : 0.f; });
        }
        if (special == 0) {
            float zero = 0.f;
#pragma unroll
            for (int n = 0; n < kBlocks; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) zero = __builtin_fmaf(acc[n][i], 0.f, zero);
            if (!__syncthreads_or(zero != 0.f)) break;
        } else if (special < 4) {
#pragma unroll
            for (int n = 0; n < kBlocks; n += 2) {
                uint32_t found = 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) found |= (uint32_t)(acc[n + i / 16][i & 15] > 0.f) << i;
                marks[special - 1][n / 2] = found;
            }
        } else {
#pragma unroll
            for (int n = 0; n < kBlocks; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int bit = 16 * (n & 1) + i;
                    if ((marks[0][n / 2] >> bit) & 1) acc[n][i] += INFINITY;
                    if ((marks[1][n / 2] >> bit) & 1) acc[n][i] -= INFINITY;
                    if ((marks[2][n / 2] >> bit) & 1) acc[n][i] = NAN;
                }
        }
    }

    l += with_other_half(l);
    const int64_t group_rows = ((int64_t)b * a.groups + group) * rows;
    if (a.parts > 1) {
        const int64_t at = (int64_t)blockIdx.x * W::kRows + wave * W::kRowsOfWave + (lane & 31);
        if (half == 0) *reinterpret_cast<f32x2*>(a.part_stats + 2 * at) = f32x2{m, l};
        if (begin_tile >= end_tile || r >= rows) return;
        float* to = a.part_sums + at * kSize;
#pragma unroll
        for (int n = 0; n < kBlocks; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) to[H::element(n, i, half)] = acc[n][i];
        return;
    }
    if (r >= rows) return;
    if (a.sums != nullptr && half == 0) a.sums[group_rows + r] = sum_of<kHalf>(m, l);
    const float share = l == 0.f ? 0.f : 1.f / l;
    char* y = a.y + b * a.y_batch + t * a.y_token + head * a.y_head;
#pragma unroll
    for (int n = 0; n < kBlocks; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] *= share;
    if constexpr (kHalf) {
#pragma unroll
        for (int n = 0; n < kBlocks; ++n)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const half4 v = {(_Float16)acc[n][i], (_Float16)acc[n][i + 1], (_Float16)acc[n][i + 2], (_Float16)acc[n][i + 3]};
                store<4>(a, y, H::element(n, i, half), v);
            }
    } else {
        constexpr int kWide = H::kWide;
#pragma unroll
        for (int n = 0; n < kBlocks; n += kWide)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float v __attribute__((ext_vector_type(kWide)));
#pragma unroll
                for (int j = 0; j < kWide; ++j) v[j] = acc[n + j][i];
                store<kWide>(a, y, H::element(n, i, half), v);
            }
    }
}

// A row's parts, by a wavefront: y = sum_i l_i 2^(m_i - m) (sums_i / l_i) over its sum of l_i 2^(m_i - m), in the order of the parts.
template <bool kHalf, int kSize>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a) {
    constexpr int kOf = kSize / 64;  // elements of a lane, next to each other
    const int lane = threadIdx.x & 63;
    const int32_t rows = a.T * a.fan;
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= (int64_t)a.B * a.groups * rows) return;
    const int32_t of = (int32_t)(row / rows), r = (int32_t)(row % rows), t = r / a.fan, head = of % a.groups * a.fan + (r - t * a.fan);
    const int32_t tile = r / a.tile_rows;
    const int64_t first = (((int64_t)of * a.row_tiles + tile) * a.parts) * a.tile_rows + (r - tile * a.tile_rows);
    f32x2 stat = {kNoMaximum, 0.f};
    if (lane < a.parts) stat = *reinterpret_cast<const f32x2*>(a.part_stats + 2 * (first + (int64_t)lane * a.tile_rows));
    float m = stat[1] != 0.f ? stat[0] : kNoMaximum;
#pragma unroll
    for (int d = 32; d; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
    const float weight = stat[1] != 0.f ? __builtin_amdgcn_exp2f(stat[0] - m) : 0.f;
    float l = weight == 0.f ? 0.f : stat[1] * weight;
#pragma unroll
    for (int d = 32; d; d /= 2) l += __shfl_xor(l, d);
    float sum[kOf] = {};
    for (int p = 0; p < a.parts; ++p) {
        const float w = __shfl(weight, p);
        if (w == 0.f) continue;
        const float* from = a.part_sums + (first + (int64_t)p * a.tile_rows) * kSize + lane * kOf;
#pragma unroll
        for (int j = 0; j < kOf; ++j) sum[j] = __builtin_fmaf(w, from[j], sum[j]);
    }
    if (a.sums != nullptr && lane == 0) a.sums[row] = sum_of<kHalf>(m, l);
    const float share = l == 0.f ? 0.f : 1.f / l;
    char* y = a.y + of / a.groups * a.y_batch + t * a.y_token + head * a.y_head;
#pragma unroll
    for (int j = 0; j < kOf; ++j) {
        if (lane * kOf + j >= a.D) break;
        if constexpr (kHalf) reinterpret_cast<_Float16*>(y)[lane * kOf + j] = (_Float16)(sum[j] * share);
        else reinterpret_cast<float*>(y)[lane * kOf + j] = sum[j] * share;
    }
}

// The weights that each place is given, over a group's rows: a wavefront takes 32 places and all rows, of which the first pass has left m + log2(l).
template <bool kHalf, int kSize>
__global__ __launch_bounds__(256) void attention_mass_kernel(AttentionArgs a) {
    using H = Head<kHalf, kSize>;
    constexpr int kSteps = H::kSteps, kPlaces = 32;
    __shared__ Nodes nodes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int32_t blocks = (a.places + 4 * kPlaces - 1) / (4 * kPlaces), block = blockIdx.x % blocks, of = blockIdx.x / blocks;
    const int32_t b = of / a.groups, group = of % a.groups, rows = a.T * a.fan, length = length_of(a, b), count = count_of(a, b);
    const int32_t end = (int32_t)min((int64_t)length + count, (int64_t)a.places), block_end = min((block + 1) * 4 * kPlaces, end);
    if (block * 4 * kPlaces >= end) return;
    if (a.kind == kTree && block_end > length) find_ancestors(&nodes, a.parents + (int64_t)b * a.T, a.T);
    const int32_t p0 = (block * 4 + wave) * kPlaces;
    if (p0 >= end) return;
    const int32_t row_bytes = a.D * H::kElement, mine = p0 + (lane & 31);
    Place at = {-1, 0};
    if (mine < end) at = place_in(a, b, mine);
    const uint32_t there = (uint32_t)__builtin_amdgcn_ballot_w64(at.page >= 0);
    u32x4 k[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
        k[s] = at.page >= 0 ? chunk_of<kHalf>(a.k + at.page * a.k_page + at.row * a.k_row + group * a.k_head, (2 * s + half) * 16, row_bytes, a.k_whole) : u32x4{0, 0, 0, 0};
    f32x16 total = {};
    // (the rows of a chain that come before the first of these places do not see them)
    const int32_t first_t = a.kind == kChain ? max(0, p0 - length) : 0;
    for (int32_t r0 = first_t * a.fan / 32 * 32; r0 < count * a.fan; r0 += 32) {
        const int32_t r = r0 + (lane & 31), t = r < rows ? r / a.fan : a.T, head = group * a.fan + (r - t * a.fan);
        const Sight sight = sight_of(a, t, length, count);
        const char* from = a.q + b * a.q_batch + t * a.q_token + head * a.q_head;
        const float less = r < rows ? a.sums[(int64_t)of * rows + r] : INFINITY;
        f32x16 score = {};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const u32x4 q = r < rows ? chunk_of<kHalf>(from, (2 * s + half) * 16, row_bytes, a.q_whole) : u32x4{0, 0, 0, 0};
            score = score_of<kHalf>(k[s], q, score);
        }
        score = hide(score, (seen_of(sight, &nodes, p0) & there) >> (4 * half));
#pragma unroll
        for (int i = 0; i < 16; ++i) total[i] += __builtin_amdgcn_exp2f(__builtin_fmaf(score[i], a.scale2, -less));
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
        for (int d = 16; d; d /= 2) total[i] += __shfl_xor(total[i], d);
        const int32_t p = p0 + 8 * (i >> 2) + 4 * half + (i & 3);
        if ((lane & 31) == i && ((there >> (p - p0)) & 1)) {
            float* to = a.mass + b * a.mass_batch + group * a.mass_head + p;
            *to = (p < length ? *to : 0.f) + total[i];
        }
    }
}

template <bool kHalf, int kSize>
int attend_of(const AttentionArgs& a, hipStream_t s) {
    using W = Tile<kHalf, kSize>;
    auto kernel = attention_kernel<kHalf, kSize>;
    if constexpr (W::kLds > 65536)  // (has to be asked for, on every device)
        CHX_HIP_CALL(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, W::kLds));
    kernel<<<(unsigned)((int64_t)a.B * a.groups * a.row_tiles * a.parts), 256, W::kLds, s>>>(a);
    return launch_check("attention_kernel");
}
template <bool kHalf, int kSize>
int join_of(const AttentionArgs& a, hipStream_t s) {
    attention_join_kernel<kHalf, kSize><<<(unsigned)(((int64_t)a.B * a.groups * a.T * a.fan + 3) / 4), 256, 0, s>>>(a);
    return launch_check("attention_join_kernel");
}
template <bool kHalf, int kSize>
int mass_of(const AttentionArgs& a, hipStream_t s) {
    attention_mass_kernel<kHalf, kSize><<<(unsigned)((int64_t)a.B * a.groups * ((a.places + 127) / 128)), 256, 0, s>>>(a);
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
