// The kernels behind linear_plan.hip, instantiated by type in linear_half.hip, linear_int8.hip and linear_float.hip.
//
//   y[m, n] = act(scale[n] * sum_k x[m, k] w[n, k] + bias[n]) + r[m, n]
//
// The sums are float32 (matrix instructions of 16 x 16 results), the epilogue works on them in float32, and the result is
// rounded once.  w is the first operand of an instruction, so that a lane's results are neighbouring columns of one row of y.
#pragma once

#include <cfloat>
#include <type_traits>

#include "linear_plan.h"

namespace chx {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at any address of an element

template <LinearType kType>
struct Of {
    static constexpr bool kFloat = kType == kFloatFloat;
    static constexpr int kElement = kFloat ? 4 : 2;          // bytes of an element of x
    static constexpr int kChunk = 16 / kElement;             // elements in 16 bytes
    static constexpr int kUnitK = unit_k(kType), kUnit = unit_bytes(kType);
    static constexpr int kPieces = kUnit / 1024;             // of 16 bytes a lane that a unit's four fragments are
    static constexpr int kFragmentsOf = 4 / kPieces;         // fragments in a piece
};

// Eight weights of 8 bits as float16.  0x6400 + b is the float16 1024 + b for a byte b; with the sign bit flipped, b is w + 128,
// and taking 1152 away is exact.
__device__ __forceinline__ u32x4 halves_of_bytes(uint32_t lo, uint32_t hi) {
    u32x4 r;
    const half2v off = {(_Float16)1152.f, (_Float16)1152.f};
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t packed = __builtin_amdgcn_perm(0x64646464u, i < 2 ? lo : hi, (i & 1) ? 0x04030402u : 0x04010400u);
        r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, packed) - off);
    }
    return r;
}

// One fragment of w times one of x.
template <LinearType kType>
__device__ __forceinline__ f32x4 product(u32x4 w, u32x4 x, f32x4 acc) {
    if constexpr (kType == kFloatFloat) {
        const f32x4 wf = __builtin_bit_cast(f32x4, w), xf = __builtin_bit_cast(f32x4, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[j], xf[j], acc, 0, 0, 0);
        return acc;
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, w), __builtin_bit_cast(half8, x), acc, 0, 0, 0);
    }
}

// Fragment f of the pieces that hold it.
template <LinearType kType>
__device__ __forceinline__ u32x4 fragment_of(const u32x4* pieces, int f) {
    if constexpr (kType == kHalfInt8) return halves_of_bytes(pieces[f / 2][2 * (f & 1)], pieces[f / 2][2 * (f & 1) + 1]);
    else return pieces[f];
}

// 16 bytes of a row of x from element k on, zeros from K on (0 * inf would be NaN); any alignment, any distance between elements.
template <LinearType kType>
__device__ __forceinline__ u32x4 chunk_of(const char* row, int64_t col, int32_t k, int32_t K) {
    constexpr int kElement = Of<kType>::kElement, kChunk = Of<kType>::kChunk;
    if (col == kElement && k + kChunk <= K) return *reinterpret_cast<const u32x4_any*>(row + (int64_t)k * kElement);
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
        if (k + j >= K) break;
        const char* p = row + (int64_t)(k + j) * col;
        if constexpr (kElement == 4) v[j] = *reinterpret_cast<const uint32_t*>(p);
        else v[j / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p) << (16 * (j & 1));
    }
    return v;
}

// gelu(v) = v Phi(v) = max(v, 0) - z Phi(-z), z = |v|.  For float16 results Phi(-z) = exp(-z^2 / 2) P(t), t = 1 / (1 + 0.4 z), with P fitted by least
// squares to the relative error over 0 <= z <= 9: 2.6e-6, with the rounding of the exponent up to 6e-6 at z = 9, where rounding the result to float16 takes 4.9e-4.  Some 15 instructions; the
// library's erff takes three times as many.
__device__ __forceinline__ float gelu_short(float v) {
    const float z = __builtin_fabsf(v);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.4f, z, 1.0f));
    float p = 5.3671894526e-02f;
    p = __builtin_fmaf(p, t, -2.4778526818e-01f);
    p = __builtin_fmaf(p, t, 3.3548150906e-01f);
    p = __builtin_fmaf(p, t, 1.0279341753e-02f);
    p = __builtin_fmaf(p, t, 1.9333978946e-01f);
    p = __builtin_fmaf(p, t, 1.5472590493e-01f);
    p = __builtin_fmaf(p, t, 2.8555855905e-04f);
    const float tail = p * __builtin_amdgcn_exp2f(-0.72134752f * z * z);  // Phi(-z); a NaN stays one
    return __builtin_fmaf(-fminf(z, 64.f), tail, fmaxf(v, 0.f));           // (infinite z: 0 of it)
}

// kShort: for a result that is rounded to float16, with hardware exponentials and reciprocals; else to float32's own accuracy.  A sum of -inf gives the limit, 0: what is
// multiplied with a factor that becomes 0 is kept finite (a NaN stays one in that factor).
template <bool kShort, int kCount>
__device__ __forceinline__ void activate(float (&v)[kCount], int32_t act) {
    auto finite = [](float o) { return fmaxf(o, -FLT_MAX); };
    switch (act) {
        case CHX_HIP_ACT_RELU:
#pragma unroll
            for (int i = 0; i < kCount; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // (a NaN stays)
            break;
        case CHX_HIP_ACT_GELU:
#pragma unroll
            for (int i = 0; i < kCount; ++i) v[i] = kShort ? gelu_short(v[i]) : 0.5f * finite(v[i]) * erfcf(-0.70710678f * v[i]);
            break;
        case CHX_HIP_ACT_GELU_TANH:
            // 0.5 v (1 + tanh u) = v / (1 + exp(-2 u))
#pragma unroll
            for (int i = 0; i < kCount; ++i) {
                const float u = 0.7978845608f * __builtin_fmaf(0.044715f * v[i] * v[i], v[i], v[i]);
                v[i] = kShort ? finite(v[i]) * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-2.8853901f * u)) : finite(v[i]) / (1.f + expf(-2.f * u));
            }
            break;
        case CHX_HIP_ACT_SILU:
#pragma unroll
            for (int i = 0; i < kCount; ++i)
                v[i] = kShort ? finite(v[i]) * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950f * v[i])) : finite(v[i]) / (1.f + expf(-v[i]));
            break;
        default: break;
    }
}

// kCount neighbouring columns (a multiple of 4, from a multiple of 4 on) of one row of the result.  Rows that are not whole 8-byte pieces are stored an element at a time: 4096 x 4096 x
// 16385 in float16 556 us, 16384 columns 422; 512 rows 92 and 78, one row 29 and 22.
template <LinearType kType, int kCount>
__device__ __forceinline__ void finish(const LinearArgs& a, float (&v)[kCount], int64_t row, int32_t n) {
    if (n >= a.N) return;
    const bool whole = n + kCount <= a.N;
    if (!Of<kType>::kFloat && a.y_half) activate<true, kCount>(v, a.activation);
    else activate<false, kCount>(v, a.activation);
    if (a.r) {
        const char* p = a.r + row * a.r_row + (int64_t)n * a.r_col;
        if (whole && a.vector_r) {
            constexpr int kBytes = kCount * 2;
            if (a.y_half) {
                _Float16 h[kCount];
                __builtin_memcpy(h, __builtin_assume_aligned(p, 8), kBytes);
#pragma unroll
                for (int i = 0; i < kCount; ++i) v[i] += (float)h[i];
            } else {
                float h[kCount];
                __builtin_memcpy(h, __builtin_assume_aligned(p, 16), 2 * kBytes);
#pragma unroll
                for (int i = 0; i < kCount; ++i) v[i] += h[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < kCount; ++i) {
                if (n + i >= a.N) break;
                v[i] += a.y_half ? (float)*reinterpret_cast<const _Float16*>(p + i * a.r_col) : *reinterpret_cast<const float*>(p + i * a.r_col);
            }
        }
    }
    char* p = a.y + row * a.y_row + (int64_t)n * a.y_col;
    if (whole && a.vector_y) {
        if (a.y_half) {
            _Float16 h[kCount];
#pragma unroll
            for (int i = 0; i < kCount; ++i) h[i] = (_Float16)v[i];
            __builtin_memcpy(__builtin_assume_aligned(p, 8), h, kCount * 2);
        } else {
            __builtin_memcpy(__builtin_assume_aligned(p, 16), v, kCount * 4);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            if (n + i >= a.N) break;
            if (a.y_half) *reinterpret_cast<_Float16*>(p + i * a.y_col) = (_Float16)v[i];
            else *reinterpret_cast<float*>(p + i * a.y_col) = v[i];
        }
    }
}

// Where a tile of rows lies: the rows themselves, or the places [first, first + count) of the routing's order.
struct Rows {
    int32_t expert, first, count;  // count 0: no such tile
};

// Tile `index` of the experts' tiles of up to `height` rows: those of expert 0, of expert 1 and so on, each expert's of one size, a multiple of `grain` (a divisor of
// height).  With whole tiles first and what is left of each expert's rows behind them, tiles of few rows were bound by their weights, which came a second time: 4096 rows to 4 of
// 32 experts of 4096 x 2048 took 313 us instead of 296, 2048 rows to 8 of 128 experts of 2048 x 768 200 instead of 188.  (384 rows to each of the 32, 256 and 128 of
// them to a tile, took as long as 512.)  Every
// wavefront finds its tile by itself, 64 experts at a time.
template <int kGrain>
__device__ __forceinline__ Rows expert_rows(const LinearArgs& a, int32_t index, int32_t height) {
    const int lane = threadIdx.x & 63;
    for (int32_t e0 = 0; e0 < a.experts; e0 += 64) {
        const int32_t e = e0 + lane;
        int32_t lo = 0, hi = 0;
        if (e < a.experts) {  // (offsets from device memory: kept inside the order whatever they say)
            lo = min(max(a.offsets[e], 0), a.M);
            hi = min(max(a.offsets[e + 1], lo), a.M);
        }
        const int32_t tiles = (hi - lo) / height + ((hi - lo) % height != 0);
        int32_t upto = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int32_t v = __shfl_up(upto, d);
            if (lane >= d) upto += v;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > index);
        if (past) {
            const int at = __builtin_ctzll(past);
            const int32_t first = __builtin_amdgcn_readlane(lo, at), count = __builtin_amdgcn_readlane(hi, at) - first, of = __builtin_amdgcn_readlane(tiles, at);
            const int32_t t = index - (__builtin_amdgcn_readlane(upto, at) - of), each = (int32_t)((((uint32_t)count + of - 1) / of + kGrain - 1) / kGrain * kGrain);
            return {e0 + at, first + t * each, min(count - t * each, each)};
        }
        index -= __builtin_amdgcn_readlane(upto, 63);
    }
    return {0, 0, 0};
}

// The row of the result (-1: none) that place i of a tile stands for.
template <bool kExperts>
__device__ __forceinline__ int32_t row_at(const LinearArgs& a, const Rows& t, int32_t i) {
    if (i >= t.count) return -1;
    if constexpr (!kExperts) return t.first + i;
    const int32_t p = a.order[t.first + i];
    return p >= 0 && p < a.M ? p : -1;  // (from device memory)
}

// An asynchronous copy of 16 bytes a lane into LDS: lane i's to lds + 16 i (the same for all lanes), counted like a load.
__device__ __forceinline__ void copy_to_lds(uint32_t offset, const char* base, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}

// ---- few rows ---------------------------------------------------------------------------------------
//
// Bound by the bytes of w, each read once.  A work-group takes kFragments fragments' columns (16 each) and all k, its kWaves wavefronts every
// kWaves-th block of two units: w goes from memory straight into registers, kDeep blocks ahead of the products, and the wavefronts' sums
// are added in LDS, in one order.  x comes from the caches.  A work-group of 16 rows loads them as fragments; one of more copies a block (128 bytes of every row)
// into LDS of the wavefront's own, because lanes next to each other that load from different rows take a cache access each: 64 rows x 4096 x
// 16384, 32 columns to a work-group, 36 us instead of 48 (with 64 columns it takes 27).  Rows that are not there repeat the last one; their results are dropped.
template <LinearType kType, int kRowTiles, int kFragments>
struct RowsShape {
    static constexpr int kWaves = 8, kPieces = kFragments / Of<kType>::kFragmentsOf;
    static constexpr bool kInLds = kRowTiles > 1;       // x
    static constexpr int kDeep = 2;
    static constexpr int kBlock = kInLds ? kRowTiles * 2048 : 0;  // bytes of x in LDS
    static constexpr int kOfBlocks = kWaves * kDeep * kBlock, kOfSums = kWaves * kRowTiles * kFragments * 1024;
    static constexpr int kLds = kOfBlocks > kOfSums ? kOfBlocks : kOfSums;
};

// kStream: w is more than the caches are likely to hold from one call to the next, and goes by them (launch_rows).
template <LinearType kType, int kRowTiles, int kFragments, bool kDirect, bool kExperts, bool kStream>
__global__ __launch_bounds__((64 * RowsShape<kType, kRowTiles, kFragments>::kWaves)) void linear_rows_kernel(LinearArgs a) {
    using O = Of<kType>;
    using S = RowsShape<kType, kRowTiles, kFragments>;
    constexpr int kWaves = S::kWaves, kDeep = S::kDeep, kPieces = S::kPieces;
    constexpr int kRows = S::kInLds ? 2 * kRowTiles : 1;  // that a lane has pieces of
    constexpr bool kCopied = S::kInLds && kDirect;
    static_assert(kFragments % O::kFragmentsOf == 0, "whole pieces");
    extern __shared__ __attribute__((aligned(128))) char rows_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t columns = blockIdx.x % a.tiles_n, tile = blockIdx.x / a.tiles_n;
    Rows t;
    if constexpr (kExperts) {
        t = expert_rows<16>(a, tile, 16 * kRowTiles);
        if (t.count <= 0) return;
    } else {
        t = {0, tile * 16 * kRowTiles, min(a.M - tile * 16 * kRowTiles, 16 * kRowTiles)};
    }
    const int32_t fragment = columns * kFragments;  // of all: 4 to a group
    const char* w = a.w + t.expert * a.w_expert + (int64_t)(fragment >> 2) * a.w_group + (fragment & 3) / O::kFragmentsOf * 1024 + lane * 16;
    // x: this lane's piece of every eighth row of a block (registers: its pieces of one row), as offsets from the tile's first row (experts: from x)
    const char* x_base = a.x + (kExperts ? 0 : (int64_t)t.first * a.x_row);
    const int32_t x_chunk = S::kInLds ? (lane & 7) ^ (lane >> 3) : lane >> 4;
    typedef typename std::conditional<kDirect, uint32_t, int64_t>::type Offset;
    Offset x_at[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int32_t row = max(row_at<kExperts>(a, t, min(S::kInLds ? 8 * i + (lane >> 3) : lane & 15, t.count - 1)), 0);
        x_at[i] = (Offset)(kExperts ? (int64_t)(row / a.fan) * a.x_row : (int64_t)(row - t.first) * a.x_row) + (kDirect ? x_chunk * 16 : 0);
    }
    char* blocks = rows_lds + wave * kDeep * S::kBlock;  // this wavefront's
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)blocks;
    f32x4 acc[kRowTiles][kFragments];
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
        for (int f = 0; f < kFragments; ++f) acc[i][f] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Block {
        u32x4 w[2][kPieces];
        u32x4 x[S::kInLds ? kRows : 2];
    };
    auto load = [&](Block& r, int place, int32_t block) __attribute__((always_inline)) {
        if constexpr (kCopied) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) copy_to_lds((uint32_t)x_at[i], x_base + (int64_t)block * 128, lds0 + place * S::kBlock + i * 1024);
        } else if constexpr (S::kInLds) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) r.x[i] = chunk_of<kType>(x_base + x_at[i], a.x_col, block * 2 * O::kUnitK + x_chunk * O::kChunk, a.K);
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if constexpr (kDirect) r.x[u] = *reinterpret_cast<const u32x4*>(x_base + (int64_t)block * 128 + u * 64 + x_at[0]);
                else r.x[u] = chunk_of<kType>(x_base + x_at[0], a.x_col, (block * 2 + u) * O::kUnitK + x_chunk * O::kChunk, a.K);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
                const u32x4* from = reinterpret_cast<const u32x4*>(w + (int64_t)(2 * block + u) * O::kUnit + p * 1024);
                if constexpr (kStream) r.w[u][p] = __builtin_nontemporal_load(from);
                else r.w[u][p] = *from;
            }
    };
    // younger: whether the loads of kDeep - 1 blocks behind this one are under way
    auto multiply = [&](Block& r, int place, int32_t block, auto younger) __attribute__((always_inline)) {
        u32x4 x[2][kRowTiles];
        if constexpr (S::kInLds) {
            char* at = blocks + place * S::kBlock;
            if constexpr (!kCopied) {
#pragma unroll
                for (int i = 0; i < kRows; ++i) *reinterpret_cast<u32x4*>(at + i * 1024 + lane * 16) = r.x[i];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            } else if constexpr (decltype(younger)::value) {
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kDeep - 1) * (kRows + 2 * kPieces)) : "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < kRowTiles; ++i)
                    x[u][i] = *reinterpret_cast<const u32x4*>(at + (i * 16 + (lane & 15)) * 128 + (((u * 4 + (lane >> 4)) ^ (lane & 7)) << 4));
        } else {
            x[0][0] = r.x[0];
            x[1][0] = r.x[1];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int f = 0; f < kFragments; ++f) {
                const u32x4 o = fragment_of<kType>(r.w[u], f);
#pragma unroll
                for (int i = 0; i < kRowTiles; ++i) acc[i][f] = product<kType>(o, x[u][i], acc[i][f]);
            }
        }
        // (what is read from this place is there before anything is copied to it)
        if constexpr (S::kInLds) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    Block ring[kDeep];
    const int32_t all = a.units / 2, mine = all > wave ? (all - wave + kWaves - 1) / kWaves : 0;
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
        if (d < mine) load(ring[d], d, wave + d * kWaves);
    int32_t j = 0;
    for (; j + 2 * kDeep <= mine; j += kDeep) {  // (without conditions, so that each product waits for its own loads alone)
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            multiply(ring[d], d, wave + (j + d) * kWaves, std::true_type());
            load(ring[d], d, wave + (j + d + kDeep) * kWaves);
        }
    }
    for (; j < mine; j += kDeep) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (j + d < mine) multiply(ring[d], d, wave + (j + d) * kWaves, std::false_type());
            if (j + d + kDeep < mine) load(ring[d], d, wave + (j + d + kDeep) * kWaves);
        }
    }
    f32x4* sums = reinterpret_cast<f32x4*>(rows_lds);  // [wave][row tile][fragment][lane]
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
        for (int f = 0; f < kFragments; ++f) sums[((wave * kRowTiles + i) * kFragments + f) * 64 + lane] = acc[i][f];
    __syncthreads();
    for (int at = threadIdx.x; at < kRowTiles * kFragments * 64; at += 64 * kWaves) {
        const int l = at & 63, f = (at >> 6) % kFragments, i = (at >> 6) / kFragments;
        f32x4 sum = sums[at];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum += sums[v * kRowTiles * kFragments * 64 + at];
        const int32_t row = row_at<kExperts>(a, t, 16 * i + (l & 15));
        const int32_t n = ((fragment + f) >> 2) * kGroupRows + group_row((fragment + f) & 3, (l >> 4) * 4);
        if (row < 0) continue;
        float v[4] = {sum[0], sum[1], sum[2], sum[3]};
        const int64_t at_n = (int64_t)t.expert * a.n_padded + n;
        // (scales and biases are filled up to whole groups)
#pragma unroll
        for (int j4 = 0; j4 < 4; ++j4) {
            if constexpr (kType == kHalfInt8) v[j4] *= a.scale[at_n + j4];
            if (a.bias) v[j4] += a.bias[at_n + j4];
        }
        finish<kType, 4>(a, v, row, n);
    }
}

// ---- tiles -------------------------------------------------------------------------------------------
//
// x lies in rows of whole blocks, in 16-byte pieces (others are brought into such first, linear_plan.hip: loaded through registers here, 4096 rows of
// 4097 x 16384 took 636 us instead of 443).
// A work-group of kWavesM x kWavesN wavefronts, each 16 kRowFragments rows (every kWavesM-th 16 of the tile's) and 64 columns.  w comes into a ring of three units in LDS, x into one of
// three blocks of two units (a block is 128 bytes of every row: of half a line at a time, the other half was fetched again where the
// rows lie a power of two apart: 435 us instead of 419 for 4096 x 4096 x 16384), by asynchronous copies two and three units ahead.  While a unit
// is multiplied from registers, the next one's fragments come from LDS into others, so its place in the ring is free a unit early.
// A row of x in a block is eight pieces of 16 bytes; piece c of row r lies at place c ^ (r & 7): the sixteen rows that a fragment is
// read from then do not meet in one bank.

template <LinearType kType, int kRowFragments, int kWavesM, int kWavesN>
struct TileShape {
    static constexpr int kThreads = 64 * kWavesM * kWavesN, kRows = kWavesM * kRowFragments * 16, kGroups = kWavesN, kRing = 3;
    static constexpr int kBlock = kRows * 128, kUnits = kGroups * unit_bytes(kType);  // bytes of x, of w
    static constexpr int kCopiesX = kBlock / 16 / kThreads, kCopiesW = kUnits / 16 / kThreads;
    static constexpr int kAtW = kRing * kBlock, kAtRows = kAtW + kRing * kUnits, kLds = kAtRows + kRows * 4;
    static_assert(kBlock % (32 * kThreads) == 0 && kUnits % (16 * kThreads) == 0, "whole copies");
};

template <LinearType kType, int kRowFragments, int kWavesM, int kWavesN, bool kExperts>
__global__ __launch_bounds__(64 * kWavesM * kWavesN, 2) void linear_tile_kernel(LinearArgs a) {
    using O = Of<kType>;
    using S = TileShape<kType, kRowFragments, kWavesM, kWavesN>;
    constexpr int kThreads = S::kThreads, kBM = S::kRows, kGroups = S::kGroups, kCopiesX = S::kCopiesX, kCopiesW = S::kCopiesW;
    extern __shared__ __attribute__((aligned(128))) char tile_lds[];
    int32_t* rows = reinterpret_cast<int32_t*>(tile_lds + S::kAtRows);  // of the result
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / kWavesN, wn = wave % kWavesN;
    // Work-groups that follow each other run on different XCDs, each with its own L2: an eighth of the tiles to each, in blocks
    // of 8 tiles of rows, so that what a block reads stays there.  Experts' tiles, of which there may be fewer than the grid has, are dealt out to the XCDs in
    // pieces, so that the last XCD is not left with those that are not there.
    int32_t tm, tn;
    if constexpr (kExperts) {
        const int32_t wide = piece_columns(a.tiles_n), across = (a.tiles_n + wide - 1) / wide, at = blockIdx.x >> 3, inside = at % (kPieceRows * wide);
        const int32_t piece = at / (kPieceRows * wide) * 8 + (blockIdx.x & 7);
        tm = piece / across * kPieceRows + inside % kPieceRows;
        tn = piece % across * wide + inside / kPieceRows;
        if (tn >= a.tiles_n) return;
    } else {
        const int32_t all = a.tiles_m * a.tiles_n, q = all >> 3, rest = all & 7, xcd = blockIdx.x & 7, id = xcd * q + min(xcd, rest) + ((int32_t)blockIdx.x >> 3);
        constexpr int32_t kBlock = 8;
        const int32_t block = id / (kBlock * a.tiles_n), height = min(a.tiles_m - block * kBlock, kBlock), inside = id - block * kBlock * a.tiles_n;
        tm = block * kBlock + inside % height;
        tn = inside / height;
    }
    Rows t;
    if constexpr (kExperts) {
        t = expert_rows<16 * kWavesM>(a, tm, kBM);
        if (t.count <= 0) return;
    } else {
        t = {0, tm * kBM, min(a.M - tm * kBM, kBM)};
    }
    for (int i = threadIdx.x; i < kBM; i += kThreads) rows[i] = row_at<kExperts>(a, t, i);

    // x: this thread's pieces of a block, as offsets from the tile's first row (experts: from x); the same piece of every row
    const char* x_base = a.x + (kExperts ? 0 : (int64_t)t.first * a.x_row);
    const int32_t x_chunk = (threadIdx.x & 7) ^ ((threadIdx.x >> 3) & 7);
    auto row_of = [&](int i) __attribute__((always_inline)) -> int64_t {
        const int32_t row = max(row_at<kExperts>(a, t, min((i * kThreads + (int)threadIdx.x) >> 3, t.count - 1)), 0);
        return kExperts ? (int64_t)(row / a.fan) * a.x_row : (int64_t)(row - t.first) * a.x_row;
    };
    uint32_t x_at[kCopiesX];
#pragma unroll
    for (int i = 0; i < kCopiesX; ++i) x_at[i] = (uint32_t)row_of(i) + x_chunk * 16;
    // w: a unit of one group after the other, in the order in which it lies
    const char* w_base = a.w + t.expert * a.w_expert + (int64_t)tn * kGroups * a.w_group;
    const int32_t last_group = (a.N + kGroupRows - 1) / kGroupRows - 1 - tn * kGroups;
    uint32_t w_at[kCopiesW];
#pragma unroll
    for (int i = 0; i < kCopiesW; ++i) {
        const int at = (i * kThreads + threadIdx.x) * 16, g = at / O::kUnit;
        w_at[i] = (uint32_t)(min(g, last_group) * a.w_group) + at % O::kUnit;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)tile_lds + wave * 1024;

    auto copy_w = [&](int c, int32_t unit, int place) __attribute__((always_inline)) {
        copy_to_lds(w_at[c], w_base + (int64_t)unit * O::kUnit, lds0 + S::kAtW + place * S::kUnits + c * kThreads * 16);
    };
    auto copy_x = [&](int c, int32_t block, int place) __attribute__((always_inline)) {
        copy_to_lds(x_at[c], x_base + (int64_t)block * 128, lds0 + place * S::kBlock + c * kThreads * 16);
    };

    f32x4 acc[kRowFragments][4];
#pragma unroll
    for (int i = 0; i < kRowFragments; ++i)
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[i][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int x_lane = (wm * 16 + (lane & 15)) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
    const int w_lane = S::kAtW + wn * O::kUnit + lane * 16;
    struct Unit {
        u32x4 w[O::kPieces], x[kRowFragments];
    };
    // (half: which of its block's two units)
    auto read_w = [&](Unit& r, int p, int place) __attribute__((always_inline)) { r.w[p] = *reinterpret_cast<const u32x4*>(tile_lds + place * S::kUnits + w_lane + p * 1024); };
    auto read_x = [&](Unit& r, int i, int place, int half) __attribute__((always_inline)) {
        r.x[i] = *reinterpret_cast<const u32x4*>(tile_lds + place * S::kBlock + (x_lane ^ (half * 64)) + i * kWavesM * 2048);
    };
    auto read_unit = [&](Unit& r, int place_x, int half, int place_w) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < O::kPieces; ++p) read_w(r, p, place_w);
#pragma unroll
        for (int i = 0; i < kRowFragments; ++i) read_x(r, i, place_x, half);
    };
    auto multiply = [&](const u32x4 (&w)[4], const Unit& r, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[i][f] = product<kType>(w[f], r.x[i], acc[i][f]);
    };
    auto fragments_of = [&](u32x4 (&w)[4], const Unit& r) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < 4; ++f) w[f] = fragment_of<kType>(r.w, f);
    };
    Unit even, odd;

    const int32_t blocks = a.units / 2;
    {
        // (copies behind the last block bring it again, to a place that nobody reads any more: no step has a condition in it)
        const int32_t last = blocks - 1;
#pragma unroll
        for (int b = 0; b < S::kRing; ++b) {
#pragma unroll
            for (int c = 0; c < kCopiesX; ++c) copy_x(c, min(b, last), b);
#pragma unroll
            for (int c = 0; c < kCopiesW; ++c) copy_w(c, min(b, 2 * blocks - 1), b);
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
        int here_x = 0, here_w = 0;  // places in the rings of this block and unit
        auto behind = [](int place) __attribute__((always_inline)) { return place + 1 == S::kRing ? 0 : place + 1; };
        const int32_t fragments = (t.count - wm * 16 + 16 * kWavesM - 1) / (16 * kWavesM);  // of this wavefront's that have rows
        // One unit, the block's first or second, from `now`, with the next one's fragments into `then`.  `whole`: with all of this wavefront's
        // fragments; else with those that have rows, each behind a branch (an expert's tile, of which a quarter or more is missing: 296 us for 4096 rows to 4 of 32 experts of 4096 x
        // 2048 instead of 310; but 600 rows of 4096 x 4096, the last 88 rows of which are a tile, 37.5 instead of 31.8).
        auto step = [&](int32_t block, auto second, auto whole, const Unit& now, Unit& then) __attribute__((always_inline)) {
            constexpr bool kSecond = decltype(second)::value, kWhole = decltype(whole)::value;
            const int next_x = behind(here_x), next_w = behind(here_w), before_x = behind(next_x);
            // The copies that the next unit needs are there, of w from two steps ago, of x from three or more; and this wavefront has read this unit.
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kCopiesX + kCopiesW) : "memory");
            __builtin_amdgcn_s_barrier();
            // ahead: half of the block three behind this one, in its place when both its units are read; else the other half of the one before
            const int32_t ahead = min(block + (kSecond ? 3 : 2), last), ahead_w = min(2 * block + (kSecond ? 1 : 0) + 3, 2 * blocks - 1);
            // What is read for the next unit and copied ahead goes between the products: copies one behind the other would keep the
            // wavefront from its products until the last of them is under way.
            u32x4 w[4];
            fragments_of(w, now);
            constexpr int kHalf = kCopiesX / 2, kCopies = kCopiesW + kHalf, kPiecesEach = (O::kPieces + kRowFragments - 1) / kRowFragments;
#pragma unroll
            for (int i = 0; i < kRowFragments; ++i) {
#pragma unroll
                for (int p = i * kPiecesEach; p < O::kPieces && p < (i + 1) * kPiecesEach; ++p) read_w(then, p, next_w);
                if (kWhole || i < fragments) read_x(then, i, kSecond ? next_x : here_x, kSecond ? 0 : 1);
#pragma unroll
                for (int c = i * kCopies / kRowFragments; c < (i + 1) * kCopies / kRowFragments; ++c) {
                    if (c < kCopiesW) copy_w(c, ahead_w, here_w);
                    else copy_x(c - kCopiesW + (kSecond ? 0 : kHalf), ahead, kSecond ? here_x : before_x);
                }
                if (kWhole || i < fragments) multiply(w, now, i);
                __builtin_amdgcn_sched_barrier(0);
            }
            here_w = next_w;
            if constexpr (kSecond) here_x = next_x;
        };
        auto all_steps = [&](auto whole) __attribute__((always_inline)) {
            read_unit(even, 0, 0, 0);
            for (int32_t block = 0; block < blocks; ++block) {
                step(block, std::false_type(), whole, even, odd);
                step(block, std::true_type(), whole, odd, even);
            }
        };
        if constexpr (!kExperts) all_steps(std::true_type());
        else if (fragments * 4 > kRowFragments * 3) all_steps(std::true_type());
        else all_steps(std::false_type());
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }

    // The results go through LDS, 32 rows of a wavefront at a time, so that the epilogue is a loop over eight columns of a lane: written out over the
    // accumulators it is 60 KB of code, which each tile fetched anew (a tenth of the time).  Piece c of 16 bytes of a row lies at place c ^ (row & 15).
    __syncthreads();
    constexpr int kPassRows = 32;
    static_assert(kWavesM * kWavesN * kPassRows * 256 <= S::kAtRows, "the rings hold them");
    char* mine = tile_lds + wave * kPassRows * 256;
    const int32_t n = (tn * kGroups + wn) * kGroupRows + (lane & 7) * 8;
    const int64_t at_n = (int64_t)t.expert * a.n_padded + (n < a.n_padded ? n : 0);
    // (scales and biases are filled up to whole groups)
    float scale[8], bias[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        scale[j] = kType == kHalfInt8 ? a.scale[at_n + j] : 1.f;
        bias[j] = a.bias ? a.bias[at_n + j] : 0.f;
    }
#pragma unroll 1
    for (int pass = 0; pass < kRowFragments / 2; ++pass) {
#pragma unroll
        for (int i0 = 0; i0 < kRowFragments; i0 += 2) {
            if (pass != i0 / 2) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int f = 0; f < 4; ++f)
                    *reinterpret_cast<f32x4*>(mine + (i * 16 + (lane & 15)) * 256 + ((((lane >> 4) * 4 + f) ^ (lane & 15)) << 4)) = acc[i0 + i][f];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 2
        for (int i = 0; i < kPassRows / 8; ++i) {
            const int r = i * 8 + (lane >> 3), row = rows[((pass * 2 + (r >> 4)) * kWavesM + wm) * 16 + (r & 15)];
            const f32x4 lo = *reinterpret_cast<const f32x4*>(mine + r * 256 + (((lane & 7) * 2 ^ (r & 15)) << 4));
            const f32x4 hi = *reinterpret_cast<const f32x4*>(mine + r * 256 + (((lane & 7) * 2 + 1) ^ (r & 15)) * 16);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = j < 4 ? lo[j & 3] : hi[j & 3];
                if constexpr (kType == kHalfInt8) v[j] *= scale[j];
                v[j] += bias[j];
            }
            if (row >= 0) finish<kType, 8>(a, v, row, n);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- launches ------------------------------------------------------------------------------------------

template <LinearType kType, int kRowTiles, int kFragments, bool kDirect, bool kExperts>
int launch_rows(const LinearArgs& a, hipStream_t s) {
    using S = RowsShape<kType, kRowTiles, kFragments>;
    // From 32 MB of weights on past the caches, in us with / without them, eight layers in turn: 134 MB of one row 25.9 / 22.9, 400 MB of 64 experts 50.6 / 44.5,
    // 67 MB of int8 14.8 / 13.6; 33 MB 8.5 / 8.4; but 17 MB of int8 6.1 / 7.3, 25 MB 10.9 / 13.8.
    const int64_t bytes = a.order ? a.w_expert * a.experts : (int64_t)a.n_padded / kGroupRows * a.w_group;
    auto kernel = kDirect && bytes >= (int64_t(32) << 20) ? linear_rows_kernel<kType, kRowTiles, kFragments, kDirect, kExperts, kDirect>
                                                           : linear_rows_kernel<kType, kRowTiles, kFragments, kDirect, kExperts, false>;
    if constexpr (S::kLds > 65536)  // (has to be asked for, on every device)
        CHX_HIP_CALL(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds));
    kernel<<<(unsigned)(a.tiles_m * a.tiles_n), 64 * S::kWaves, S::kLds, s>>>(a);
    return launch_check("linear_rows_kernel");
}

template <LinearType kType, int kRowFragments, int kWavesM, int kWavesN, bool kExperts>
int launch_tile(const LinearArgs& a, hipStream_t s) {
    using S = TileShape<kType, kRowFragments, kWavesM, kWavesN>;
    auto kernel = linear_tile_kernel<kType, kRowFragments, kWavesM, kWavesN, kExperts>;
    if constexpr (S::kLds > 65536)  // (has to be asked for, on every device)
        CHX_HIP_CALL(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds));
    kernel<<<(unsigned)(kExperts ? expert_grid(a.tiles_m, a.tiles_n) : (int64_t)a.tiles_m * a.tiles_n), S::kThreads, S::kLds, s>>>(a);
    return launch_check("linear_tile_kernel");
}

// kForExperts: whether experts take this size too.
template <LinearType kType, int kRowTiles, int kFragments, bool kForExperts>
int rows_of(const LinearArgs& a, bool direct, hipStream_t s) {
    if (a.order) {
        if constexpr (kForExperts) return direct ? launch_rows<kType, kRowTiles, kFragments, true, true>(a, s) : launch_rows<kType, kRowTiles, kFragments, false, true>(a, s);
        CHX_FAIL(CHX_HIP_EUNSUPPORTED, "linear plan: no kernel for experts' %d tiles of rows and %d fragments", kRowTiles, kFragments);
    }
    return direct ? launch_rows<kType, kRowTiles, kFragments, true, false>(a, s) : launch_rows<kType, kRowTiles, kFragments, false, false>(a, s);
}

template <LinearType kType, int kRowFragments, int kWavesM, int kWavesN, bool kForExperts>
int tile_of(const LinearArgs& a, hipStream_t s) {
    if (a.order) {
        if constexpr (kForExperts) return launch_tile<kType, kRowFragments, kWavesM, kWavesN, true>(a, s);
        CHX_FAIL(CHX_HIP_EUNSUPPORTED, "linear plan: no kernel for experts' tiles of %d rows", 16 * kRowFragments * kWavesM);
    }
    return launch_tile<kType, kRowFragments, kWavesM, kWavesN, false>(a, s);
}

}  // namespace

template <LinearType kType>
int LinearKernels<kType>::rows(const LinearArgs& a, int row_tiles, int fragments, bool direct, hipStream_t s) {
    // (the grid is made for these numbers: any others are refused.  What a choice never gives is not built.)
    switch (row_tiles * 8 + fragments) {
        case 8 + 1: if constexpr (kType != kHalfInt8) return rows_of<kType, 1, 1, true>(a, direct, s); else break;  // (two fragments of int8 are one piece)
        case 16 + 1: if constexpr (kType != kHalfInt8) return rows_of<kType, 2, 1, true>(a, direct, s); else break;
        case 8 + 2: return rows_of<kType, 1, 2, true>(a, direct, s);
        case 8 + 4: return rows_of<kType, 1, 4, true>(a, direct, s);
        case 16 + 2: return rows_of<kType, 2, 2, true>(a, direct, s);
        case 16 + 4: return rows_of<kType, 2, 4, true>(a, direct, s);
        case 32 + 2: if constexpr (kType == kFloatFloat) return rows_of<kType, 4, 2, false>(a, direct, s); else break;
        case 32 + 4: return rows_of<kType, 4, 4, true>(a, direct, s);
        default: break;
    }
    CHX_FAIL(CHX_HIP_EUNSUPPORTED, "linear plan: no kernel for %d tiles of rows and %d fragments", row_tiles, fragments);
}

template <LinearType kType>
int LinearKernels<kType>::tile(const LinearArgs& a, LinearTile t, hipStream_t s) {
    if (t == kTile64) return tile_of<kType, 2, 2, 2, true>(a, s);
    if constexpr (kType != kFloatFloat) return t == kTile256 ? tile_of<kType, 8, 2, 4, kType == kHalfHalf>(a, s) : tile_of<kType, 4, 2, 2, true>(a, s);
    CHX_FAIL(CHX_HIP_EUNSUPPORTED, "linear plan: no kernel for tiles of 128 rows of float32");
}

}  // namespace chx
