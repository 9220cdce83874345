// The kernels behind linear_plan.hip, instantiated by type in linear_half.hip, linear_int8.hip and linear_float.hip.
//
//   y[m, n] = act(scale[n] * sum_k x[m, k] w[n, k] + bias[n]) + r[m, n]
//
// The sums are float32 (matrix instructions of 16 x 16 results), the epilogue works on them in float32, and the result is
// rounded once.  w is the first operand of an instruction, so that a lane's results are neighbouring columns of one row of y.
#pragma once

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
    static constexpr int kElement = kFloat ? 4 : 2;                 // bytes of an element of x
    static constexpr int kChunk = 16 / kElement;                    // elements in 16 bytes
    static constexpr int kStep = 128 / kElement;                    // k of a step: 128 bytes of a row of x
    static constexpr int kUnits = kType == kHalfInt8 ? 1 : 2;       // units of w in a step
    static constexpr int kSteps = kType == kHalfInt8 ? 2 : 1;       // fragments of x (64 bytes of each of 16 rows) to a unit of w
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

// One fragment of w (for int8 its part `s`) times one of x.
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

template <LinearType kType>
__device__ __forceinline__ u32x4 operand(u32x4 w, int s) {
    if constexpr (kType == kHalfInt8) return halves_of_bytes(w[2 * s], w[2 * s + 1]);
    return w;
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

// gelu(v) = v Phi(v).  For float16 results Phi(-z) = exp(-z^2 / 2) P(t), t = 1 / (1 + 0.4 z), with P fitted by least squares to the relative
// error over 0 <= z <= 9: 2.6e-6, where rounding the result to float16 takes 4.9e-4.  Some 15 instructions; the library's erff takes three
// times as many, which a work-group that has its compute unit for itself hides under nothing.
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
    const float tail = p * __builtin_amdgcn_exp2f(-0.72134752f * z * z);  // Phi(-z)
    return v * (v > 0.f ? 1.f - tail : tail);
}

template <LinearType kType>
__device__ __forceinline__ float activated(float v, int32_t act) {
    switch (act) {
        case CHX_HIP_ACT_RELU: return v < 0.f ? 0.f : v;  // (a NaN stays)
        case CHX_HIP_ACT_GELU:
            if constexpr (kType == kFloatFloat) return 0.5f * v * erfcf(-0.70710678f * v);
            else return gelu_short(v);
        case CHX_HIP_ACT_GELU_TANH: {
            // 0.5 v (1 + tanh u) = v / (1 + exp(-2 u))
            const float u = 0.7978845608f * __builtin_fmaf(0.044715f * v * v, v, v);
            if constexpr (kType == kFloatFloat) return v / (1.f + expf(-2.f * u));
            else return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-2.8853901f * u));
        }
        case CHX_HIP_ACT_SILU:
            if constexpr (kType == kFloatFloat) return v / (1.f + expf(-v));
            else return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950f * v));
        default: return v;
    }
}

// kCount neighbouring columns (a multiple of 4, from a multiple of 4 on) of one row of the result.
template <LinearType kType, int kCount>
__device__ __forceinline__ void finish(const LinearArgs& a, float* v, int64_t row, int32_t n, const float* scale, const float* bias) {
    if (n >= a.N) return;
    const bool whole = n + kCount <= a.N;
    if (scale) {
#pragma unroll
        for (int i = 0; i < kCount; ++i) v[i] *= scale[i];
    }
    if (bias) {
#pragma unroll
        for (int i = 0; i < kCount; ++i) v[i] += bias[i];
    }
    if (a.activation != CHX_HIP_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < kCount; ++i) v[i] = activated<kType>(v[i], a.activation);
    }
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

// Tile `index` of the experts' tiles of `height` rows each, counted from expert 0 on.  Every wavefront finds it by itself, 64 experts at a time.
__device__ __forceinline__ Rows expert_rows(const LinearArgs& a, int32_t index, int32_t height) {
    const int lane = threadIdx.x & 63;
    for (int32_t e0 = 0; e0 < a.experts; e0 += 64) {
        const int32_t e = e0 + lane;
        int32_t lo = 0, hi = 0;
        if (e < a.experts) {  // (offsets from device memory: kept inside the order whatever they say)
            lo = min(max(a.offsets[e], 0), a.M);
            hi = min(max(a.offsets[e + 1], lo), a.M);
        }
        const int32_t tiles = (hi - lo + height - 1) / height;
        int32_t upto = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int32_t v = __shfl_up(upto, d);
            if (lane >= d) upto += v;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > index);
        if (past) {
            const int at = __builtin_ctzll(past);
            const int32_t first = __builtin_amdgcn_readlane(lo, at), end = __builtin_amdgcn_readlane(hi, at);
            const int32_t t = index - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(tiles, at));
            return {e0 + at, first + t * height, min(end - first - t * height, height)};
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

// ---- few rows ---------------------------------------------------------------------------------------
//
// Bound by the bytes of w, each read once.  A work-group takes kFragments fragments' columns (16 each) and all k, its kWaves wavefronts every
// kWaves-th unit of k: fragments go from memory straight into registers, kDeep units ahead of the products, and the wavefronts' sums
// are added in LDS, in one order.  x comes from the caches as fragments (rows that are not there repeat the last one; their results are dropped).
template <LinearType kType, int kRowTiles, int kFragments, int kWaves, bool kDirect, bool kExperts>
__global__ __launch_bounds__(64 * kWaves) void linear_rows_kernel(LinearArgs a) {
    using O = Of<kType>;
    constexpr int kDeep = kRowTiles * kFragments >= 8 ? 2 : 4;
    extern __shared__ f32x4 rows_sums[];  // [wave][row tile][fragment][lane]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t columns = blockIdx.x % a.tiles_n, tile = blockIdx.x / a.tiles_n;
    Rows t;
    if constexpr (kExperts) {
        t = expert_rows(a, tile, 16 * kRowTiles);
        if (t.count <= 0) return;
    } else {
        t = {0, tile * 16 * kRowTiles, min(a.M - tile * 16 * kRowTiles, 16 * kRowTiles)};
    }
    const int32_t fragment = columns * kFragments;  // of all: 4 to a group
    const char* w = a.w + t.expert * a.w_expert + (int64_t)(fragment >> 2) * a.w_group + (fragment & 3) * kFragment + lane * 16;
    const char* x[kRowTiles];
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i) {
        const int32_t row = max(row_at<kExperts>(a, t, min(16 * i + (lane & 15), t.count - 1)), 0);
        x[i] = a.x + (int64_t)(kExperts ? row / a.fan : row) * a.x_row;
    }
    const int32_t chunk = (lane >> 4) * O::kChunk;
    f32x4 acc[kRowTiles][kFragments];
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
        for (int f = 0; f < kFragments; ++f) acc[i][f] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Unit {
        u32x4 w[kFragments];
        u32x4 x[kRowTiles][O::kSteps];
    };
    auto load = [&](Unit& u, int32_t unit) {
#pragma unroll
        for (int f = 0; f < kFragments; ++f) u.w[f] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w + (int64_t)unit * kUnit + f * kFragment));
#pragma unroll
        for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
            for (int s = 0; s < O::kSteps; ++s) {
                const int32_t k = (unit * O::kSteps + s) * 4 * O::kChunk + chunk;
                if constexpr (kDirect) u.x[i][s] = *reinterpret_cast<const u32x4*>(x[i] + (int64_t)k * O::kElement);
                else u.x[i][s] = chunk_of<kType>(x[i], a.x_col, k, a.K);
            }
    };
    auto multiply = [&](const Unit& u) {
#pragma unroll
        for (int s = 0; s < O::kSteps; ++s)
#pragma unroll
            for (int f = 0; f < kFragments; ++f) {
                const u32x4 o = operand<kType>(u.w[f], s);
#pragma unroll
                for (int i = 0; i < kRowTiles; ++i) acc[i][f] = product<kType>(o, u.x[i][s], acc[i][f]);
            }
    };
    Unit ring[kDeep];
    const int32_t mine = a.units > wave ? (a.units - wave + kWaves - 1) / kWaves : 0;
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
        if (d < mine) load(ring[d], wave + d * kWaves);
    for (int32_t j = 0; j < mine; j += kDeep) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (j + d < mine) multiply(ring[d]);
            if (j + d + kDeep < mine) load(ring[d], wave + (j + d + kDeep) * kWaves);
        }
    }
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
        for (int f = 0; f < kFragments; ++f) rows_sums[((wave * kRowTiles + i) * kFragments + f) * 64 + lane] = acc[i][f];
    __syncthreads();
    for (int at = threadIdx.x; at < kRowTiles * kFragments * 64; at += 64 * kWaves) {
        const int l = at & 63, f = (at >> 6) % kFragments, i = (at >> 6) / kFragments;
        f32x4 sum = rows_sums[at];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum += rows_sums[v * kRowTiles * kFragments * 64 + at];
        const int32_t row = row_at<kExperts>(a, t, 16 * i + (l & 15));
        const int32_t n = ((fragment + f) >> 2) * kGroupRows + group_row((fragment + f) & 3, (l >> 4) * 4);
        if (row < 0) continue;
        float v[4] = {sum[0], sum[1], sum[2], sum[3]};
        const int64_t at_n = (int64_t)t.expert * a.n_padded + n;
        finish<kType, 4>(a, v, row, n, kType == kHalfInt8 ? a.scale + at_n : nullptr, a.bias ? a.bias + at_n : nullptr);
    }
}

// ---- tiles -------------------------------------------------------------------------------------------
//
// Both operands of a step (128 bytes of every row) are brought into LDS while the step before it is multiplied.  A row of x is eight pieces of
// 16 bytes; piece c of row r lies at place c ^ (r & 7), so that the sixteen rows that a fragment is read from do not meet in one bank.
__device__ __forceinline__ void copy_to_lds(uint32_t offset, const char* base, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}

template <LinearType kType, int kRowFragments, int kWavesM, int kWavesN, bool kDirect, bool kExperts>
__global__ __launch_bounds__(64 * kWavesM * kWavesN) void linear_tile_kernel(LinearArgs a) {
    using O = Of<kType>;
    constexpr int kThreads = 64 * kWavesM * kWavesN;
    constexpr int kBM = kWavesM * kRowFragments * 16, kGroups = kWavesN;
    constexpr int kBytesX = kBM * 128, kBytesW = kGroups * O::kUnits * kUnit, kStage = kBytesX + kBytesW;
    constexpr int kCopiesX = kBytesX / 16 / kThreads, kCopiesW = kBytesW / 16 / kThreads;
    extern __shared__ __attribute__((aligned(128))) char tile_lds[];
    int32_t* rows = reinterpret_cast<int32_t*>(tile_lds + 2 * kStage);  // of the result
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / kWavesN, wn = wave % kWavesN;
    // Work-groups that follow each other run on different XCDs, each with its own L2: an eighth of the tiles to each, in blocks
    // of 8 tiles of rows, so that what a block reads stays there.
    const int32_t all = a.tiles_m * a.tiles_n;
    int32_t id = blockIdx.x;
    {
        const int32_t q = all >> 3, rest = all & 7, xcd = id & 7;
        id = xcd * q + min(xcd, rest) + (id >> 3);
    }
    constexpr int32_t kBlock = 8;
    const int32_t block = id / (kBlock * a.tiles_n), height = min(a.tiles_m - block * kBlock, kBlock), inside = id - block * kBlock * a.tiles_n;
    const int32_t tm = block * kBlock + inside % height, tn = inside / height;
    Rows t;
    if constexpr (kExperts) {
        t = expert_rows(a, tm, kBM);
        if (t.count <= 0) return;
    } else {
        t = {0, tm * kBM, min(a.M - tm * kBM, kBM)};
    }
    for (int i = threadIdx.x; i < kBM; i += kThreads) rows[i] = row_at<kExperts>(a, t, i);

    // x: this thread's pieces of a step
    uint32_t x_at[kCopiesX];
    const char* x_row[kCopiesX];
    int32_t x_chunk[kCopiesX];
    const char* x_base = a.x + (kExperts ? 0 : (int64_t)t.first * a.x_row);
#pragma unroll
    for (int i = 0; i < kCopiesX; ++i) {
        const int slot = i * kThreads + threadIdx.x, r = slot >> 3;
        const int32_t row = max(row_at<kExperts>(a, t, min(r, t.count - 1)), 0);
        const int64_t off = kExperts ? (int64_t)(row / a.fan) * a.x_row : (int64_t)(row - t.first) * a.x_row;
        x_chunk[i] = (slot & 7) ^ (r & 7);
        x_row[i] = x_base + off;
        x_at[i] = (uint32_t)off + x_chunk[i] * 16;
    }
    // w: whole units, in the order in which they lie
    uint32_t w_at[kCopiesW];
    const char* w_base = a.w + t.expert * a.w_expert + (int64_t)tn * kGroups * a.w_group;
    const int32_t last_group = (a.N + kGroupRows - 1) / kGroupRows - 1 - tn * kGroups;
#pragma unroll
    for (int i = 0; i < kCopiesW; ++i) {
        const int at = (i * kThreads + threadIdx.x) * 16, g = at / (O::kUnits * kUnit);
        w_at[i] = (uint32_t)(min(g, last_group) * a.w_group) + at % (O::kUnits * kUnit);
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)tile_lds + wave * 1024;
    const int32_t steps = (a.K + O::kStep - 1) / O::kStep;

    u32x4 staged[kCopiesX];
    auto is_direct = [&](int32_t step) { return kDirect && (step + 1) * O::kStep <= a.K; };
    auto copy = [&](int32_t step, int buffer) {
        const uint32_t lds = lds0 + buffer * kStage;
        if (is_direct(step)) {
            const char* base = x_base + (int64_t)step * 128;
#pragma unroll
            for (int i = 0; i < kCopiesX; ++i) copy_to_lds(x_at[i], base, lds + i * kThreads * 16);
        } else {
#pragma unroll
            for (int i = 0; i < kCopiesX; ++i) staged[i] = chunk_of<kType>(x_row[i], a.x_col, step * O::kStep + x_chunk[i] * O::kChunk, a.K);
        }
        const char* base = w_base + (int64_t)step * (O::kUnits * kUnit);
#pragma unroll
        for (int i = 0; i < kCopiesW; ++i) copy_to_lds(w_at[i], base, lds + kBytesX + i * kThreads * 16);
    };
    auto settle = [&](int32_t step, int buffer) {
        if (!is_direct(step)) {
#pragma unroll
            for (int i = 0; i < kCopiesX; ++i) *reinterpret_cast<u32x4*>(tile_lds + buffer * kStage + (i * kThreads + threadIdx.x) * 16) = staged[i];
        }
    };

    f32x4 acc[kRowFragments][4];
#pragma unroll
    for (int i = 0; i < kRowFragments; ++i)
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[i][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int x_lane = (wm * kRowFragments * 16 + (lane & 15)) * 128, x_swizzle = lane & 7, x_quarter = lane >> 4;
    const int w_lane = kBytesX + wn * O::kUnits * kUnit + lane * 16;

    copy(0, 0);
    settle(0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int32_t step = 0; step < steps; ++step) {
        const int now = step & 1;
        if (step + 1 < steps) copy(step + 1, now ^ 1);
        const char* at = tile_lds + now * kStage;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            u32x4 w[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                if constexpr (kType == kHalfInt8) w[f] = operand<kType>(*reinterpret_cast<const u32x4*>(at + w_lane + f * kFragment), half);
                else w[f] = *reinterpret_cast<const u32x4*>(at + w_lane + half * kUnit + f * kFragment);
            }
#pragma unroll
            for (int i = 0; i < kRowFragments; ++i) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(at + x_lane + i * 16 * 128 + (((half * 4 + x_quarter) ^ x_swizzle) << 4));
#pragma unroll
                for (int f = 0; f < 4; ++f) acc[i][f] = product<kType>(w[f], x, acc[i][f]);
            }
        }
        if (step + 1 < steps) settle(step + 1, now ^ 1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }

    const int32_t n = (tn * kGroups + wn) * kGroupRows + (lane >> 4) * 16;
    const int64_t at_n = (int64_t)t.expert * a.n_padded + n;
    float scale[16], bias[16];
    if (n < a.N) {  // (both are filled up to whole groups)
        if constexpr (kType == kHalfInt8) {
#pragma unroll
            for (int i = 0; i < 16; ++i) scale[i] = a.scale[at_n + i];
        }
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < 16; ++i) bias[i] = a.bias[at_n + i];
        }
    }
#pragma unroll
    for (int i = 0; i < kRowFragments; ++i) {
        const int32_t row = rows[(wm * kRowFragments + i) * 16 + (lane & 15)];
        if (row < 0) continue;
        float v[16];
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[f * 4 + j] = acc[i][f][j];
        finish<kType, 16>(a, v, row, n, kType == kHalfInt8 ? scale : nullptr, a.bias ? bias : nullptr);
    }
}

// ---- launches ------------------------------------------------------------------------------------------

template <LinearType kType, int kRowTiles, int kFragments, bool kDirect, bool kExperts>
int launch_rows(const LinearArgs& a, hipStream_t s) {
    constexpr int kWaves = kRowTiles * kFragments >= 8 ? 4 : 8;
    constexpr int kLds = kWaves * kRowTiles * kFragments * 1024;
    linear_rows_kernel<kType, kRowTiles, kFragments, kWaves, kDirect, kExperts><<<(unsigned)(a.tiles_m * a.tiles_n), 64 * kWaves, kLds, s>>>(a);
    return launch_check("linear_rows_kernel");
}

template <LinearType kType, int kRowFragments, int kWavesM, int kWavesN, bool kDirect, bool kExperts>
int launch_tile(const LinearArgs& a, hipStream_t s) {
    constexpr int kBM = kWavesM * kRowFragments * 16;
    constexpr int kLds = 2 * (kBM * 128 + kWavesN * Of<kType>::kUnits * kUnit) + kBM * 4;
    auto kernel = linear_tile_kernel<kType, kRowFragments, kWavesM, kWavesN, kDirect, kExperts>;
    if constexpr (kLds > 65536)  // (has to be asked for, on every device)
        CHX_HIP_CALL(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
    kernel<<<(unsigned)(a.tiles_m * a.tiles_n), 64 * kWavesM * kWavesN, kLds, s>>>(a);
    return launch_check("linear_tile_kernel");
}

template <LinearType kType, int kRowTiles, int kFragments>
int rows_of(const LinearArgs& a, bool direct, hipStream_t s) {
    if (a.order) return direct ? launch_rows<kType, kRowTiles, kFragments, true, true>(a, s) : launch_rows<kType, kRowTiles, kFragments, false, true>(a, s);
    return direct ? launch_rows<kType, kRowTiles, kFragments, true, false>(a, s) : launch_rows<kType, kRowTiles, kFragments, false, false>(a, s);
}

template <LinearType kType, int kRowFragments, int kWavesM, int kWavesN>
int tile_of(const LinearArgs& a, bool direct, hipStream_t s) {
    if (a.order)
        return direct ? launch_tile<kType, kRowFragments, kWavesM, kWavesN, true, true>(a, s) : launch_tile<kType, kRowFragments, kWavesM, kWavesN, false, true>(a, s);
    return direct ? launch_tile<kType, kRowFragments, kWavesM, kWavesN, true, false>(a, s) : launch_tile<kType, kRowFragments, kWavesM, kWavesN, false, false>(a, s);
}

}  // namespace

template <LinearType kType>
int LinearKernels<kType>::rows(const LinearArgs& a, int row_tiles, int fragments, bool direct, hipStream_t s) {
    switch (row_tiles * 8 + fragments) {
        case 8 + 1: return rows_of<kType, 1, 1>(a, direct, s);
        case 8 + 2: return rows_of<kType, 1, 2>(a, direct, s);
        case 8 + 4: return rows_of<kType, 1, 4>(a, direct, s);
        case 16 + 1: return rows_of<kType, 2, 1>(a, direct, s);
        case 16 + 2: return rows_of<kType, 2, 2>(a, direct, s);
        case 16 + 4: return rows_of<kType, 2, 4>(a, direct, s);
        case 32 + 1: return rows_of<kType, 4, 1>(a, direct, s);
        case 32 + 2: return rows_of<kType, 4, 2>(a, direct, s);
        default: return rows_of<kType, 4, 4>(a, direct, s);
    }
}

template <LinearType kType>
int LinearKernels<kType>::tile(const LinearArgs& a, LinearTile t, bool direct, hipStream_t s) {
    return t == kTile256 ? tile_of<kType, 8, 2, 4>(a, direct, s) : tile_of<kType, 4, 2, 2>(a, direct, s);
}

}  // namespace chx
